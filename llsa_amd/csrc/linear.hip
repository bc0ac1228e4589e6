// The linear layers of a transformer block around the attention: products of a long matrix of token rows with a weight matrix,
// with bias, activation, gate and residual on the way out, and the products and sums of their backward.
//
//     forward   z = x W^T + b,   out = residual + gate * act(z)
//     backward  dz = dout * gate * act'(z),   dx = dz W,   dW = dz^T x,   db = sum dz,   dgate = sum over a sample's rows of dout * act(z)
//
// All three products are one kernel, C[m][n] = sum over k of X[m,k] Y[n,k], whose operands lie in memory either with the contraction
// along a row ("rows": x and W of the forward, dz of dx) or across the rows ("columns": W of dx, both operands of dW).
#include <algorithm>

#include "llsa_device.h"
#include "llsa_host.h"

namespace llsa {
namespace {

typedef __attribute__((ext_vector_type(4))) _Float16 f16x4;
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
template <typename T> struct Vec8;
template <> struct Vec8<bf16> { typedef bf16x8 type; typedef bf16x4 half; };
template <> struct Vec8<_Float16> { typedef f16x8 type; typedef f16x4 half; };
template <typename T> using vec8 = typename Vec8<T>::type;
template <typename T> using vec4 = typename Vec8<T>::half;

__device__ __forceinline__ f32x4 product16(bf16x8 a, bf16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x4 product16(f16x8 a, f16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }

// ---------------------------------------------------------------------------------------
// activations, in fp32.  Written with the logistic function: 0.5 (1 + tanh u) = s(2u), which saturates to 0 and 1 without an
// overflow.  The derivatives are taken at z held to +-16, where they are 0 and 1 to the last bit of fp32, so that a large z does not
// multiply an infinite inner derivative by zero.
// ---------------------------------------------------------------------------------------
constexpr float kGeluC = 0.7978845608028654f, kGeluA = 0.044715f, kRsqrt2 = 0.7071067811865476f, kRsqrt2Pi = 0.3989422804014327f;

__device__ __forceinline__ float logistic(float u) { return __builtin_amdgcn_rcpf(1.f + exp2_fast(-kLog2e * u)); }
__device__ __forceinline__ float activate(int act, float z) {
    switch (act) {
        case LLSA_ACT_SILU: return z * logistic(z);
        case LLSA_ACT_GELU: return 0.5f * z * erfcf(-z * kRsqrt2);
        case LLSA_ACT_GELU_TANH: return z * logistic(2.f * kGeluC * (z + kGeluA * z * z * z));
        default: return z;
    }
}
__device__ __forceinline__ float activate_slope(int act, float z) {
    z = z > 16.f ? 16.f : z < -16.f ? -16.f : z;              // (a NaN stays one)
    switch (act) {
        case LLSA_ACT_SILU: {
            const float s = logistic(z);
            return s * (1.f + z * (1.f - s));
        }
        case LLSA_ACT_GELU: return 0.5f * erfcf(-z * kRsqrt2) + z * kRsqrt2Pi * exp2_fast(-0.5f * kLog2e * z * z);
        case LLSA_ACT_GELU_TANH: {
            const float s = logistic(2.f * kGeluC * (z + kGeluA * z * z * z));
            return s * (1.f + 2.f * kGeluC * z * (1.f - s) * (1.f + 3.f * kGeluA * z * z));
        }
        default: return 1.f;
    }
}

// ---------------------------------------------------------------------------------------
// operands in LDS
//
// A step takes 64 of the contraction.  Copies go straight into LDS, 16 bytes a lane and 1 KB an instruction, so a tile's layout is
// the order of its source pieces; it is the source address that is permuted, never the place in LDS.
//   rows     ROWS rows of 64 elements (128 bytes).  Piece p (8 elements) of row r holds the row's piece p ^ ((r >> 1) & 7): the 16 rows a
//            fragment read touches then lie in 16 different 16-byte columns of the 256 bytes that all banks hold.
//   columns  64 rows of ROWS elements.  32-byte granule g of row k holds the row's granule g ^ f(k), f out of bits 0, 1 and 3 of k
//            (ROWS = 64: 1 and 3): the transposing read takes granules of 4 neighbouring rows in each group of 16 lanes and of
//            rows 8 further in the next, which then lie in different banks.
// What lies outside the matrix: rows are clamped (their results are not stored), and beyond the end of the contraction zeros are fetched.
// ---------------------------------------------------------------------------------------
constexpr int kStep = 64;                 // of the contraction
__device__ const u32x4 kZeros[1] = {{0u, 0u, 0u, 0u}};

template <typename T>
__device__ __forceinline__ void copy_to_lds(const T* g_lane, T* lds_wave_base) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)g_lane, (__attribute__((address_space(3))) void*)lds_wave_base, 16, 0, 0);
}

template <typename T, bool COLUMNS, int ROWS>
struct Operand {
    static constexpr int kCopies = ROWS * kStep / 512 / 4;    // instructions of a wave for one step
    static constexpr int kPerRow = ROWS / 8;                  // columns: 16-byte pieces of a row
    static constexpr int kMaskG = ROWS == 64 ? 3 : 7;
    unsigned off[kCopies];                                    // elements from the step's first, of this lane's pieces
    int place[kCopies];                                       // along the contraction

    static __device__ __forceinline__ int turn(int k) { return ROWS == 64 ? ((k >> 1) & 1) | ((k >> 3) & 1) << 1 : (k & 3) | ((k >> 3) & 1) << 2; }

    // left: rows (columns: elements of a row, a multiple of 8) from the tile's first to the matrix's last
    __device__ __forceinline__ void init(int wave, int lane, int64_t ld, int left) {
#pragma unroll
        for (int j = 0; j < kCopies; j++) {
            const int i = wave * kCopies + j;
            if constexpr (COLUMNS) {
                const int k = i * (64 / kPerRow) + lane / kPerRow, unit = lane % kPerRow;
                const int col = (((unit >> 1) ^ turn(k)) * 2 + (unit & 1)) * 8;
                place[j] = k;
                off[j] = (unsigned)(k * ld) + (unsigned)min(col, left - 8);
            } else {
                const int r = i * 8 + (lane >> 3), piece = (lane & 7) ^ ((r >> 1) & 7);
                place[j] = piece * 8;
                off[j] = (unsigned)(min(r, left - 1) * ld) + (unsigned)(piece * 8);
            }
        }
    }
    // k_left: what is left of the contraction from this step on
    __device__ __forceinline__ void request(const T* base, T* tile, int wave, int k_left) const {
        if (k_left >= kStep) {
#pragma unroll
            for (int j = 0; j < kCopies; j++) copy_to_lds(base + off[j], tile + (wave * kCopies + j) * 512);
        } else {
#pragma unroll
            for (int j = 0; j < kCopies; j++) copy_to_lds(place[j] < k_left ? base + off[j] : reinterpret_cast<const T*>(kZeros), tile + (wave * kCopies + j) * 512);
        }
    }
    // the fragment of the 16 rows from `row` on (a multiple of 16), half `ks` of the step: lane l gets row l%16, contraction 32 ks + 8 (l/16) .. +7
    static __device__ __forceinline__ vec8<T> fragment(const T* tile, int row, int ks, int lane) {
        if constexpr (COLUMNS) {
            const int q = lane >> 4, j = lane & 15, k = 32 * ks + 8 * q + (j >> 2);
            const T* p = tile + k * ROWS + ((row >> 4) ^ turn(8 * q + (j >> 2))) * 16 + (j & 3) * 4;
            const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)p);
            const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(p + 4 * ROWS));
            return __builtin_shufflevector(__builtin_bit_cast(vec4<T>, lo), __builtin_bit_cast(vec4<T>, hi), 0, 1, 2, 3, 4, 5, 6, 7);
        } else {
            const int r = row + (lane & 15), piece = (4 * ks + (lane >> 4)) ^ ((lane >> 1) & 7);
            return *reinterpret_cast<const vec8<T>*>(tile + r * kStep + piece * 8);
        }
    }
};

// ---------------------------------------------------------------------------------------
// the product
// ---------------------------------------------------------------------------------------
template <typename T>
struct Product {
    const T *x, *y;
    int64_t ldx, ldy;
    int M, N;                             // rows (token rows, or channels out of dW) and columns of C
    int nx, ny;                           // elements of a row of x / y where it has its columns in C (a multiple of 8)
    int64_t K;                            // contraction
    int64_t k_per_split;                  // of one piece of it (a multiple of 64)
    int tiles_m, tiles_n, group;          // tiles are taken `group` rows of tiles at a time
    // way out
    const T *bias, *gate, *residual, *slope_at;
    int64_t s_gate, ldr, ldz, ldo;
    T *out, *z;
    int per_sample, act;
    int wide;                             // N and the pointers and strides of bias, gate and residual allow 16-byte accesses
    int wide_out;                         // and those of out; or its rows are padded with zeros to a multiple of 8 elements (those of z always are)
    // dW: pieces of the sum
    float *part, *part_sum;               // [split][M][ld_part], [split][M] or NULL
    int64_t ld_part;
};

// Workgroups go round the eight XCDs: each gets a run of consecutive tiles, which share rows of x and y in its L2.
__device__ __forceinline__ int xcd_order(int id, int total) {
    const int xcd = id & 7, q = total >> 3, r = total & 7;
    return xcd * q + min(xcd, r) + (id >> 3);
}

template <typename T>
__device__ __forceinline__ void load8(float (&v)[8], const T* p, bool wide, int n) {
    if (wide) {
        const vec8<T> a = *reinterpret_cast<const vec8<T>*>(p);
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = (float)a[e];
    } else {
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = e < n ? (float)p[e] : 0.f;
    }
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&v)[8], bool wide, int n) {
    if (wide) {
        vec8<T> a;
#pragma unroll
        for (int e = 0; e < 8; e++) a[e] = (T)v[e];
        *reinterpret_cast<vec8<T>*>(p) = a;
    } else {
#pragma unroll
        for (int e = 0; e < 8; e++)
            if (e < n) p[e] = (T)v[e];
    }
}

// Eight values of one row of C on their way out: columns n .. n + 7 (left of them inside the matrix) of row m
template <typename T>
__device__ __forceinline__ void way_out(const Product<T>& a, float (&v)[8], const float (&bias)[8], int64_t m, int sample, int n, int left) {
    const bool wide = a.wide;
    if (a.bias != nullptr) {
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] += bias[e];
    }
    if (a.z != nullptr) store8(a.z + m * a.ldz + n, v, true, 8);
    if (a.act != LLSA_ACT_NONE) {
        if (a.slope_at != nullptr) {
            float z[8];
            load8(z, a.slope_at + m * a.ldz + n, true, 8);
#pragma unroll
            for (int e = 0; e < 8; e++) v[e] *= activate_slope(a.act, z[e]);
        } else {
#pragma unroll
            for (int e = 0; e < 8; e++) v[e] = activate(a.act, v[e]);
        }
    }
    if (a.gate != nullptr) {
        float g[8];
        load8(g, a.gate + sample * a.s_gate + n, wide, left);
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] *= g[e];
    }
    if (a.residual != nullptr) {
        float r[8];
        load8(r, a.residual + m * a.ldr + n, wide, left);
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] += r[e];
    }
    if (a.wide_out && left < 8) {
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = e < left ? v[e] : 0.f;
    }
    store8(a.out + m * a.ldo + n, v, a.wide_out, left);
}

template <typename T, bool XC, bool YC, int BM, int BN>
__global__ __launch_bounds__(256, 2) void product_kernel(const Product<T> a) {
    constexpr int WM = BM / 2, WN = BN / 2, MT = WM / 16, NT = WN / 16, kTileX = BM * kStep, kTileY = BN * kStep;
    HIP_DYNAMIC_SHARED(char, shared)
    T* const lds = reinterpret_cast<T*>(shared);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int quad = lane >> 4;

    const int per_split = a.tiles_m * a.tiles_n;
    const int at = xcd_order((int)blockIdx.x, (int)gridDim.x);
    const int split = at / per_split, tile = at - split * per_split;
    const int in_group = a.group * a.tiles_n, g = tile / in_group, rest = tile - g * in_group;
    const int rows_here = min(a.group, a.tiles_m - g * a.group);
    const int tn = rest / rows_here, tm = g * a.group + rest - tn * rows_here;
    const int m0 = tm * BM, n0 = tn * BN;
    const int64_t k0 = (int64_t)split * a.k_per_split, k1 = min(a.K, k0 + a.k_per_split);

    Operand<T, XC, BM> ox;
    Operand<T, YC, BN> oy;
    ox.init(wave, lane, a.ldx, min(BM, (XC ? a.nx : a.M) - m0));
    oy.init(wave, lane, a.ldy, min(BN, (YC ? a.ny : a.N) - n0));
    const T* px = a.x + (XC ? k0 * a.ldx + m0 : (int64_t)m0 * a.ldx + k0);
    const T* py = a.y + (YC ? k0 * a.ldy + n0 : (int64_t)n0 * a.ldy + k0);
    const int64_t stepx = XC ? kStep * a.ldx : kStep, stepy = YC ? kStep * a.ldy : kStep;

    const int wm = (wave & 1) * WM, wn = (wave >> 1) * WN;
    const bool sums = XC && a.part_sum != nullptr && tn == 0 && wn == 0;
    f32x4 acc[NT][MT], sum[XC ? MT : 1];
#pragma unroll
    for (int i = 0; i < NT; i++)
#pragma unroll
        for (int j = 0; j < MT; j++) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < (XC ? MT : 1); j++) sum[j] = f32x4{0.f, 0.f, 0.f, 0.f};
    vec8<T> ones;
#pragma unroll
    for (int e = 0; e < 8; e++) ones[e] = (T)1.f;

    const int steps = (int)((k1 - k0 + kStep - 1) / kStep);
    int64_t k_left = k1 - k0;
    auto request = [&](int buffer) {
        T* const t = lds + buffer * (kTileX + kTileY);
        const int left = (int)min(k_left, (int64_t)kStep);
        ox.request(px, t, wave, left);
        oy.request(py, t + kTileX, wave, left);
        px += stepx;
        py += stepy;
        k_left -= kStep;
    };
    request(0);
    for (int s = 0; s < steps; s++) {
        wait_vm0();
        __syncthreads();                                      // everyone's copies of this step are there, and everyone is done with the other buffer
        if (s + 1 < steps) request((s + 1) & 1);
        const T* const tx = lds + (s & 1) * (kTileX + kTileY);
        const T* const ty = tx + kTileX;
#pragma unroll
        for (int ks = 0; ks < 2; ks++) {
            vec8<T> fx[MT], fy[NT];
#pragma unroll
            for (int j = 0; j < MT; j++) fx[j] = Operand<T, XC, BM>::fragment(tx, wm + 16 * j, ks, lane);
#pragma unroll
            for (int i = 0; i < NT; i++) fy[i] = Operand<T, YC, BN>::fragment(ty, wn + 16 * i, ks, lane);
#pragma unroll
            for (int i = 0; i < NT; i++)
#pragma unroll
                for (int j = 0; j < MT; j++) acc[i][j] = product16(fy[i], fx[j], acc[i][j]);
            if constexpr (XC) {
                if (sums) {
#pragma unroll
                    for (int j = 0; j < MT; j++) sum[j] = product16(ones, fx[j], sum[j]);
                }
            }
        }
    }

    int sample[MT];
#pragma unroll
    for (int j = 0; j < MT; j++) sample[j] = !XC && a.gate != nullptr ? (m0 + wm + 16 * j + (lane & 15)) / a.per_sample : 0;
    // Lane l holds rows n of four: columns 4 (l/16) .. +3 of every 16, of row l%16 of C.  Swapped between sixteens of lanes, a pair of tiles gives it
    // eight neighbouring ones, so that everything on the way out is read and written in pieces of 16 bytes.
#pragma unroll
    for (int p = 0; p < NT / 2; p++) {
        const int n = n0 + wn + 32 * p + 16 * (quad & 1) + 8 * (quad >> 1), left = a.N - n;
        float bias[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        if (!XC && a.bias != nullptr && left > 0) load8(bias, a.bias + n, a.wide, left);
#pragma unroll
        for (int j = 0; j < MT; j++) {
            const int m = m0 + wm + 16 * j + (lane & 15);
            float v[8];
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const u32x2 w = __builtin_amdgcn_permlane16_swap(__float_as_uint(acc[2 * p][j][e]), __float_as_uint(acc[2 * p + 1][j][e]), false, false);
                v[e] = __uint_as_float(w[0]);
                v[4 + e] = __uint_as_float(w[1]);
            }
            if (m >= a.M || left <= 0) continue;
            if constexpr (XC) {
                float* const o = a.part + ((int64_t)split * a.M + m) * a.ld_part + n;
                *reinterpret_cast<f32x4*>(o) = f32x4{v[0], v[1], v[2], v[3]};
                *reinterpret_cast<f32x4*>(o + 4) = f32x4{v[4], v[5], v[6], v[7]};
            } else {
                way_out(a, v, bias, m, sample[j], n, left);
            }
        }
    }
    if constexpr (XC) {
        if (sums && quad == 0) {
#pragma unroll
            for (int j = 0; j < MT; j++) {
                const int m = m0 + wm + 16 * j + lane;
                if (m < a.M) a.part_sum[(int64_t)split * a.M + m] = sum[j][0];
            }
        }
    }
}

// The pieces of dW and db added up
template <typename T>
__global__ __launch_bounds__(256) void product_join_kernel(const float* part, const float* part_sum, T* out, int64_t ldo, T* sums, int64_t M, int N, int64_t ld_part,
                                                           int splits) {
    const int64_t n4 = ld_part / 4, i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i < M * n4) {
        const int64_t m = i / n4;
        const int n = (int)(i - m * n4) * 4;
        f32x4 v = {0.f, 0.f, 0.f, 0.f};
        for (int s = 0; s < splits; s++) v += *reinterpret_cast<const f32x4*>(part + ((int64_t)s * M + m) * ld_part + n);
#pragma unroll
        for (int e = 0; e < 4; e++)
            if (n + e < N) out[m * ldo + n + e] = (T)v[e];
    } else if (part_sum != nullptr && i - M * n4 < M) {
        const int64_t m = i - M * n4;
        float v = 0.f;
        for (int s = 0; s < splits; s++) v += part_sum[(int64_t)s * M + m];
        sums[m] = (T)v;
    }
}

// ---------------------------------------------------------------------------------------
// dz = dout * gate * act'(z), and pieces of dgate = sum over a sample's rows of dout * act(z).  A workgroup takes 128 columns of up to `rows` rows
// of one sample: 16 threads along a row, 16 rows at a time.
// ---------------------------------------------------------------------------------------
constexpr int kDzColumns = 128;
template <typename T>
struct Dz {
    const T *dout, *z, *gate;
    int64_t ldd, ldz, s_gate, lddz, per_sample;
    T* dz;
    float* part;                          // [sample][piece][N] or NULL
    int N, act, pieces, rows, columns, wide;      // columns: workgroups along a row
};
template <typename T>
__global__ __launch_bounds__(256) void dz_kernel(const Dz<T> a) {
    __shared__ float sum[16][kDzColumns];
    const int tid = threadIdx.x, at = (int)blockIdx.x / a.columns, n0 = ((int)blockIdx.x - at * a.columns) * kDzColumns;
    const int c = (tid & 15) * 8, n = n0 + c, left = a.N - n, sample = at / a.pieces, piece = at - sample * a.pieces;
    const int64_t t0 = (int64_t)piece * a.rows, t1 = min(a.per_sample, t0 + a.rows);
    float g[8], s[8];
#pragma unroll
    for (int e = 0; e < 8; e++) g[e] = 1.f, s[e] = 0.f;
    if (left > 0) {
        if (a.gate != nullptr) load8(g, a.gate + sample * a.s_gate + n, a.wide, left);
        for (int64_t t = t0 + (tid >> 4); t < t1; t += 16) {
            const int64_t m = sample * a.per_sample + t;
            float d[8], z[8], v[8];
            load8(d, a.dout + m * a.ldd + n, a.wide, left);
            if (a.z != nullptr) load8(z, a.z + m * a.ldz + n, true, 8);
#pragma unroll
            for (int e = 0; e < 8; e++) {
                v[e] = d[e] * g[e];
                if (a.act != LLSA_ACT_NONE) v[e] *= activate_slope(a.act, z[e]);
                if (a.part != nullptr) s[e] += d[e] * activate(a.act, z[e]);
                if (e >= left) v[e] = 0.f;                    // (the rows of dz are padded with zeros)
            }
            store8(a.dz + m * a.lddz + n, v, true, 8);
        }
    }
    if (a.part == nullptr) return;
#pragma unroll
    for (int e = 0; e < 8; e++) sum[tid >> 4][c + e] = s[e];
    __syncthreads();
    const int col = n0 + tid;
    if (tid < kDzColumns && col < a.N) {
        float v = 0.f;
#pragma unroll
        for (int r = 0; r < 16; r++) v += sum[r][tid];
        a.part[(int64_t)at * a.N + col] = v;
    }
}
template <typename T>
__global__ __launch_bounds__(256) void dgate_kernel(const float* part, T* dgate, int64_t total, int N, int pieces) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= total) return;
    const int64_t b = i / N;
    const int n = (int)(i - b * N);
    float v = 0.f;
    for (int p = 0; p < pieces; p++) v += part[(b * pieces + p) * N + n];
    dgate[i] = (T)v;
}

// Rows of an odd length or at odd addresses, copied to rows that the products can read: 16-byte aligned, padded with zeros
__global__ __launch_bounds__(256) void pad_kernel(const uint16_t* x, int64_t ldx, uint16_t* y, int64_t ldy, int64_t rows, int cols) {
    const int64_t per = ldy / 8, i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= rows * per) return;
    const int64_t r = i / per;
    const int c = (int)(i - r * per) * 8;
    typedef __attribute__((ext_vector_type(8))) uint16_t u16x8;
    u16x8 v;
#pragma unroll
    for (int e = 0; e < 8; e++) v[e] = c + e < cols ? x[r * ldx + c + e] : (uint16_t)0;
    *reinterpret_cast<u16x8*>(y + r * ldy + c) = v;
}

// ---------------------------------------------------------------------------------------
// launches
// ---------------------------------------------------------------------------------------
constexpr int64_t kMaxGrid = (int64_t(1) << 31) - 1;
int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

template <typename T, bool XC, bool YC, int BM, int BN>
int launch_tiles(Product<T>& a, int splits, hipStream_t stream) {
    const int64_t tm = ceil_div(a.M, BM), tn = ceil_div(a.N, BN);
    if (tm * tn * splits > kMaxGrid) return fail(-1, "linear: too many rows");
    a.tiles_m = (int)tm;
    a.tiles_n = (int)tn;
    constexpr size_t lds = 2 * (BM + BN) * kStep * sizeof(T);
    hipLaunchKernelGGL(HIP_KERNEL_NAME(product_kernel<T, XC, YC, BM, BN>), dim3((unsigned)(tm * tn * splits)), dim3(256), lds, stream, a);
    return 0;
}
template <typename T, bool XC, bool YC>
int launch_product(Product<T>& a, int splits, hipStream_t stream) {
    a.group = (int64_t)a.N * a.K <= (1 << 20) || XC ? 1 : 8;  // (rows of tiles that share y while it does not fit the L2 beside them)
    if (ceil_div(a.M, 128) * ceil_div(a.N, 128) * splits >= 256) return launch_tiles<T, XC, YC, 128, 128>(a, splits, stream);
    return launch_tiles<T, XC, YC, 64, 64>(a, splits, stream);
}

bool wide8(const void* p, int64_t ld) { return p == nullptr || (aligned16(p) && ld % 8 == 0); }

// The pieces of dW's contraction over the token rows
struct Pieces { int count; int64_t length; };
Pieces weight_pieces(int64_t M, int N, int K) {
    const int64_t tiles = ceil_div(N, 128) * ceil_div(K, 128);
    int64_t count = std::max<int64_t>(1, std::min(512 / tiles, ceil_div(M, 512)));
    const int64_t length = ceil_div(ceil_div(M, count), kStep) * kStep;
    return {(int)ceil_div(M, length), length};
}
int64_t pad8(int64_t n) { return (n + 7) / 8 * 8; }

constexpr int64_t kMaxRows = (int64_t(1) << 31) - (1 << 16);
constexpr int64_t kMaxLd = int64_t(1) << 23;                  // 128 rows of 16 bits then lie within 2^32 bytes
bool rows16(const void* p, int64_t ld) { return p != nullptr && aligned16(p) && ld % 8 == 0 && ld > 0 && ld <= kMaxLd; }

int check_sizes(const char* what, int64_t M, int N, int K, int dtype, int act) {
    LLSA_REQUIRE(M >= 0 && M <= kMaxRows && N > 0 && K > 0 && N < (1 << 23) && K < (1 << 23), "%s: bad sizes (M %lld, N %d, K %d)", what, (long long)M, N, K);
    LLSA_REQUIRE(dtype == LLSA_DTYPE_BF16 || dtype == LLSA_DTYPE_F16, "%s: bf16 or fp16 only", what);
    LLSA_REQUIRE(act >= LLSA_ACT_NONE && act <= LLSA_ACT_GELU_TANH, "%s: unknown activation %d", what, act);
    return 0;
}

template <typename T>
int linear_fwd(const llsa_linear_args& q, hipStream_t stream) {
    Product<T> a{};
    a.x = (const T*)q.x; a.ldx = q.ldx;
    a.y = (const T*)q.w; a.ldy = q.ldw;
    a.M = (int)q.M; a.N = q.N; a.K = q.K; a.k_per_split = ceil_div(q.K, kStep) * kStep;
    a.bias = (const T*)q.bias; a.gate = (const T*)q.gate; a.s_gate = q.s_gate; a.per_sample = (int)q.per_sample;
    a.residual = (const T*)q.residual; a.ldr = q.ldr;
    a.out = (T*)q.out; a.ldo = q.ldo; a.z = (T*)q.z; a.ldz = q.ldz;
    a.act = q.act;
    a.wide = q.N % 8 == 0 && wide8(q.bias, 0) && wide8(q.gate, q.s_gate) && wide8(q.residual, q.ldr);
    a.wide_out = (q.N % 8 == 0 && wide8(q.out, q.ldo)) || q.padded;
    if (int rc = launch_product<T, false, false>(a, 1, stream)) return rc;
    return launch_status("linear_fwd");
}
template <typename T>
int linear_dx(const llsa_linear_args& q, hipStream_t stream) {
    Product<T> a{};
    a.x = (const T*)q.dz; a.ldx = q.lddz;
    a.y = (const T*)q.w; a.ldy = q.ldw;
    a.M = (int)q.M; a.N = q.K; a.ny = (int)pad8(q.K); a.K = q.N; a.k_per_split = ceil_div(q.N, kStep) * kStep;
    a.out = (T*)q.out; a.ldo = q.ldo;
    a.slope_at = (const T*)q.z; a.ldz = q.ldz; a.act = q.z != nullptr ? q.act : LLSA_ACT_NONE;
    a.wide_out = (q.K % 8 == 0 && wide8(q.out, q.ldo)) || q.padded;
    if (int rc = launch_product<T, false, true>(a, 1, stream)) return rc;
    return launch_status("linear_dx");
}
template <typename T>
int linear_dw(const llsa_linear_args& q, hipStream_t stream) {
    const Pieces p = weight_pieces(q.M, q.N, q.K);
    Product<T> a{};
    a.x = (const T*)q.dz; a.ldx = q.lddz; a.nx = (int)pad8(q.N);
    a.y = (const T*)q.x; a.ldy = q.ldx; a.ny = (int)pad8(q.K);
    a.M = q.N; a.N = q.K; a.K = q.M; a.k_per_split = p.length;
    a.ld_part = pad8(q.K);
    a.part = (float*)q.workspace;
    a.part_sum = q.dbias != nullptr ? a.part + (int64_t)p.count * a.M * a.ld_part : nullptr;
    if (int rc = launch_product<T, true, true>(a, p.count, stream)) return rc;
    const int64_t threads = (int64_t)a.M * (a.ld_part / 4) + (q.dbias != nullptr ? a.M : 0);
    hipLaunchKernelGGL(HIP_KERNEL_NAME(product_join_kernel<T>), dim3((unsigned)ceil_div(threads, 256)), dim3(256), 0, stream, a.part, a.part_sum, (T*)q.out, q.ldo,
                       (T*)q.dbias, a.M, a.N, a.ld_part, p.count);
    return launch_status("linear_dw");
}
struct DzPieces { int count, rows; };
DzPieces dz_pieces(int64_t M, int64_t per_sample, int N) {
    // about 2048 workgroups, each of at least 32 rows
    const int64_t cols = ceil_div(N, kDzColumns), samples = M / per_sample;
    const int64_t want = std::max<int64_t>(1, 2048 / std::max<int64_t>(1, cols * samples));
    const int64_t rows = std::max<int64_t>(32, ceil_div(ceil_div(per_sample, want), 16) * 16);
    return {(int)ceil_div(per_sample, rows), (int)rows};
}
template <typename T>
int linear_dz(const llsa_linear_args& q, hipStream_t stream) {
    const DzPieces p = dz_pieces(q.M, q.per_sample, q.N);
    const int64_t samples = q.M / q.per_sample;
    Dz<T> a{};
    a.dout = (const T*)q.dout; a.ldd = q.lddout; a.z = (const T*)q.z; a.ldz = q.ldz;
    a.gate = (const T*)q.gate; a.s_gate = q.s_gate; a.per_sample = q.per_sample;
    a.dz = (T*)q.dz_out; a.lddz = q.lddz; a.N = q.N; a.act = q.act; a.pieces = p.count; a.rows = p.rows; a.columns = (int)ceil_div(q.N, kDzColumns);
    a.wide = q.N % 8 == 0 && wide8(q.dout, q.lddout) && wide8(q.gate, q.s_gate);
    a.part = q.dgate != nullptr ? (float*)q.workspace : nullptr;
    LLSA_REQUIRE(samples * p.count * a.columns <= kMaxGrid, "linear_dz: too many rows");
    hipLaunchKernelGGL(HIP_KERNEL_NAME(dz_kernel<T>), dim3((unsigned)(samples * p.count * a.columns)), dim3(256), 0, stream, a);
    if (q.dgate != nullptr)
        hipLaunchKernelGGL(HIP_KERNEL_NAME(dgate_kernel<T>), dim3((unsigned)ceil_div(samples * q.N, 256)), dim3(256), 0, stream, a.part, (T*)q.dgate, samples * q.N, q.N,
                           p.count);
    return launch_status("linear_dz");
}
}  // namespace
}  // namespace llsa

using namespace llsa;

#define BY_TYPE(fn) (a->dtype == LLSA_DTYPE_BF16 ? fn<bf16>(*a, (hipStream_t)stream) : fn<_Float16>(*a, (hipStream_t)stream))

extern "C" int64_t llsa_linear_dw_workspace_bytes(int64_t M, int N, int K) {
    if (M <= 0 || N <= 0 || K <= 0) return 0;
    return 4 * (int64_t)weight_pieces(M, N, K).count * N * (pad8(K) + 1);
}
extern "C" int64_t llsa_linear_dz_workspace_bytes(int64_t M, int64_t per_sample, int N) {
    if (M <= 0 || N <= 0 || per_sample <= 0) return 0;
    return 4 * (M / per_sample) * dz_pieces(M, per_sample, N).count * N;
}
extern "C" int llsa_linear_fwd(const llsa_linear_args* a, void* stream) {
    LLSA_REQUIRE(a != nullptr, "linear_fwd: no arguments");
    if (int rc = check_sizes("linear_fwd", a->M, a->N, a->K, a->dtype, a->act)) return rc;
    if (a->M == 0) return 0;
    LLSA_REQUIRE(rows16(a->x, a->ldx) && rows16(a->w, a->ldw) && a->K % 8 == 0 && a->ldx >= a->K && a->ldw >= a->K,
                 "linear_fwd: rows of x and w must be 16-byte aligned and a multiple of 8 long (zeros beyond the end)");
    LLSA_REQUIRE(a->out != nullptr && (!a->padded || (rows16(a->out, a->ldo) && a->ldo >= pad8(a->N))), "linear_fwd: output, padded rows 16-byte aligned and a multiple of 8 long");
    LLSA_REQUIRE(a->z == nullptr || (rows16(a->z, a->ldz) && a->ldz >= pad8(a->N)), "linear_fwd: rows of z must be 16-byte aligned and padded to a multiple of 8");
    LLSA_REQUIRE(a->gate == nullptr || a->per_sample > 0, "linear_fwd: rows of a sample");
    return BY_TYPE(linear_fwd);
}
extern "C" int llsa_linear_dx(const llsa_linear_args* a, void* stream) {
    LLSA_REQUIRE(a != nullptr, "linear_dx: no arguments");
    if (int rc = check_sizes("linear_dx", a->M, a->N, a->K, a->dtype, a->act)) return rc;
    if (a->M == 0) return 0;
    LLSA_REQUIRE(rows16(a->dz, a->lddz) && rows16(a->w, a->ldw) && a->lddz >= pad8(a->N) && a->ldw >= pad8(a->K),
                 "linear_dx: rows of dz and w must be 16-byte aligned and padded to a multiple of 8");
    LLSA_REQUIRE(a->out != nullptr && (!a->padded || (rows16(a->out, a->ldo) && a->ldo >= pad8(a->K))), "linear_dx: output, padded rows 16-byte aligned and a multiple of 8 long");
    LLSA_REQUIRE(a->z == nullptr || (rows16(a->z, a->ldz) && a->ldz >= pad8(a->K)), "linear_dx: rows of z must be 16-byte aligned and padded to a multiple of 8");
    return BY_TYPE(linear_dx);
}
extern "C" int llsa_linear_dw(const llsa_linear_args* a, void* stream) {
    LLSA_REQUIRE(a != nullptr, "linear_dw: no arguments");
    if (int rc = check_sizes("linear_dw", a->M, a->N, a->K, a->dtype, a->act)) return rc;
    LLSA_REQUIRE(a->M > 0, "linear_dw: no rows");
    LLSA_REQUIRE(rows16(a->dz, a->lddz) && rows16(a->x, a->ldx) && a->lddz >= pad8(a->N) && a->ldx >= pad8(a->K),
                 "linear_dw: rows of dz and x must be 16-byte aligned and padded to a multiple of 8");
    LLSA_REQUIRE(a->out != nullptr && a->workspace != nullptr && aligned16(a->workspace), "linear_dw: output and workspace (16-byte aligned)");
    return BY_TYPE(linear_dw);
}
extern "C" int llsa_linear_dz(const llsa_linear_args* a, void* stream) {
    LLSA_REQUIRE(a != nullptr, "linear_dz: no arguments");
    if (int rc = check_sizes("linear_dz", a->M, a->N, 8, a->dtype, a->act)) return rc;
    if (a->M == 0) return 0;
    LLSA_REQUIRE(a->per_sample > 0 && a->M % a->per_sample == 0, "linear_dz: rows of a sample");
    LLSA_REQUIRE(a->dout != nullptr && rows16(a->dz_out, a->lddz) && a->lddz >= pad8(a->N), "linear_dz: dz must have rows that are 16-byte aligned and padded to a multiple of 8");
    LLSA_REQUIRE((a->act == LLSA_ACT_NONE && a->dgate == nullptr) || (rows16(a->z, a->ldz) && a->ldz >= pad8(a->N)), "linear_dz: z is needed, in padded rows");
    LLSA_REQUIRE(a->dgate == nullptr || a->workspace != nullptr, "linear_dz: workspace");
    return BY_TYPE(linear_dz);
}
extern "C" int llsa_pad_rows(const void* x, int64_t ldx, void* y, int64_t ldy, int64_t rows, int cols, void* stream) {
    LLSA_REQUIRE(rows >= 0 && cols > 0 && ldy >= cols && rows16(y, ldy) && x != nullptr, "pad_rows: bad arguments");
    if (rows == 0) return 0;
    LLSA_REQUIRE(ceil_div(rows * (ldy / 8), 256) <= kMaxGrid, "pad_rows: too many rows");
    hipLaunchKernelGGL(pad_kernel, dim3((unsigned)ceil_div(rows * (ldy / 8), 256)), dim3(256), 0, (hipStream_t)stream, (const uint16_t*)x, ldx, (uint16_t*)y, ldy, rows, cols);
    return launch_status("pad_rows");
}
