// The linear layers of a transformer block around the attention: products of a long matrix of token rows with a weight matrix,
// with bias, activation, gate and residual on the way out, and the products and sums of their backward.
//
//     forward   z = x W^T + b,   out = residual + gate * act(z)
//     backward  dz = dout * gate * act'(z),   dx = dz W,   dW = dz^T x,   db = sum dz,   dgate = sum over a sample's rows of dout * act(z)
//
// All three products are one kernel, C[m][n] = sum over k of X[m,k] Y[n,k], whose operands lie in memory either with the contraction
// along a row ("rows": x and W of the forward, dz of dx) or across the rows ("columns": W of dx, both operands of dW).
//
// Sums are fp32 and what is added, multiplied or activated on the way out is too.  Rounded to 16 bits, besides the results: z where it is kept, and what a
// product takes in that another made, the hidden rows of a feed-forward block, dz, and gate * W.  The matrix instructions of 16-bit operands are 16 times as
// fast as those of 32; each such rounding is off by up to 2^-8 of an element (bf16; fp16 2^-11), as a result's own is.  In fp16 that ends at 2^-14, below which
// half a step is 2^-25: z, hidden rows and dz lie there as a result would, and a scale of the loss moves dz.  Of gate * W it does not, so that is scaled here.

#include "product_device.h"

namespace llsa {
namespace {

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
    int tiles_m, tiles_n, group;          // tiles are taken `group` rows of tiles at a time
    // dx with weights of its own for each sample: rows and rows of tiles of a sample, elements from one sample's weights to the next's.  Else: one sample.
    int rows, tiles_rows;
    int64_t y_sample;
    const bf16* scales;                   // fp16: powers of two that the columns of each sample's weights were divided by, rows s_scales apart, or NULL
    int64_t s_scales;
    // dW: the contraction in pieces, `pieces` of k_piece rows (a multiple of 64) for every k_sample of them.  Else: one piece.
    int64_t k_piece, k_sample;
    int pieces;
    // way out
    const T *bias, *gate, *residual, *slope_at;
    int64_t s_gate, ldr, ldz, ldo;
    T *out, *z;
    int per_sample, act;
    // whether 16-byte accesses are allowed: to bias and gate; to the residual; to out, or its rows are padded with zeros to a multiple of 8 elements (those
    // of z always are)
    int wide, wide_side, wide_out;
    // dW: pieces of the sum, or out and its sums of rows where there is one piece
    T* sums;
    float *part, *part_sum;               // [sample][piece][M][ld_part], [sample][piece][M] or NULL
    int64_t ld_part;
};

struct Place { int m0, m_end, n0, split, tn, sample; };
template <int BM, int BN, typename P>
__device__ __forceinline__ Place place_of_tile(const P& a, int at) {
    const int per_split = a.tiles_m * a.tiles_n, split = at / per_split, tile = at - split * per_split;
    const int in_group = a.group * a.tiles_n, g = tile / in_group, rest = tile - g * in_group;
    const int rows_here = min(a.group, a.tiles_m - g * a.group);
    const int tn = rest / rows_here, tm = g * a.group + rest - tn * rows_here;
    const int sample = tm / a.tiles_rows;
    return {sample * a.rows + (tm - sample * a.tiles_rows) * BM, (sample + 1) * a.rows, tn * BN, split, tn, sample};
}

// What happens on the way out, as far as the kernel is compiled for it: an activation (its LLSA_ACT_ number), the slope of one, or anything, with
// rows and vectors of any alignment.  All forms but the last read and write pieces of 16 bytes.
enum Way { kSlope = 4, kAnything = 8 };

// Where a lane's eight values of one row of C lie in the tensors of the way out.  Uniform parts are kept apart from the lane's (32 bits, the same for
// all rows of its tile), so that one register a tensor addresses them all.
struct Lane { unsigned out, z, residual; };

// Those of a lane's eight columns, and the columns multiplied by them: nothing but in dx of fp16
template <bool YC, typename T>
__device__ __forceinline__ bf16x8 take_scales(const Product<T>& a, int sample, int n, bool inside) {
    bf16x8 up = take8<bf16>(nullptr, true, 8);
    if constexpr (YC && std::is_same_v<T, _Float16>) {
        if (a.scales != nullptr && inside) up = *reinterpret_cast<const bf16x8*>(a.scales + sample * a.s_scales + n);
    }
    return up;
}
template <bool YC, typename T>
__device__ __forceinline__ void put_back(const Product<T>& a, float (&v)[8], const bf16x8& up) {
    if constexpr (YC && std::is_same_v<T, _Float16>) {
        if (a.scales == nullptr) return;
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] *= (float)up[e];
    }
}

// Eight values on their way out: columns n .. n + 7 of row m, `left` of them inside the matrix; row and col are the uniform parts of m and n.  Returns
// what out gets, and in z what the backward wants of it.
template <int WAY, typename T>
__device__ __forceinline__ vec8<T> way_out(const Product<T>& a, float (&v)[8], const vec8<T>& bias, const vec8<T>& gate, const vec8<T>& early, int64_t row, int col,
                                           const Lane& at, int left, vec8<T>& z) {
    constexpr bool any = WAY == kAnything;
    const bool slope = any ? a.slope_at != nullptr : WAY >= kSlope;
    const int act = any ? a.act : WAY & 3;
    if (!slope) {
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] += (float)bias[e];
        if (a.z != nullptr) {
#pragma unroll
            for (int e = 0; e < 8; e++) z[e] = (T)v[e];
        }
    }
    if (any ? act != LLSA_ACT_NONE : (WAY & 3) != 0) {
        if (slope) {
            float at_z[8];
            if (any) load8(at_z, a.slope_at + (row * a.ldz + col) + at.z, true, 8);
#pragma unroll
            for (int e = 0; e < 8; e++) v[e] *= activate_slope(act, any ? at_z[e] : (float)early[e]);
        } else {
#pragma unroll
            for (int e = 0; e < 8; e++) v[e] = activate(act, v[e]);
        }
    }
    if (!slope && a.gate != nullptr) {
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] *= (float)gate[e];
    }
    if (!slope && a.residual != nullptr) {
        float r[8];
        if (any) load8(r, a.residual + (row * a.ldr + col) + at.residual, a.wide_side, left);
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] += any ? r[e] : (float)early[e];
    }
    vec8<T> o;
#pragma unroll
    for (int e = 0; e < 8; e++) o[e] = (T)(e >= left ? 0.f : v[e]);
    return o;
}

// Two stages of LDS and two workgroups a CU that fill each other's waits.  131072 rows of 384 and 1536 channels, us: forward 1536 > 384 with gate and
// residual 194 (0.80 PFLOP/s; 128 x 128 205), dx 1536 > 384 205 (213), dW 196 (0.79; 215); 8192 x 4096 x 4096 229 to 250 by card (1.10 to 1.20; a library's 200), its dW 332.  What
// bounds it is the way of the operands from L2 (11 TB/s with 128 x 128 tiles): without the copies 134, 118, 127 (of 128 x 128) and 189, 198, while half of
// the LDS reads or of the products take off 1 to 9 %.  More stages of 32, three of 64 with 256 x 128, and 256 x 192 tiles, with a third less to fetch, are
// one workgroup a CU or more barriers: dW 280, 270, 226.
template <typename T, bool XC, bool YC, int BM, int BN, int WAVES_M, int WAVES_N, int WAY>
__global__ __launch_bounds__(64 * WAVES_M * WAVES_N, 2) void product_kernel(const Product<T> a) {
    constexpr int kWaves = WAVES_M * WAVES_N, WM = BM / WAVES_M, WN = BN / WAVES_N, MT = WM / 16, NT = WN / 16, kTileX = BM * kStep, kTileY = BN * kStep;
    typedef Operand<T, XC, BM, kWaves> OperandX;
    typedef Operand<T, YC, BN, kWaves> OperandY;
    HIP_DYNAMIC_SHARED(char, shared)
    T* const lds = reinterpret_cast<T*>(shared);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int quad = lane >> 4, wm = (wave % WAVES_M) * WM, wn = (wave / WAVES_M) * WN;

    const Place here = place_of_tile<BM, BN>(a, xcd_order((int)blockIdx.x, (int)gridDim.x));
    const int k_of = here.split / a.pieces;
    const int64_t k_first = (int64_t)(here.split - k_of * a.pieces) * a.k_piece, k0 = k_of * a.k_sample + k_first;
    int64_t k_left = min(a.k_sample - k_first, a.k_piece);
    const int steps = (int)((k_left + kStep - 1) / kStep);
    OperandX ox;
    OperandY oy;
    ox.init(wave, lane, a.ldx, min(BM, (XC ? a.nx : here.m_end) - here.m0));
    oy.init(wave, lane, a.ldy, min(BN, (YC ? a.ny : a.N) - here.n0));
    const T* px = a.x + (XC ? k0 * a.ldx + here.m0 : (int64_t)here.m0 * a.ldx + k0);
    const T* py = a.y + here.sample * a.y_sample + (YC ? k0 * a.ldy + here.n0 : (int64_t)here.n0 * a.ldy + k0);
    const int64_t stepx = XC ? kStep * a.ldx : kStep, stepy = YC ? kStep * a.ldy : kStep;
    auto request = [&](int buffer) {
        T* const t = lds + buffer * (kTileX + kTileY);
        const int left = (int)min(k_left, (int64_t)kStep);
        ox.request(px, t, wave, lane, left);
        oy.request(py, t + kTileX, wave, lane, left);
        px += stepx;
        py += stepy;
        k_left -= kStep;
    };

    const bool sums = XC && (a.part_sum != nullptr || a.sums != nullptr) && here.tn == 0 && wn == 0;
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
    auto multiply = [&](int buffer) {
        const T* const tx = lds + buffer * (kTileX + kTileY);
        const T* const ty = tx + kTileX;
#pragma unroll
        for (int ks = 0; ks < kStep / 32; ks++) {
            vec8<T> fx[MT], fy[NT];
#pragma unroll
            for (int j = 0; j < MT; j++) fx[j] = OperandX::fragment(tx, wm + 16 * j, ks, lane);
#pragma unroll
            for (int i = 0; i < NT; i++) fy[i] = OperandY::fragment(ty, wn + 16 * i, ks, lane);
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
    };

    // Lane l holds rows n of four: columns 4 (l/16) .. +3 of every 16, of row l%16 of C.  Swapped between sixteens of lanes, a pair of tiles gives it
    // eight neighbouring ones, so that everything on the way out is read and written in pieces of 16 bytes.
    const int lane_row = lane & 15, lane_col = 16 * (quad & 1) + 8 * (quad >> 1);
    const int row0 = here.m0 + wm, col0 = here.n0 + wn, rows_left = here.m_end - row0 - lane_row, cols_left = a.N - col0 - lane_col;
    const Lane at = {(unsigned)(lane_row * a.ldo) + lane_col, (unsigned)(lane_row * a.ldz) + lane_col, (unsigned)(lane_row * a.ldr) + lane_col};
    const T* const side = WAY == kAnything || XC || (YC && WAY < kSlope) ? nullptr : WAY >= kSlope ? a.slope_at : a.residual;
    constexpr int kPair = NT % 4 == 0 && !XC ? 2 : 1;     // pieces of 32 columns that leave together
    const bool whole = kPair == 2 && here.m0 + BM <= here.m_end && here.n0 + BN <= a.N && (WAY != kAnything || a.wide_out);
    vec8<T> early[kPair][MT];                             // what is read on the way out
    auto read_side = [&](int p0) {
        if (side == nullptr) return;
        const int64_t ld = WAY >= kSlope ? a.ldz : a.ldr;
        const unsigned lane_at = WAY >= kSlope ? at.z : at.residual;
        if constexpr (kPair == 2) {
            if (whole) {
#pragma unroll
                for (int j = 0; j < MT; j++)
                    request_lines(early[0][j], early[1][j], side + ((row0 + 16 * j) * ld + (col0 + 32 * p0)), lane_at, (unsigned)(8 * ld), lane);
                return;
            }
        }
#pragma unroll
        for (int j = 0; j < MT; j++)
#pragma unroll
            for (int h = 0; h < kPair; h++) {
                const int p = p0 + h;
                if (16 * j < rows_left && 32 * p < cols_left) early[h][j] = *reinterpret_cast<const vec8<T>*>(side + ((row0 + 16 * j) * ld + (col0 + 32 * p)) + lane_at);
            }
    };

    request(0);
    for (int s = 0; s + 1 < steps; s++) {
        wait_vm0();
        __syncthreads();                                      // everyone's copies of this step are there, and everyone is done with the other buffer
        request((s + 1) & 1);
        multiply(s & 1);
    }
    wait_vm0();
    __syncthreads();
    read_side(0);                                             // (on its way during the last step's products)
    multiply((steps - 1) & 1);

    const bool gated = !XC && !YC && a.gate != nullptr;
    const int sample = gated ? here.m0 / a.per_sample : 0;
    const bool one_sample = gated && min(here.m0 + BM, here.m_end) <= (int64_t)(sample + 1) * a.per_sample;
#pragma unroll
    for (int p0 = 0; p0 < NT / 2; p0 += kPair) {
        constexpr int kPairs = kPair;
        vec8<T> bias[kPair], gate[kPair];
        bf16x8 up[kPair];
#pragma unroll
        for (int h = 0; h < kPairs; h++) {
            const int n = col0 + lane_col + 32 * (p0 + h), left = cols_left - 32 * (p0 + h);
            bias[h] = take8(!XC && a.bias != nullptr && left > 0 ? a.bias + n : nullptr, a.wide, left);
            gate[h] = take8(one_sample && left > 0 ? a.gate + sample * a.s_gate + n : nullptr, a.wide, left);
            up[h] = take_scales<!XC && YC>(a, here.sample, n, left > 0);
        }
#pragma unroll
        for (int j = 0; j < MT; j++) {
            const int64_t row = row0 + 16 * j;
            vec8<T> o[kPair], z[kPair];
            if constexpr (kPair == 2) {
                if (side != nullptr && whole) arrange_lines<T>(early[0][j], early[1][j], lane);
            }
#pragma unroll
            for (int h = 0; h < kPairs; h++) {
                const int p = p0 + h, col = col0 + 32 * p, left = cols_left - 32 * p;
                float v[8];
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const u32x2 w = __builtin_amdgcn_permlane16_swap(__float_as_uint(acc[2 * p][j][e]), __float_as_uint(acc[2 * p + 1][j][e]), false, false);
                    v[e] = __uint_as_float(w[0]);
                    v[4 + e] = __uint_as_float(w[1]);
                }
                const bool inside = 16 * j < rows_left && left > 0;
                if constexpr (XC) {
                    if (!inside) continue;
                    if (a.part == nullptr) {                  // (the whole sum)
                        store8(a.out + (row * a.ldo + col) + at.out, v, a.wide_out, left);
                        continue;
                    }
                    float* const o = a.part + (((int64_t)here.split * a.M + row) * a.ld_part + col) + at.out;
                    *reinterpret_cast<f32x4*>(o) = f32x4{v[0], v[1], v[2], v[3]};
                    *reinterpret_cast<f32x4*>(o + 4) = f32x4{v[4], v[5], v[6], v[7]};
                } else {
                    if (inside) {
                        put_back<YC>(a, v, up[h]);
                        if (gated && !one_sample) gate[h] = take8(a.gate + (int)(row + lane_row) / a.per_sample * a.s_gate + col + lane_col, a.wide, left);
                        o[h] = way_out<WAY>(a, v, bias[h], gate[h], early[h][j], row, col, at, left, z[h]);
                    }
                    if (whole || !inside) continue;
                    if (!YC && a.z != nullptr) *reinterpret_cast<vec8<T>*>(a.z + (row * a.ldz + col) + at.z) = z[h];
                    T* const to = a.out + (row * a.ldo + col) + at.out;
                    if (WAY != kAnything || a.wide_out) {
                        *reinterpret_cast<vec8<T>*>(to) = o[h];
                    } else {
#pragma unroll
                        for (int e = 0; e < 8; e++)
                            if (e < left) to[e] = o[h][e];
                    }
                }
            }
            if constexpr (!XC && kPair == 2) {
                if (whole) {
                    if (!YC && a.z != nullptr) store_lines(a.z + (row * a.ldz + (col0 + 32 * p0)), at.z, (unsigned)(8 * a.ldz), z[0], z[1], lane);
                    store_lines(a.out + (row * a.ldo + (col0 + 32 * p0)), at.out, (unsigned)(8 * a.ldo), o[0], o[1], lane);
                }
            }
            __builtin_amdgcn_sched_barrier(0);            // (rows one after another: all at once do not fit the registers)
        }
        if (p0 + kPair < NT / 2) read_side(p0 + kPair);
    }
    if constexpr (XC) {
        if (sums && quad == 0) {
#pragma unroll
            for (int j = 0; j < MT; j++) {
                const int m = here.m0 + wm + 16 * j + lane;
                if (m >= here.m_end) continue;
                if (a.sums != nullptr) a.sums[m] = (T)sum[j][0];
                else a.part_sum[(int64_t)here.split * a.M + m] = sum[j][0];
            }
        }
    }
}

// ---------------------------------------------------------------------------------------
// Few rows: single tokens, one vector for each image, a small image.  A workgroup takes 32 columns of up to 64 rows of C, its eight waves an eighth of the
// contraction each, through two stages of LDS of their own that nobody else waits for; the sums meet at the end.  Where a row of tiles is all there is the
// weight is read once, and there is little else.  us, tiles of 64 x 64 / this: 8 rows of 4096 > 4096 29.7 / 7.1 (33 MB of weights: 4.8 TB/s), its dx 40.5 /
// 13.9; and with up to a workgroup for each CU: 512, 1024 > 1024 (256 workgroups) 10.4 / 7.5, 1024, 1536 > 384 (192) 13.5 / 9.5, 256, 2048 > 2048 (256) 16.8 /
// 11.6;  beyond: 1024, 1024 > 1024 (512) 10.5 / 12.7, 256, 4096 > 4096 (512) 31 / 36.7, 512, 384 > 1536 (384) 5.9 / 7.3.
// ---------------------------------------------------------------------------------------
constexpr int kFewWaves = 8, kFewColumns = 32, kFewStage = kFewColumns * kStep, kFewRows = 64;
template <typename T, bool YC, int MT, int WAY>
__global__ __launch_bounds__(64 * kFewWaves, 2) void few_rows_kernel(const Product<T> a) {
    typedef Operand<T, YC, kFewColumns, 1> OperandY;
    HIP_DYNAMIC_SHARED(char, shared)
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), quad = lane >> 4;
    T* const stage = reinterpret_cast<T*>(shared) + wave * 2 * kFewStage;
    const int n0 = (int)blockIdx.x * kFewColumns, row0 = (int)blockIdx.y * 16 * MT;
    const int all = (int)((a.K + kStep - 1) / kStep), each = (all + kFewWaves - 1) / kFewWaves, first = min(all, wave * each), steps = min(all - first, each);

    OperandY oy;
    oy.init(0, lane, a.ldy, min(kFewColumns, (YC ? a.ny : a.N) - n0));
    const int k0 = first * kStep, K = (int)a.K;
    const T* py = a.y + (YC ? k0 * a.ldy + n0 : n0 * a.ldy + k0);
    const T* px[MT];
#pragma unroll
    for (int j = 0; j < MT; j++) px[j] = a.x + min(row0 + 16 * j + (lane & 15), a.M - 1) * a.ldx;
    f32x4 acc[2][MT];
#pragma unroll
    for (int i = 0; i < 2; i++)
#pragma unroll
        for (int j = 0; j < MT; j++) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    vec8<T> next[MT][2];
    auto request = [&](int s) {
        const int k = k0 + s * kStep;
        oy.request(py + (YC ? s * kStep * a.ldy : s * kStep), stage + (s & 1) * kFewStage, 0, lane, K - k);
#pragma unroll
        for (int j = 0; j < MT; j++)
#pragma unroll
            for (int ks = 0; ks < 2; ks++) {
                const int at = k + 32 * ks + 8 * quad;
                next[j][ks] = *reinterpret_cast<const vec8<T>*>(at < K ? px[j] + at : reinterpret_cast<const T*>(kZeros));
            }
    };
    if (steps > 0) request(0);
    for (int s = 0; s < steps; s++) {
        vec8<T> fx[MT][2];
        wave_waits_for_copies();
#pragma unroll
        for (int j = 0; j < MT; j++)
#pragma unroll
            for (int ks = 0; ks < 2; ks++) fx[j][ks] = next[j][ks];
        if (s + 1 < steps) request(s + 1);
        const T* const ty = stage + (s & 1) * kFewStage;
#pragma unroll
        for (int ks = 0; ks < 2; ks++)
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const vec8<T> fy = OperandY::fragment(ty, 16 * i, ks, lane);
#pragma unroll
                for (int j = 0; j < MT; j++) acc[i][j] = product16(fy, fx[j][ks], acc[i][j]);
            }
        wave_waits_for_reads();                               // (done, before the next request but one writes there)
    }

    // wave j adds up tile j of rows, in the order of the waves
    __syncthreads();
    f32x4* const sums = reinterpret_cast<f32x4*>(shared);     // [wave][tile][half][lane]
#pragma unroll
    for (int j = 0; j < MT; j++)
#pragma unroll
        for (int i = 0; i < 2; i++) sums[((wave * MT + j) * 2 + i) * 64 + lane] = acc[i][j];
    __syncthreads();
    if (wave >= MT) return;
    f32x4 t[2];
#pragma unroll
    for (int i = 0; i < 2; i++) {
        t[i] = sums[(wave * 2 + i) * 64 + lane];
#pragma unroll
        for (int w = 1; w < kFewWaves; w++) t[i] += sums[((w * MT + wave) * 2 + i) * 64 + lane];
    }
    float v[8];
#pragma unroll
    for (int e = 0; e < 4; e++) {
        const u32x2 w = __builtin_amdgcn_permlane16_swap(__float_as_uint(t[0][e]), __float_as_uint(t[1][e]), false, false);
        v[e] = __uint_as_float(w[0]);
        v[4 + e] = __uint_as_float(w[1]);
    }
    const int lane_col = 16 * (quad & 1) + 8 * (quad >> 1), lane_row = lane & 15, row = row0 + 16 * wave, left = a.N - n0 - lane_col, m = row + lane_row;
    if (m >= a.M || left <= 0) return;
    const Lane at = {(unsigned)(lane_row * a.ldo) + lane_col, (unsigned)(lane_row * a.ldz) + lane_col, (unsigned)(lane_row * a.ldr) + lane_col};
    const T* const side = WAY == kAnything || (YC && WAY < kSlope) ? nullptr : WAY >= kSlope ? a.slope_at : a.residual;
    vec8<T> early = take8<T>(nullptr, true, 0), z;
    if (side != nullptr) early = *reinterpret_cast<const vec8<T>*>(side + ((int64_t)row * (WAY >= kSlope ? a.ldz : a.ldr) + n0) + (WAY >= kSlope ? at.z : at.residual));
    const vec8<T> bias = take8(!YC && a.bias != nullptr ? a.bias + n0 + lane_col : nullptr, a.wide, left);
    const vec8<T> gate = take8(!YC && a.gate != nullptr ? a.gate + m / a.per_sample * a.s_gate + n0 + lane_col : nullptr, a.wide, left);
    const vec8<T> o = way_out<WAY>(a, v, bias, gate, early, row, n0, at, left, z);
    if (!YC && a.z != nullptr) *reinterpret_cast<vec8<T>*>(a.z + ((int64_t)row * a.ldz + n0) + at.z) = z;
    T* const to = a.out + ((int64_t)row * a.ldo + n0) + at.out;
    if (WAY != kAnything || a.wide_out) {
        *reinterpret_cast<vec8<T>*>(to) = o;
    } else {
#pragma unroll
        for (int e = 0; e < 8; e++)
            if (e < left) to[e] = o[e];
    }
}

// ---------------------------------------------------------------------------------------
// Many rows, a short contraction: the weights stay in registers.  A workgroup of twelve waves keeps 384 columns' weights, 32 columns a wave, and takes its
// rows of x through LDS, 32 at a time and two such tiles ahead: a row is read once for 384 columns of C, and no weight a second time.  131072 rows, us of the
// tiles / this: 384 > 1536 with GELU and z kept 325 / 252, without 228 / 165 (0.94 PFLOP/s; without its stores 155), dx 384 > 1536 242 / 162, with act'(z) 329 /
// 248 (3.7 TB/s), 384 > 384 with gate and residual 85 / 72 (4.2 TB/s).  What is left is the multiplication itself (96 registers of weights leave three waves a
// SIMD and no fragments read ahead).  Eight waves of 48 columns, taking turns on a SIMD with C through LDS as whole rows, measured the same: 240, 164, 176, 283, 74.
// ---------------------------------------------------------------------------------------
constexpr int kResWaves = 12, kResColumns = 32 * kResWaves, kResRows = 32, kResStages = 3, kResOwn = 32 * kStep + 64;
struct Resident { int blocks, slots, tiles, per_sample; };   // blocks of columns, workgroups for each, tiles of rows in all and of a sample
template <typename T, bool YC, int WAY, int STEPS>
__global__ __launch_bounds__(64 * kResWaves) void resident_kernel(const Product<T> a, const Resident q) {
    typedef Operand<T, false, kResRows, 1> OperandX;          // of a step: 4 copies
    typedef Operand<T, YC, 32, 1> OperandY;
    constexpr int kStage = kResRows * kStep * STEPS;
    static_assert(4 * STEPS <= 2 * kResWaves, "two copies of a wave take in a tile");
    HIP_DYNAMIC_SHARED(char, shared)
    T* const lds = reinterpret_cast<T*>(shared);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), quad = lane >> 4;
    // workgroups of an XCD: the blocks of columns of the same rows side by side
    const int xcd = blockIdx.x & 7, local = blockIdx.x >> 3, block = local % q.blocks, slot = (local / q.blocks) * 8 + xcd;
    if (slot >= q.slots) return;
    const int t0 = (int)((int64_t)q.tiles * slot / q.slots), t1 = (int)((int64_t)q.tiles * (slot + 1) / q.slots);
    if (t0 >= t1) return;
    const int n0 = block * kResColumns + 32 * wave;
    const bool columns = n0 < a.N;                            // (a wave beyond the last column copies, and does no more)
    const int lane_col = 16 * (quad & 1) + 8 * (quad >> 1), lane_row = lane & 15;
    // LDS of the wave's own: its weights on their way, 64 of the contraction at a time; bias and gate of its columns, 32 of either
    T* const own = lds + kResStages * kStage + wave * kResOwn;
    T* const vectors = own + 32 * kStep;

    vec8<T> fy[2 * STEPS][2];
    auto weights = [&](const T* w) {
        OperandY oy;
        oy.init(0, lane, a.ldy, 32);
#pragma unroll
        for (int s = 0; s < STEPS; s++) {
            oy.request(w + (YC ? s * kStep * a.ldy + n0 : n0 * a.ldy + s * kStep), own, 0, lane, kStep);
            wave_waits_for_copies();
#pragma unroll
            for (int ks = 0; ks < 2; ks++)
#pragma unroll
                for (int i = 0; i < 2; i++) fy[2 * s + ks][i] = OperandY::fragment(own, 16 * i, ks, lane);
            wave_waits_for_reads();
        }
    };

    unsigned off[2];                                          // of this wave's two copies of a tile
#pragma unroll
    for (int c = 0; c < 2; c++) {
        const int i = 2 * wave + c, r = OperandX::row_of(i & 3, lane);
        off[c] = (unsigned)(r * a.ldx) + (i >> 2) * kStep + OperandX::place_of(i & 3, r, lane);
    }
    // The last rows of a sample are a whole tile as well: it takes in rows of the one before, and stores the same values a second time.
    auto row_of_tile = [&](int t, int sample) { return sample * a.rows + min((t - sample * q.per_sample) * kResRows, a.rows - kResRows); };
    auto request = [&](int t) {
        if (t >= t1 || wave >= 2 * STEPS) return;
        T* const stage = lds + (t % kResStages) * kStage;
        const T* const base = a.x + row_of_tile(t, t / q.per_sample) * a.ldx;
#pragma unroll
        for (int c = 0; c < 2; c++) copy_to_lds(base + off[c], stage + (2 * wave + c) * 512);
    };
    request(t0);
    request(t0 + 1);
    const Lane at = {(unsigned)(lane_row * a.ldo) + lane_col, (unsigned)(lane_row * a.ldz) + lane_col, (unsigned)(lane_row * a.ldr) + lane_col};
    const T* const side = YC && WAY < kSlope ? nullptr : WAY >= kSlope ? a.slope_at : a.residual;
    if (!YC && columns) {
        if (lane_row == 0) *reinterpret_cast<vec8<T>*>(vectors + lane_col) = take8(a.bias != nullptr ? a.bias + n0 + lane_col : nullptr, true, 8);
        weights(a.y);
    }
    wait_vm0();
    for (int t = t0, have = -1; t < t1; t++) {
        const int sample = t / q.per_sample, m0 = row_of_tile(t, sample);
        if (sample != have && columns) {
            if (YC && (have < 0 || a.y_sample != 0)) weights(a.y + sample * a.y_sample);
            if constexpr (YC && std::is_same_v<T, _Float16>) {
                if (lane_row == 0) *reinterpret_cast<bf16x8*>(vectors + lane_col) = take_scales<YC>(a, sample, n0 + lane_col, true);
            }
            if (!YC && a.gate != nullptr && lane_row == 0) *reinterpret_cast<vec8<T>*>(vectors + 32 + lane_col) = *reinterpret_cast<const vec8<T>*>(a.gate + sample * a.s_gate + n0 + lane_col);
        }
        have = sample;
        // this tile is there (every wave has waited for its copies before its last stores), and the one before it is read
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_waitcnt(0xC07F);
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        request(t + 2);
        if (!columns) {
            wait_vm0();
            continue;
        }
        vec8<T> early[2];                                     // what is read on the way out
        if (side != nullptr) {
#pragma unroll
            for (int j = 0; j < 2; j++)
                early[j] = __builtin_nontemporal_load(
                    reinterpret_cast<const vec8<T>*>(side + ((int64_t)(m0 + 16 * j) * (WAY >= kSlope ? a.ldz : a.ldr) + n0) + (WAY >= kSlope ? at.z : at.residual)));
        }
        f32x4 acc[2][2];
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
            for (int j = 0; j < 2; j++) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
        const T* const tx = lds + (t % kResStages) * kStage;
#pragma unroll
        for (int ks = 0; ks < 2 * STEPS; ks++) {
            vec8<T> fx[2];
#pragma unroll
            for (int j = 0; j < 2; j++) fx[j] = OperandX::fragment(tx + (ks >> 1) * (kResRows * kStep), 16 * j, ks & 1, lane);
#pragma unroll
            for (int i = 0; i < 2; i++)
#pragma unroll
                for (int j = 0; j < 2; j++) acc[i][j] = product16(fy[ks][i], fx[j], acc[i][j]);
        }
        wait_vm0();
#pragma unroll
        for (int j = 0; j < 2; j++) {
            __builtin_amdgcn_sched_barrier(0);                // (the weights leave no registers for both at once, nor for bias and gate but here)
            vec8<T> bias = take8<T>(nullptr, true, 8), gate = bias, z;
            if (!YC) {
                bias = *reinterpret_cast<const vec8<T>*>(vectors + lane_col);
                gate = *reinterpret_cast<const vec8<T>*>(vectors + 32 + lane_col);
            }
            float v[8];
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const u32x2 w = __builtin_amdgcn_permlane16_swap(__float_as_uint(acc[0][j][e]), __float_as_uint(acc[1][j][e]), false, false);
                v[e] = __uint_as_float(w[0]);
                v[4 + e] = __uint_as_float(w[1]);
            }
            if constexpr (YC) put_back<YC>(a, v, *reinterpret_cast<const bf16x8*>(vectors + lane_col));
            const int64_t row = m0 + 16 * j;
            const vec8<T> o = way_out<WAY>(a, v, bias, gate, early[j], row, n0, at, 8, z);
            if (!YC && a.z != nullptr) *reinterpret_cast<vec8<T>*>(a.z + (row * a.ldz + n0) + at.z) = z;
            *reinterpret_cast<vec8<T>*>(a.out + (row * a.ldo + n0) + at.out) = o;
        }
    }
}

// The pieces of dW and db added up.  Each of a workgroup's four waves takes every fourth piece, of the same 64 places: 56 pieces of 384 x 384 (33 MB) are seven
// loads deep then, not 28.
template <typename T>
__global__ __launch_bounds__(256) void product_join_kernel(const float* part, const float* part_sum, T* out, int64_t ldo, T* sums, int64_t M, int N, int64_t ld_part,
                                                           int splits) {
    __shared__ f32x4 rest[3][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t n4 = ld_part / 4, i = (int64_t)blockIdx.x * 64 + lane, m = i < M * n4 ? i / n4 : i - M * n4;
    const int n = (int)(i - m * n4) * 4;
    const bool sum = i >= M * n4;                             // of dz's rows
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    if (!sum) {
#pragma unroll 8
        for (int s = wave; s < splits; s += 4) v += *reinterpret_cast<const f32x4*>(part + ((int64_t)s * M + m) * ld_part + n);
    } else if (part_sum != nullptr && m < M) {
        for (int s = wave; s < splits; s += 4) v[0] += part_sum[(int64_t)s * M + m];
    }
    if (wave > 0) rest[wave - 1][lane] = v;
    __syncthreads();
    if (wave > 0) return;
#pragma unroll
    for (int r = 0; r < 3; r++) v += rest[r][lane];
    if (!sum) {
#pragma unroll
        for (int e = 0; e < 4; e++)
            if (n + e < N) out[m * ldo + n + e] = (T)v[e];
    } else if (part_sum != nullptr && m < M) {
        sums[m] = (T)v[0];
    }
}

// The same for a layer whose gate was left out of the products: G_b = dout^T x of sample b, S_b = sum of its rows of dout, in pieces.
//     dW = sum over b of gate_b G_b,   db = sum of gate_b S_b,   dgate_b = sum over k of W G_b + bias S_b
// (the last is sum over the rows of dout (x W^T + bias), without those rows).  A workgroup takes a row of G, in eight waves for every eighth sample of 256
// columns and eight more for those of the next 256: that many loads are under way at a time (40 pieces of 384 x 1536, 94 MB: 32 us, 2.9 TB/s; four waves 40).
struct GatedJoin {
    const float *part, *part_sum;
    const void *gate, *w, *bias;
    void *out, *sums, *dgate;
    int64_t ld_part, s_gate, ldw, ldo;
    int M, N, samples, pieces;
};
constexpr int kJoinSamples = 8, kJoinGroups = 2, kJoinThreads = 64 * kJoinSamples * kJoinGroups;
template <typename T>
__global__ __launch_bounds__(kJoinThreads) void gated_join_kernel(const GatedJoin a) {
    constexpr int kColumns = 256;                             // of a wave at a time
    __shared__ f32x4 rows[kJoinGroups][kJoinSamples][64];
    HIP_DYNAMIC_SHARED(float, dots)                           // [group][sample]
    const int m = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6, group = wave / kJoinSamples, of = wave % kJoinSamples;
    const T* const gate = static_cast<const T*>(a.gate) + m;
    const T* const w = static_cast<const T*>(a.w);
    if (a.dgate != nullptr)
        for (int b = threadIdx.x; b < kJoinGroups * a.samples; b += kJoinThreads) dots[b] = 0.f;
    for (int first = 0; first < a.N; first += kJoinGroups * kColumns) {
        const int n = first + group * kColumns + lane * 4;
        f32x4 v = {0.f, 0.f, 0.f, 0.f}, wn = {0.f, 0.f, 0.f, 0.f};
        if (a.dgate != nullptr)
#pragma unroll
            for (int e = 0; e < 4; e++) wn[e] = n + e < a.N ? (float)w[m * a.ldw + n + e] : 0.f;
        __syncthreads();                                      // (dots are cleared, and the rows of the columns before are read)
        for (int b = of; b < a.samples; b += kJoinSamples) {
            f32x4 g = {0.f, 0.f, 0.f, 0.f};
            if (n < a.N) {
                const float* part = a.part + ((int64_t)b * a.pieces * a.M + m) * a.ld_part + n;
#pragma unroll 8
                for (int p = 0; p < a.pieces; p++) g += *reinterpret_cast<const f32x4*>(part + (int64_t)p * a.M * a.ld_part);
            }
            v += (float)gate[b * a.s_gate] * g;
            if (a.dgate != nullptr) {
                float d = 0.f;
#pragma unroll
                for (int e = 0; e < 4; e++) d += n + e < a.N ? g[e] * wn[e] : 0.f;
                d = octet_sum(d);
                d += across<8>(d);
                d = quad_sum(d);
                if (lane == 0) dots[group * a.samples + b] += d;      // (a sample is one wave's of each group)
            }
        }
        rows[group][of][lane] = v;
        __syncthreads();
        if (of == 0 && a.out != nullptr) {
#pragma unroll
            for (int r = 1; r < kJoinSamples; r++) v += rows[group][r][lane];
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (n + e < a.N) static_cast<T*>(a.out)[m * a.ldo + n + e] = (T)v[e];
        }
    }
    __syncthreads();
    if (wave > 0) return;
    float sum = 0.f;
    const float bias = a.bias != nullptr ? (float)static_cast<const T*>(a.bias)[m] : 0.f;
    for (int b = lane; b < a.samples; b += 64) {
        float s = 0.f;
        if (a.part_sum != nullptr)
            for (int p = 0; p < a.pieces; p++) s += a.part_sum[(int64_t)(b * a.pieces + p) * a.M + m];
        sum += (float)gate[b * a.s_gate] * s;
        if (a.dgate != nullptr) {
            const float d = dots[b] + dots[a.samples + b] + bias * s;
            static_cast<T*>(a.dgate)[(int64_t)b * a.M + m] = (T)d;
        }
    }
    if (a.sums != nullptr) {
        sum = quad_sum(octet_sum(sum));
        sum += across<8>(sum);
        if (lane == 0) static_cast<T*>(a.sums)[m] = (T)sum;
    }
}

// The weights of every sample with its gate: gate_b[n] W[n][k] (8 samples of 384 x 1536: 5.7 us).  Rounded to 16 bits, as dout * gate would be: the products
// take operands of that size.  bf16 has fp32's range for it.
__global__ __launch_bounds__(256) void gate_rows_kernel(const bf16* w, int64_t ldw, const bf16* gate, int64_t s_gate, bf16* out, int64_t ldo, int N, int64_t pieces) {
    const int64_t per = ldo / 8, i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= pieces) return;
    const int64_t r = i / per, b = r / N;
    const int n = (int)(r - b * N), c = (int)(i - r * per) * 8;
    const float g = (float)gate[b * s_gate + n];
    bf16x8 v = *reinterpret_cast<const bf16x8*>(w + n * ldw + c);
#pragma unroll
    for (int e = 0; e < 8; e++) v[e] = (bf16)((float)v[e] * g);
    *reinterpret_cast<bf16x8*>(out + r * ldo + c) = v;
}
// fp16 has not: the gates of an adaLN-zero block begin at zero, and a product below 2^-14 loses its bits.  Every column of a sample is divided by a power of two
// that brings the largest of its products to 2^14 .. 2^15, and dx is multiplied by it in fp32.  What is 2^-28 and less of that largest one is rounded by up to
// 2^-39 of it, far below the 2^-24 that a sum in fp32 is off by.  A workgroup takes 32 columns of a sample, 256 rows at a time, and reads them twice, the second time
// out of L2.  Bound by the latency of those reads: 8 samples of 384 x 1536 12.2 us, of 384 x 384 7.2 (256 threads with 64 columns, 32 rows at a time: 20).
// The multiplication takes 3 to 11 us of dx (131072 rows 384 > 1536 behind act' 257 -> 268).
constexpr int kScaleColumns = 32, kScaleThreads = 1024, kScaleRows = kScaleThreads * 8 / kScaleColumns;
__global__ __launch_bounds__(kScaleThreads) void gate_rows_scaled_kernel(const _Float16* w, int64_t ldw, const _Float16* gate, int64_t s_gate, _Float16* out, int64_t ldo, bf16* scales,
                                                               int N, int groups) {
    constexpr int kLanes = kScaleColumns / 8, kWaves = kScaleThreads / 64;      // lanes of a row
    __shared__ float most[kWaves][kScaleColumns];
    const int64_t b = (int)blockIdx.x / groups;
    const int group = (int)blockIdx.x - (int)b * groups, lane = threadIdx.x % kLanes, row = threadIdx.x / kLanes, c = group * kScaleColumns + lane * 8;
    const bool inside = c < ldo;                              // (whole pieces of eight)
    auto products = [&](int n, float (&v)[8]) {
        const float g = (float)gate[b * s_gate + n];
        const f16x8 a = *reinterpret_cast<const f16x8*>(w + n * ldw + c);
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = (float)a[e] * g;   // (exact)
    };
    float top[8], v[8];
#pragma unroll
    for (int e = 0; e < 8; e++) top[e] = 0.f;
    if (inside)
        for (int n = row; n < N; n += kScaleRows) {
            products(n, v);
#pragma unroll
            for (int e = 0; e < 8; e++) top[e] = fmaxf(top[e], fabsf(v[e]));       // (of a NaN and a number the number)
        }
#pragma unroll
    for (int e = 0; e < 8; e++) {
#pragma unroll
        for (int step = kLanes; step < 64; step *= 2) top[e] = fmaxf(top[e], __shfl_xor(top[e], step));
        if ((threadIdx.x & 63) < kLanes) most[threadIdx.x >> 6][lane * 8 + e] = top[e];
    }
    __syncthreads();
    if (!inside) return;
    float down[8];
    bf16x8 up;
#pragma unroll
    for (int e = 0; e < 8; e++) {
        float m = 0.f;
#pragma unroll
        for (int wave = 0; wave < kWaves; wave++) m = fmaxf(m, most[wave][lane * 8 + e]);
        // the exponent of m, which is 0 or in 2^-48 .. 2^32, or an infinity
        const int exponent = (int)(__float_as_uint(m) >> 23), k = m == 0.f || exponent == 255 ? 0 : exponent - 127 - 14;
        down[e] = __uint_as_float((unsigned)(127 - k) << 23);
        up[e] = (bf16)__uint_as_float((unsigned)(127 + k) << 23);
    }
    if (row == 0) *reinterpret_cast<bf16x8*>(scales + b * ldo + c) = up;
    for (int n = row; n < N; n += kScaleRows) {
        products(n, v);
        f16x8 o;
#pragma unroll
        for (int e = 0; e < 8; e++) o[e] = (_Float16)(v[e] * down[e]);
        *reinterpret_cast<f16x8*>(out + (b * N + n) * ldo + c) = o;
    }
}

// ---------------------------------------------------------------------------------------
// dz = dout * gate * act'(z), and pieces of dgate = sum over a sample's rows of dout * act(z).  A workgroup takes 128 columns of up to `rows` rows
// of one sample: 16 threads along a row, 16 rows at a time.  Bound by memory: it reads dout and z and writes dz once, and nothing here is reused.
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

// Rows of an odd length or at odd addresses, copied to rows that the products can read: 16-byte aligned, padded with zeros.  Several matrices a launch.
struct Pads {
    llsa_pad_job job[LLSA_PAD_JOBS];
    int64_t end[LLSA_PAD_JOBS];           // pieces of eight, of this and the jobs before it
};
__global__ __launch_bounds__(256) void pad_kernel(const Pads a) {
    int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    int k = 0;
    while (k < LLSA_PAD_JOBS && i >= a.end[k]) k++;
    if (k == LLSA_PAD_JOBS) return;
    if (k > 0) i -= a.end[k - 1];
    const llsa_pad_job q = a.job[k];
    const int64_t per = q.ldy / 8, r = i / per;
    const int c = (int)(i - r * per) * 8;
    const uint16_t* const x = static_cast<const uint16_t*>(q.x) + r * q.ldx;
    typedef __attribute__((ext_vector_type(8))) uint16_t u16x8;
    u16x8 v;
#pragma unroll
    for (int e = 0; e < 8; e++) {
        const uint16_t t = x[min(c + e, q.cols - 1)];
        v[e] = c + e < q.cols ? t : (uint16_t)0;
    }
    *reinterpret_cast<u16x8*>(static_cast<uint16_t*>(q.y) + r * q.ldy + c) = v;
}

// ---------------------------------------------------------------------------------------
// launches
// ---------------------------------------------------------------------------------------
template <typename T, bool XC, bool YC, int BM, int BN, int WAVES_M, int WAVES_N, int WAY>
int launch_tiles(Product<T>& a, int splits, hipStream_t stream) {
    a.tiles_rows = (int)ceil_div(a.rows, BM);
    const int64_t tm = (int64_t)(a.M / a.rows) * a.tiles_rows, tn = ceil_div(a.N, BN);
    if (tm * tn * splits > kMaxGrid) return fail(-1, "linear: too many rows");
    a.tiles_m = (int)tm;
    a.tiles_n = (int)tn;
    constexpr int lds = 2 * (BM + BN) * kStep * (int)sizeof(T);
    auto kernel = product_kernel<T, XC, YC, BM, BN, WAVES_M, WAVES_N, WAY>;
    if (lds > 64 * 1024) {
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, lds);
        if (e != hipSuccess) return fail(-101, "linear: %s", hipGetErrorString(e));
    }
    hipLaunchKernelGGL(kernel, dim3((unsigned)(tm * tn * splits)), dim3(64 * WAVES_M * WAVES_N), lds, stream, a);
    return 0;
}
// Which tiles.  Measured (us, forward of M rows, K channels in, N out), 64 x 64 / 128 x 128 / 192 x 128 / 256 x 256:
//     2048, 1024 > 1024    9.6 / 14.6 / 18.7 / 31       131072, 1536 > 384     - / 208 / 197 / 259
//     4096, 1024 > 1024     15 / 15.2 / 19.1 / 32        65536, 1024 > 1024    - / 188 / 177 / 189
//     8192, 1024 > 1024     27 / 24.0 / 30.9 / 40        16384, 768 > 768      - / 34 / 41 / 36
//     8192, 2048 > 2048     98 / 77 / 85 / 75             8192, 4096 > 4096    - / 260 / 260 / 226
// Small tiles keep a grid of few tiles busy, up to four for each CU.  Beyond that it is rounds times the length of one: two workgroups of 128 x 128 or
// 192 x 128 fit a CU, one of 256 x 256, and a round of these takes 1, 1.3 and 1.8 + 220 / K forward (the shorter the contraction, the more weighs a way out with
// gate and residual that no second workgroup fills), 1, 1.38 and 1.8 in dx.
enum Tiles { k64, k128, k192, k256 };
Tiles tiles_for(int64_t M, int64_t N, int64_t K, bool dx) {
    if (ceil_div(M, 64) * ceil_div(N, 64) <= 4 * kCus) return k64;
    const auto rounds = [&](int bm, int bn, int slots) {      // (many rounds run into one another: only the last one is not full)
        const double n = (double)(ceil_div(M, bm) * ceil_div(N, bn)) / slots;
        return n > 4 ? n + 0.5 : std::ceil(n);
    };
    const double t128 = rounds(128, 128, 2 * kCus), t192 = (dx ? 1.38 : 1.3) * rounds(192, 128, 2 * kCus), t256 = (dx ? 1.8 : 1.8 + 220. / (double)K) * rounds(256, 256, kCus);
    return t256 < std::min(t128, t192) ? k256 : t192 < t128 ? k192 : k128;
}
template <typename T, bool YC, int WAY, int STEPS>
int launch_resident(const Product<T>& in, hipStream_t stream) {
    Product<T> a = in;
    if (!YC && a.gate != nullptr) a.rows = a.per_sample;     // (tiles of one sample)
    Resident q{};
    q.blocks = (int)ceil_div(a.N, kResColumns);
    q.slots = kCus / 8 / q.blocks * 8;
    q.per_sample = (int)ceil_div(a.rows, kResRows);
    q.tiles = a.M / a.rows * q.per_sample;
    constexpr int lds = (kResStages * kResRows * kStep * STEPS + kResWaves * kResOwn) * (int)sizeof(T);
    auto kernel = resident_kernel<T, YC, WAY, STEPS>;
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, lds);
    if (e != hipSuccess) return fail(-101, "linear: %s", hipGetErrorString(e));
    hipLaunchKernelGGL(kernel, dim3(kCus), dim3(64 * kResWaves), lds, stream, a, q);
    return 0;
}
// Whether the weights stay in registers: a contraction of five or six steps (four measured no gain, more leave no registers), columns of which a wave has
// 32 or none and at most a quarter of the waves none, and four tiles for each workgroup, which pay for the weights' way there.  us, tiles / this:
//     131072, 384 > 384     70 / 52       16384, 384 > 1536    29 / 25      131072, 320 > 1280    161 / 137      samples of 256 rows, each with weights of its own
//      32768, 384 > 384   17.1 / 17.2      8192, 384 > 1536    17 / 16       32768, 320 > 1280     47 / 39       (131072, dx 384 > 1536)   350 / 269
//      16384, 384 > 384     11 / 12.5      4096, 384 > 1536    11 / 11.4    131072, 256 > 1024    109 / 109       32768, 384 > 480   21 / 23
template <bool YC, typename T>
bool resident(const Product<T>& a) {
    const int64_t rows = YC ? a.rows : a.gate != nullptr ? a.per_sample : a.M, blocks = ceil_div(a.N, kResColumns);
    if ((a.K != 5 * kStep && a.K != 6 * kStep) || a.N % 32 != 0 || !a.wide || 4 * a.N < 3 * kResColumns * blocks || blocks > kCus / 8) return false;
    return rows >= 8 * kResRows && a.M % rows == 0 && (int64_t)a.M * a.N >= 4 * kResRows * kResColumns * blocks * (kCus / 8 / blocks * 8);
}
bool few_rows(int64_t M, int64_t N) { return M <= kFewRows || ceil_div(M, kFewRows) * ceil_div(N, kFewColumns) <= kCus; }
template <typename T, bool YC, int WAY>
int launch_few_rows(const Product<T>& a, hipStream_t stream) {
    const dim3 grid((unsigned)ceil_div(a.N, kFewColumns), (unsigned)ceil_div(a.M, kFewRows)), block(64 * kFewWaves);
    constexpr int lds = kFewWaves * 2 * kFewStage * (int)sizeof(T);                            // (the sums of up to 64 rows fit in it as well)
    if (a.M <= 16) hipLaunchKernelGGL(HIP_KERNEL_NAME(few_rows_kernel<T, YC, 1, WAY>), grid, block, lds, stream, a);
    else if (a.M <= 32) hipLaunchKernelGGL(HIP_KERNEL_NAME(few_rows_kernel<T, YC, 2, WAY>), grid, block, lds, stream, a);
    else hipLaunchKernelGGL(HIP_KERNEL_NAME(few_rows_kernel<T, YC, 4, WAY>), grid, block, lds, stream, a);
    return 0;
}
// dW in tiles of 192 x 128 where they cover its rows with no more than those of 128 x 128 do: a fifth less to fetch for a product, and two of them fit a CU
// as well.  us, 128 / 192 rows: 131072 rows of 384 and 1536 channels 215 / 196 either way round, of 8 gated samples 256 / 230, 384 x 384 73 / 73
int dw_rows(int64_t N) { return ceil_div(N, 192) * 192 <= ceil_div(N, 128) * 128 ? 192 : 128; }
template <typename T, bool XC, bool YC, int WAY>
int launch_way(Product<T>& a, int splits, hipStream_t stream) {
    a.group = (int64_t)a.N * a.K <= (1 << 20) || XC ? 1 : 8;  // (rows of tiles that share y while it does not fit the L2 beside them)
    if constexpr (XC) {
        if (dw_rows(a.M) == 192 && ceil_div(a.M, 192) * ceil_div(a.N, 128) * splits >= kCus) return launch_tiles<T, XC, YC, 192, 128, 2, 2, WAY>(a, splits, stream);
        if (ceil_div(a.M, 128) * ceil_div(a.N, 128) * splits >= kCus) return launch_tiles<T, XC, YC, 128, 128, 2, 2, WAY>(a, splits, stream);
        return launch_tiles<T, XC, YC, 64, 64, 2, 2, WAY>(a, splits, stream);
    } else {
        if (few_rows(a.M, a.N) && a.y_sample == 0) return launch_few_rows<T, YC, WAY>(a, stream);
        if constexpr (WAY != kAnything) {
            if (resident<YC>(a)) return a.K == 5 * kStep ? launch_resident<T, YC, WAY, 5>(a, stream) : launch_resident<T, YC, WAY, 6>(a, stream);
        }
        switch (tiles_for(a.M, a.N, a.K, YC)) {
            case k64: return launch_tiles<T, XC, YC, 64, 64, 2, 2, WAY>(a, splits, stream);
            case k128: return launch_tiles<T, XC, YC, 128, 128, 2, 2, WAY>(a, splits, stream);
            case k192: return launch_tiles<T, XC, YC, 192, 128, 2, 2, WAY>(a, splits, stream);
            default: return launch_tiles<T, XC, YC, 256, 256, 2, 4, WAY>(a, splits, stream);
        }
    }
}
template <typename T, bool XC, bool YC>
int launch_product(Product<T>& a, int splits, hipStream_t stream) {
    if constexpr (XC) {
        return launch_way<T, XC, YC, 0>(a, splits, stream);
    } else {
        if (!a.wide_side || !a.wide_out) return launch_way<T, XC, YC, kAnything>(a, splits, stream);
        if constexpr (YC) {
            switch (a.act) {
                case LLSA_ACT_SILU: return launch_way<T, XC, YC, kSlope + LLSA_ACT_SILU>(a, splits, stream);
                case LLSA_ACT_GELU: return launch_way<T, XC, YC, kSlope + LLSA_ACT_GELU>(a, splits, stream);
                case LLSA_ACT_GELU_TANH: return launch_way<T, XC, YC, kSlope + LLSA_ACT_GELU_TANH>(a, splits, stream);
                default: return launch_way<T, XC, YC, LLSA_ACT_NONE>(a, splits, stream);
            }
        } else {
            switch (a.act) {
                case LLSA_ACT_SILU: return launch_way<T, XC, YC, LLSA_ACT_SILU>(a, splits, stream);
                case LLSA_ACT_GELU: return launch_way<T, XC, YC, LLSA_ACT_GELU>(a, splits, stream);
                case LLSA_ACT_GELU_TANH: return launch_way<T, XC, YC, LLSA_ACT_GELU_TANH>(a, splits, stream);
                default: return launch_way<T, XC, YC, LLSA_ACT_NONE>(a, splits, stream);
            }
        }
    }
}

// The pieces of dW's contraction over the token rows, of which `samples` runs have to be kept apart.  More pieces fill the chip's workgroups more evenly
// but are more sums to write and read: the products run at about 0.72 PFLOP/s where all workgroups are busy, the sums at 4 TB/s.  131072 rows of 1536 and
// 384 channels, in 128 x 128: 14 pieces (504 workgroups of 512) 216 + 7 us; of 8 samples, 1 piece each (288 workgroups) 324 + 15.
struct Pieces { int samples, pieces; int64_t sample, piece; int count() const { return samples * pieces; } };
Pieces weight_pieces(int64_t M, int64_t samples, int N, int K) {
    const int64_t tiles = ceil_div(N, dw_rows(N)) * ceil_div(K, 128), rows = M / samples;
    const double all = 2. * (double)M * N * K / 0.72e9, sums = 8. * (double)samples * N * K / 4e6;      // us
    int64_t best = 1;
    double least = 0;
    for (int64_t p = 1; p <= std::max<int64_t>(1, rows / 256) && (p - 1) * tiles * samples < 8 * kCus; p++) {
        const double n = (double)(tiles * samples * p) / (2 * kCus), t = all * std::ceil(n) / n + sums * p;
        if (p == 1 || t < least) best = p, least = t;
    }
    const int64_t length = ceil_div(ceil_div(rows, best), kStep) * kStep;
    return {(int)samples, (int)ceil_div(rows, length), rows, length};
}
template <typename T>
void one_piece(Product<T>& a) {
    a.rows = a.M;
    a.k_sample = a.k_piece = a.K;
    a.pieces = 1;
}
template <typename T>
int linear_fwd(const llsa_linear_args& q, hipStream_t stream) {
    Product<T> a{};
    a.x = (const T*)q.x; a.ldx = q.ldx;
    a.y = (const T*)q.w; a.ldy = q.ldw;
    a.M = (int)q.M; a.N = q.N; a.K = q.K;
    one_piece(a);
    a.bias = (const T*)q.bias; a.gate = (const T*)q.gate; a.s_gate = q.s_gate; a.per_sample = (int)q.per_sample;
    a.residual = (const T*)q.residual; a.ldr = q.ldr;
    a.out = (T*)q.out; a.ldo = q.ldo; a.z = (T*)q.z; a.ldz = q.ldz;
    a.act = q.act;
    a.wide = q.N % 8 == 0 && wide8(q.bias, 0) && wide8(q.gate, q.s_gate);
    a.wide_side = q.residual == nullptr || (q.N % 8 == 0 && wide8(q.residual, q.ldr));
    a.wide_out = (q.N % 8 == 0 && wide8(q.out, q.ldo)) || q.padded;
    if (int rc = launch_product<T, false, false>(a, 1, stream)) return rc;
    return launch_status("linear_fwd");
}
template <typename T>
int linear_dx(const llsa_linear_args& q, hipStream_t stream) {
    Product<T> a{};
    a.x = (const T*)q.dz; a.ldx = q.lddz;
    a.y = (const T*)q.w; a.ldy = q.ldw; a.y_sample = q.s_w;
    a.scales = (const bf16*)q.scales; a.s_scales = pad8(q.K);
    a.M = (int)q.M; a.N = q.K; a.ny = (int)pad8(q.K); a.K = q.N;
    one_piece(a);
    if (q.s_w != 0) a.rows = (int)q.per_sample;
    a.out = (T*)q.out; a.ldo = q.ldo;
    a.slope_at = (const T*)q.z; a.ldz = q.ldz; a.act = q.z != nullptr ? q.act : LLSA_ACT_NONE;
    a.wide = a.wide_side = 1;
    a.wide_out = (q.K % 8 == 0 && wide8(q.out, q.ldo)) || q.padded;
    if (int rc = launch_product<T, false, true>(a, 1, stream)) return rc;
    return launch_status("linear_dx");
}
template <typename T>
int linear_dw(const llsa_linear_args& q, hipStream_t stream) {
    const Pieces p = weight_pieces(q.M, q.gate != nullptr ? q.M / q.per_sample : 1, q.N, q.K);
    Product<T> a{};
    a.x = (const T*)q.dz; a.ldx = q.lddz; a.nx = (int)pad8(q.N);
    a.y = (const T*)q.x; a.ldy = q.ldx; a.ny = (int)pad8(q.K);
    a.M = q.N; a.N = q.K; a.K = q.M;
    one_piece(a);
    a.k_sample = p.sample; a.k_piece = p.piece; a.pieces = p.pieces;
    a.ld_part = pad8(q.K);
    if (q.gate == nullptr && p.count() == 1) {
        a.out = (T*)q.out; a.ldo = q.ldo; a.sums = (T*)q.dbias;
        a.wide_out = q.K % 8 == 0 && wide8(q.out, q.ldo);
        if (int rc = launch_product<T, true, true>(a, 1, stream)) return rc;
        return launch_status("linear_dw");
    }
    a.part = (float*)q.workspace;
    a.ldo = a.ld_part;
    const bool sums = q.dbias != nullptr || (q.dgate != nullptr && q.bias != nullptr);
    a.part_sum = sums ? a.part + (int64_t)p.count() * a.M * a.ld_part : nullptr;
    if (int rc = launch_product<T, true, true>(a, p.count(), stream)) return rc;
    if (q.gate != nullptr) {
        GatedJoin j{};
        j.part = a.part; j.part_sum = a.part_sum; j.gate = q.gate; j.s_gate = q.s_gate; j.w = q.w; j.ldw = q.ldw; j.bias = q.bias;
        j.out = q.out; j.ldo = q.ldo; j.sums = q.dbias; j.dgate = q.dgate;
        j.ld_part = a.ld_part; j.M = a.M; j.N = a.N; j.samples = p.samples; j.pieces = p.pieces;
        hipLaunchKernelGGL(HIP_KERNEL_NAME(gated_join_kernel<T>), dim3((unsigned)a.M), dim3(kJoinThreads), 4 * kJoinGroups * p.samples, stream, j);
    } else {
        const int64_t places = (int64_t)a.M * (a.ld_part / 4) + (q.dbias != nullptr ? a.M : 0);
        hipLaunchKernelGGL(HIP_KERNEL_NAME(product_join_kernel<T>), dim3((unsigned)ceil_div(places, 64)), dim3(256), 0, stream, a.part, a.part_sum, (T*)q.out, q.ldo,
                           (T*)q.dbias, a.M, a.N, a.ld_part, p.count());
    }
    return launch_status("linear_dw");
}
template <typename T>
int gate_rows(const llsa_linear_args& q, hipStream_t stream) {
    if constexpr (std::is_same_v<T, _Float16>) {
        const int groups = (int)ceil_div(q.ldo, kScaleColumns);
        hipLaunchKernelGGL(gate_rows_scaled_kernel, dim3((unsigned)(q.M / q.per_sample * groups)), dim3(kScaleThreads), 0, stream, (const T*)q.w, q.ldw, (const T*)q.gate, q.s_gate, (T*)q.out,
                           q.ldo, (bf16*)q.scales, q.N, groups);
    } else {
        const int64_t pieces = q.M / q.per_sample * q.N * (q.ldo / 8);
        hipLaunchKernelGGL(gate_rows_kernel, dim3((unsigned)ceil_div(pieces, 256)), dim3(256), 0, stream, (const T*)q.w, q.ldw, (const T*)q.gate, q.s_gate, (T*)q.out, q.ldo, q.N, pieces);
    }
    return launch_status("linear_gate_rows");
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

extern "C" int64_t llsa_linear_dw_workspace_bytes(int64_t M, int64_t samples, int N, int K) {
    if (M <= 0 || samples <= 0 || N <= 0 || K <= 0) return 0;
    return 4 * (int64_t)weight_pieces(M, samples, N, K).count() * N * (pad8(K) + 1);      // (also where the one piece of a layer without a gate goes straight to dW)
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
    LLSA_REQUIRE(a->gate == nullptr || (a->per_sample > 0 && a->M % a->per_sample == 0), "linear_fwd: rows of a sample, whole samples");
    LLSA_REQUIRE(offsets32(a->ldo) && (a->residual == nullptr || offsets32(a->ldr)), "linear_fwd: rows of out and residual at most %lld apart", (long long)kMaxLd);
    return BY_TYPE(linear_fwd);
}
extern "C" int llsa_linear_dx(const llsa_linear_args* a, void* stream) {
    LLSA_REQUIRE(a != nullptr, "linear_dx: no arguments");
    if (int rc = check_sizes("linear_dx", a->M, a->N, a->K, a->dtype, a->act)) return rc;
    if (a->M == 0) return 0;
    LLSA_REQUIRE(rows16(a->dz, a->lddz) && rows16(a->w, a->ldw) && a->lddz >= pad8(a->N) && a->ldw >= pad8(a->K),
                 "linear_dx: rows of dz and w must be 16-byte aligned and padded to a multiple of 8");
    LLSA_REQUIRE(a->scales == nullptr || (a->s_w != 0 && a->dtype == LLSA_DTYPE_F16 && aligned16(a->scales)), "linear_dx: scales go with fp16 weights of each sample");
    LLSA_REQUIRE(a->s_w == 0 || (a->s_w % 8 == 0 && a->per_sample > 0 && a->M % a->per_sample == 0), "linear_dx: weights of each sample: whole samples, 16-byte aligned");
    LLSA_REQUIRE(a->out != nullptr && (!a->padded || (rows16(a->out, a->ldo) && a->ldo >= pad8(a->K))), "linear_dx: output, padded rows 16-byte aligned and a multiple of 8 long");
    LLSA_REQUIRE(a->z == nullptr || (rows16(a->z, a->ldz) && a->ldz >= pad8(a->K)), "linear_dx: rows of z must be 16-byte aligned and padded to a multiple of 8");
    LLSA_REQUIRE(offsets32(a->ldo), "linear_dx: rows of dx at most %lld apart", (long long)kMaxLd);
    return BY_TYPE(linear_dx);
}
extern "C" int llsa_linear_dw(const llsa_linear_args* a, void* stream) {
    LLSA_REQUIRE(a != nullptr, "linear_dw: no arguments");
    if (int rc = check_sizes("linear_dw", a->M, a->N, a->K, a->dtype, a->act)) return rc;
    LLSA_REQUIRE(a->M > 0, "linear_dw: no rows");
    LLSA_REQUIRE(rows16(a->dz, a->lddz) && rows16(a->x, a->ldx) && a->lddz >= pad8(a->N) && a->ldx >= pad8(a->K),
                 "linear_dw: rows of dz and x must be 16-byte aligned and padded to a multiple of 8");
    LLSA_REQUIRE(a->out != nullptr && offsets32(a->ldo) && a->workspace != nullptr && aligned16(a->workspace), "linear_dw: output and workspace (16-byte aligned)");
    LLSA_REQUIRE(a->gate == nullptr || (a->per_sample > 0 && a->M % a->per_sample == 0 && a->M / a->per_sample <= LLSA_LINEAR_MAX_GATED_SAMPLES),
                 "linear_dw: a gate needs whole samples, at most %d", LLSA_LINEAR_MAX_GATED_SAMPLES);
    LLSA_REQUIRE(a->dgate == nullptr || (a->gate != nullptr && a->w != nullptr), "linear_dw: dgate needs the gate and the weight");
    return BY_TYPE(linear_dw);
}
extern "C" int llsa_linear_gate_rows(const llsa_linear_args* a, void* stream) {
    LLSA_REQUIRE(a != nullptr, "linear_gate_rows: no arguments");
    if (int rc = check_sizes("linear_gate_rows", a->M, a->N, a->K, a->dtype, a->act)) return rc;
    if (a->M == 0) return 0;
    LLSA_REQUIRE(a->gate != nullptr && a->per_sample > 0 && a->M % a->per_sample == 0, "linear_gate_rows: gate, whole samples");
    LLSA_REQUIRE(rows16(a->w, a->ldw) && rows16(a->out, a->ldo) && a->ldo == pad8(a->K) && a->ldw >= a->ldo, "linear_gate_rows: rows 16-byte aligned and padded to a multiple of 8");
    LLSA_REQUIRE(a->dtype != LLSA_DTYPE_F16 || (a->scales != nullptr && aligned16(a->scales)), "linear_gate_rows: fp16 needs room for the scales, 16-byte aligned");
    LLSA_REQUIRE(ceil_div(a->M / a->per_sample * a->N * (a->ldo / 8), 256) <= kMaxGrid && a->M / a->per_sample * ceil_div(a->ldo, kScaleColumns) <= kMaxGrid,
                 "linear_gate_rows: too many samples");
    return BY_TYPE(gate_rows);
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
extern "C" int llsa_pad_rows(const llsa_pad_job* jobs, int n, void* stream) {
    LLSA_REQUIRE(jobs != nullptr && n >= 1 && n <= LLSA_PAD_JOBS, "pad_rows: 1 to %d matrices", LLSA_PAD_JOBS);
    Pads a{};
    int64_t total = 0;
    for (int i = 0; i < LLSA_PAD_JOBS; i++) {
        if (i < n) {
            const llsa_pad_job& q = jobs[i];
            LLSA_REQUIRE(q.rows >= 0 && q.cols > 0 && q.ldy >= q.cols && rows16(q.y, q.ldy) && (q.rows == 0 || q.x != nullptr), "pad_rows: bad arguments");
            a.job[i] = q;
            total += q.rows * (q.ldy / 8);
        }
        a.end[i] = total;
    }
    if (total == 0) return 0;
    LLSA_REQUIRE(ceil_div(total, 256) <= kMaxGrid, "pad_rows: too many rows");
    hipLaunchKernelGGL(pad_kernel, dim3((unsigned)ceil_div(total, 256)), dim3(256), 0, (hipStream_t)stream, a);
    return launch_status("pad_rows");
}
