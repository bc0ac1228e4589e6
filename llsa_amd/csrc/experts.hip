// Products of rows with the weights of the expert that each belongs to, and the feed-forward block made of two of them.  Rows stand sorted by expert,
// those of expert e at offsets[e] .. offsets[e + 1] - 1; the offsets stay on the device, so a launch has a workgroup for every piece of rows there can be,
// and each finds its expert by itself (experts_device.h).
//
//     forward   z = x W_e^T + b_e,   h = act(z)                     of a block: y = h W_out^T + b_out,   out = residual + gate * sum of a token's w y
//     backward  dx = dz W_e,   dW_e = dz^T x,   db_e = sum dz
//
// Of a block: with g = w gate dout, a row for each of a token's experts,   dz = act'(z) (g W_out),   dW_out = g^T h,   db_out = sum g,   dw = gate dout . y.
// Rows of tokens (x, g) are brought into the order of the places once, where a product for each of a row's columns would gather them again (262144 rows of
// 384 and 1536 channels, us: dW of gathered rows 573 and 530, of rows in order 376, and some 50 for the copy, which multiplies by w as well); few rows and the
// smallest tiles of a forward without a backward gather them on their way into LDS.  The weight stays out of the products: in the hidden rows (h' = w act(z), so
// that dout needs no factor) dw is a sum over act(z) (dout W_out) on the way out of that product, whose waves have no registers left for it (20 to 30
// spilled: 1050 us instead of 490).
//
// Sums are fp32, and so are what happens on the way out and the rows that each expert gives a token (y, and dx of each), which are added up.  Rounded to 16 bits
// besides the results is what a product takes in that another made (h, g, dz), as in the linear layers: half a step of each, 2^-8 of it in bf16 (fp16 2^-11, and 2^-25 below
// 2^-14, where g and dz lie as the linear layers' dz does: a scale of the loss moves them).  What a
// backward wants of z is act'(z), which lies between -0.13 and 1.13: 16 bits hold it in steps of 2^-14, and to seven bits and more where it is small, far below zero; z
// itself would be half a step of bf16 off.
#include "experts_device.h"

namespace llsa {
namespace {

// ---------------------------------------------------------------------------------------
// forward and dx
// ---------------------------------------------------------------------------------------
template <typename T>
struct Grouped {
    const T *x, *y;                       // rows of tokens (or of places, without an order), weights
    int64_t ldx, ldy, y_expert;
    const int32_t* offsets;
    Order order;
    int experts, rows, N, ny, K;          // rows: of places
    int tiles_n, group, gaps;             // gaps: zeros go to the rows that no expert has
    // way out
    const T* bias;
    const int16_t* slope_at;              // dx
    int64_t ldo, ldz;
    void* out;                            // T, or fp32 (kWide)
    int16_t* slopes;                      // forward: kept unless NULL
    int wide, wide_out;                   // wide: 16-byte accesses to bias; wide_out: to out, or its rows are padded with zeros to a multiple of 8
};
struct Here { int expert, m0, m_end, n0, tn; };
// What is on the way out: in the forward an activation (its LLSA_ACT_ number), in dx the slopes that the forward kept; neither, to T or (kWide) to fp32
enum { kBySlope = 1, kWide = 4 };
template <int BM, int BN, typename P>
__device__ __forceinline__ bool find_tile(const P& a, Here& h, int lane) {
    Runs runs;
    runs.load(a.offsets, a.experts, a.rows, BM, a.gaps != 0, lane);
    const int total = runs.total * a.tiles_n;
    if ((int)blockIdx.x >= total) return false;
    const int at = xcd_order((int)blockIdx.x, total), in_group = a.group * a.tiles_n, g = at / in_group, rest = at - g * in_group;
    const int rows_here = min(a.group, runs.total - g * a.group), tn = rest / rows_here, t = g * a.group + rest - tn * rows_here;
    const Piece p = runs.find(t);
    h = {p.expert, p.begin + (t - p.first) * BM, p.end, tn * BN, tn};
    return true;
}

// act'(z) in 16 bits.  What matters for the products is its error beside 1: from -0.13 to 1.13 steps of 2^-14.  What matters to a unit far below zero, where all three
// activations' slopes are negative and shrink to the least numbers, is its error beside itself: negative ones above -2^-4 are kept with an exponent.  (Positive ones
// below 2^-4 lie where act' crosses zero, and are no better known than z.)  The steps are numbers from 0 on, 4096 of them below zero.  Numbers with the sign bit are one
// more than: from -0 on the upper half of the float (seven bits behind the leading one), and from 2^-19 to 2^-4 ten bits behind it.  The two meet where they are equal, and
// above it the second, below it the first is the larger.  0x8000 is left for a NaN, and reads as one by itself.
typedef __attribute__((ext_vector_type(8))) int16_t s16x8;
constexpr unsigned kSlopeJoin = (108u << 23) - (108u << 20);          // 2^-19: number 108 << 7 of either kind
// (a value that is made in any case: of a choice between two the compiler makes a branch for each element, and 262144 rows 384 > 1536 back by the slopes took 520 us where
// they take 450)
__device__ __forceinline__ unsigned made(unsigned v) {
#ifndef LLSA_CPU_EMU_BUILD
    asm("" : "+v"(v));
#endif
    return v;
}
__device__ __forceinline__ int16_t slope_kept(float z, float slope) {
    const unsigned bits = __float_as_uint(slope);
    const int seven = (int)((bits + 0x18000u) >> 16), ten = (int)(bits + 0x3000u - 0x80000000u - kSlopeJoin + (0x8000u << 13)) >> 13;
    // (added to 1.5 2^23 a number's last bits are its whole part, rounded)
    const unsigned step = __float_as_uint(fmaf(slope, 16384.f, 12582912.f + 4096.f)), small = made((unsigned)max(seven, ten));
    return z != z ? (int16_t)-32768 : (int16_t)((int)bits < (int)0xbd800000u ? small : step);      // (0xbd800000: -2^-4; as integers negative floats are the lowest)
}
__device__ __forceinline__ float slope_of(int16_t kept) {
    const unsigned k = (uint16_t)kept, seven = (k << 16) - 0x10000u, ten = (k << 13) + (kSlopeJoin + 0x80000000u - (0x8001u << 13));
    const unsigned step = __float_as_uint(fmaf((float)kept, 0x1p-14f, -0.25f)), small = made(min(seven, ten));
    return __uint_as_float(kept < 0 ? small : step);
}

// Eight values of a row on their way out.  kept: the slopes, in the forward; early: those of the layer in front, in dx
template <bool YC, int ACT, bool TIGHT = false, typename T>
__device__ __forceinline__ void way_out(const Grouped<T>& a, float (&v)[8], const vec8<T>& bias, const s16x8& early, s16x8& kept) {
    if constexpr (!YC) {
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] += (float)bias[e];
        if constexpr (ACT != LLSA_ACT_NONE && ACT != kWide) {
            if (a.slopes != nullptr) {
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    float value, slope;
                    activate_both(ACT, v[e], value, slope);
                    kept[e] = slope_kept(v[e], slope);
                    v[e] = value;
                    if (TIGHT && e % 2 == 1) __builtin_amdgcn_sched_barrier(0);      // (two at a time: there are no registers for more)
                }
            } else {
#pragma unroll
                for (int e = 0; e < 8; e++) v[e] = activate(ACT, v[e]);
            }
        }
    } else if constexpr (ACT == kBySlope) {
#pragma unroll
        for (int e = 0; e < 8; e++) {
            v[e] *= slope_of(early[e]);
            if (TIGHT && e % 2 == 1) __builtin_amdgcn_sched_barrier(0);
        }
    }
}
template <typename T>
__device__ __forceinline__ vec8<T> rounded(const float (&v)[8], int left) {
    vec8<T> o;
#pragma unroll
    for (int e = 0; e < 8; e++) o[e] = (T)(e >= left ? 0.f : v[e]);
    return o;
}
template <typename T>
__device__ __forceinline__ void put8(T* to, const vec8<T>& o, bool wide, int left) {
    if (wide) {
        *reinterpret_cast<vec8<T>*>(to) = o;
    } else {
#pragma unroll
        for (int e = 0; e < 8; e++)
            if (e < left) to[e] = o[e];
    }
}
__device__ __forceinline__ void put8_wide(float* to, const float (&v)[8]) {
    *reinterpret_cast<f32x4*>(to) = f32x4{v[0], v[1], v[2], v[3]};
    *reinterpret_cast<f32x4*>(to + 4) = f32x4{v[4], v[5], v[6], v[7]};
}
template <int BM, int BN, int ACT, typename T>
__device__ __forceinline__ void write_zeros(const Grouped<T>& a, const Here& h) {
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; e++) v[e] = 0.f;
    for (int i = threadIdx.x; i < BM * (BN / 8); i += blockDim.x) {
        const int r = i / (BN / 8), n = h.n0 + (i - r * (BN / 8)) * 8;
        if (h.m0 + r >= h.m_end || n >= a.N) continue;
        const int64_t at = (int64_t)(h.m0 + r) * a.ldo + n;
        if constexpr (ACT == kWide) put8_wide(static_cast<float*>(a.out) + at, v);
        else store8(static_cast<T*>(a.out) + at, v, a.wide_out, a.N - n);
    }
}

// The tiles of linear.hip's product_kernel, with an expert's weights; GATHERED: rows of tokens, brought into order on their way into LDS.  Bound as those are by the
// operands' way, whose copies every step of 64 waits for, and by the last tile of each expert, half of it empty on the average.  us, rows of eight experts: 16384, 2048 > 2048 171 (0.81 PFLOP/s;
// 256 x 256 181), its dx 168 to 180; 262144, 1536 > 384 to fp32 385 to 396 (0.78; a library's product of as many rows with one weight, to bf16, 324), dx 1536 > 384 428 to
// 447; the matrix units work 28 to 32 % of the last two's time.
template <typename T, bool YC, bool GATHERED, int BM, int BN, int WAVES_M, int WAVES_N, int ACT>
__global__ __launch_bounds__(64 * WAVES_M * WAVES_N, 2) void grouped_kernel(const Grouped<T> a) {
    constexpr int kWaves = WAVES_M * WAVES_N, WM = BM / WAVES_M, WN = BN / WAVES_N, MT = WM / 16, NT = WN / 16, kTileX = BM * kStep, kTileY = BN * kStep;
    constexpr bool kSlope = YC && ACT == kBySlope;
    constexpr bool kKeeps = !YC && ACT != LLSA_ACT_NONE && ACT != kWide;
    typedef Operand<T, false, BM, kWaves> OperandX;
    typedef Operand<T, YC, BN, kWaves> OperandY;
    HIP_DYNAMIC_SHARED(char, shared)
    T* const lds = reinterpret_cast<T*>(shared);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int quad = lane >> 4, wm = (wave % WAVES_M) * WM, wn = (wave / WAVES_M) * WN;
    Here here;
    if (!find_tile<BM, BN>(a, here, lane)) return;
    if (here.expert < 0) {
        write_zeros<BM, BN, ACT>(a, here);
        return;
    }
    RowsAlong<T, BM, kWaves, GATHERED> ox;
    OperandY oy;
    ox.init(a.x, a.ldx, a.order, here.m0, min(BM, here.m_end - here.m0), wave, lane);
    oy.init(wave, lane, a.ldy, min(BN, (YC ? a.ny : a.N) - here.n0));
    const T* py = a.y + here.expert * a.y_expert + (YC ? (int64_t)here.n0 : (int64_t)here.n0 * a.ldy);
    const int64_t stepy = YC ? kStep * a.ldy : kStep;
    int k = 0;
    auto request = [&](int buffer) {
        T* const t = lds + buffer * (kTileX + kTileY);
        ox.request(t, wave, lane, a.K - k);
        oy.request(py, t + kTileX, wave, lane, a.K - k);
        py += stepy;
        k += kStep;
    };
    f32x4 acc[NT][MT];
#pragma unroll
    for (int i = 0; i < NT; i++)
#pragma unroll
        for (int j = 0; j < MT; j++) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
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
        }
    };

    const int lane_row = lane & 15, lane_col = 16 * (quad & 1) + 8 * (quad >> 1);
    const int row0 = here.m0 + wm, col0 = here.n0 + wn, rows_left = here.m_end - row0 - lane_row, cols_left = a.N - col0 - lane_col;
    const unsigned at_out = (unsigned)(lane_row * a.ldo) + lane_col, at_z = (unsigned)(lane_row * a.ldz) + lane_col;
    constexpr int kPair = NT % 4 == 0 ? 2 : 1;                // pieces of 32 columns that leave together
    const bool whole = kPair == 2 && here.m0 + BM <= here.m_end && here.n0 + BN <= a.N && a.wide_out;
    s16x8 early[kPair][MT];
    auto read_side = [&](int p0) {
        if constexpr (kSlope) {
            if constexpr (kPair == 2) {
                if (whole) {
#pragma unroll
                    for (int j = 0; j < MT; j++)
                        request_lines(reinterpret_cast<vec8<T>&>(early[0][j]), reinterpret_cast<vec8<T>&>(early[1][j]),
                                      reinterpret_cast<const T*>(a.slope_at) + ((int64_t)(row0 + 16 * j) * a.ldz + (col0 + 32 * p0)), at_z, (unsigned)(8 * a.ldz), lane);
                    return;
                }
            }
#pragma unroll
            for (int j = 0; j < MT; j++)
#pragma unroll
                for (int h = 0; h < kPair; h++)
                    if (16 * j < rows_left && 32 * (p0 + h) < cols_left)
                        early[h][j] = *reinterpret_cast<const s16x8*>(a.slope_at + ((int64_t)(row0 + 16 * j) * a.ldz + (col0 + 32 * (p0 + h))) + at_z);
        }
    };
    const int steps = (a.K + kStep - 1) / kStep;
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

    const T* const bias_row = !YC && a.bias != nullptr ? a.bias + (int64_t)here.expert * a.N + col0 + lane_col : nullptr;
#pragma unroll
    for (int p0 = 0; p0 < NT / 2; p0 += kPair) {
        vec8<T> bias[kPair];
#pragma unroll
        for (int h = 0; h < kPair; h++) {
            const int left = cols_left - 32 * (p0 + h);
            bias[h] = take8(bias_row != nullptr && left > 0 ? bias_row + 32 * (p0 + h) : nullptr, a.wide, left);
        }
#pragma unroll
        for (int j = 0; j < MT; j++) {
            const int64_t row = row0 + 16 * j;
            vec8<T> o[kPair];
            s16x8 kept[kPair];
            if constexpr (kPair == 2 && kSlope) {
                if (whole) arrange_lines<T>(reinterpret_cast<vec8<T>&>(early[0][j]), reinterpret_cast<vec8<T>&>(early[1][j]), lane);
            }
#pragma unroll
            for (int h = 0; h < kPair; h++) {
                const int p = p0 + h, col = col0 + 32 * p, left = cols_left - 32 * p;
                float v[8];
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const u32x2 w = __builtin_amdgcn_permlane16_swap(__float_as_uint(acc[2 * p][j][e]), __float_as_uint(acc[2 * p + 1][j][e]), false, false);
                    v[e] = __uint_as_float(w[0]);
                    v[4 + e] = __uint_as_float(w[1]);
                }
                if (16 * j >= rows_left || left <= 0) continue;
                way_out<YC, ACT>(a, v, bias[h], early[h][j], kept[h]);
                if constexpr (ACT == kWide) {
                    put8_wide(static_cast<float*>(a.out) + (row * a.ldo + col) + at_out, v);
                } else {
                    o[h] = rounded<T>(v, left);
                    if (whole) continue;
                    if (kKeeps && a.slopes != nullptr) *reinterpret_cast<s16x8*>(a.slopes + (row * a.ldz + col) + at_z) = kept[h];
                    put8(static_cast<T*>(a.out) + (row * a.ldo + col) + at_out, o[h], a.wide_out, left);
                }
            }
            if constexpr (kPair == 2 && ACT != kWide) {
                if (whole) {
                    if (kKeeps && a.slopes != nullptr)
                        store_lines(reinterpret_cast<T*>(a.slopes) + (row * a.ldz + (col0 + 32 * p0)), at_z, (unsigned)(8 * a.ldz), __builtin_bit_cast(vec8<T>, kept[0]),
                                    __builtin_bit_cast(vec8<T>, kept[1]), lane);
                    store_lines(static_cast<T*>(a.out) + (row * a.ldo + (col0 + 32 * p0)), at_out, (unsigned)(8 * a.ldo), o[0], o[1], lane);
                }
            }
            __builtin_amdgcn_sched_barrier(0);                // (rows one after another: all at once do not fit the registers)
        }
        if (p0 + kPair < NT / 2) read_side(p0 + kPair);
    }
}

// Few rows for each expert: a workgroup takes 32 columns of up to 64 rows of one, its eight waves an eighth of the contraction each, through two stages of
// LDS of their own; the sums meet at the end (linear.hip's few_rows_kernel).  An expert's weight is read once for them, and there is little else: 16 rows of eight
// experts 384 > 1536, 9.5 MB of weights, 5.2 us.  With up to a workgroup for each CU; at two for each (2048 rows 1536 > 384) the smallest tiles take 14 and this 19.5.
constexpr int kFewWaves = 8, kFewColumns = 32, kFewStage = kFewColumns * kStep;
template <typename T, bool YC, int MT, int ACT>
__global__ __launch_bounds__(64 * kFewWaves, 2) void grouped_few_kernel(const Grouped<T> a) {
    constexpr bool kSlope = YC && ACT == kBySlope;
    constexpr bool kKeeps = !YC && ACT != LLSA_ACT_NONE && ACT != kWide;
    typedef Operand<T, YC, kFewColumns, 1> OperandY;
    HIP_DYNAMIC_SHARED(char, shared)
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), quad = lane >> 4;
    T* const stage = reinterpret_cast<T*>(shared) + wave * 2 * kFewStage;
    Here here;
    if (!find_tile<16 * MT, kFewColumns>(a, here, lane)) return;
    if (here.expert < 0) {
        write_zeros<16 * MT, kFewColumns, ACT>(a, here);
        return;
    }
    const int n0 = here.n0, row0 = here.m0, all = (a.K + kStep - 1) / kStep, each = (all + kFewWaves - 1) / kFewWaves, first = min(all, wave * each), steps = min(all - first, each);
    OperandY oy;
    oy.init(0, lane, a.ldy, min(kFewColumns, (YC ? a.ny : a.N) - n0));
    const int k0 = first * kStep;
    const T* py = a.y + here.expert * a.y_expert + (YC ? k0 * a.ldy + n0 : n0 * a.ldy + k0);
    const T* px[MT];
#pragma unroll
    for (int j = 0; j < MT; j++) {
        const int place = min(row0 + 16 * j + (lane & 15), here.m_end - 1);
        px[j] = a.x + (a.order.slots != nullptr ? a.order.token(place) : place) * a.ldx;
    }
    f32x4 acc[2][MT];
#pragma unroll
    for (int i = 0; i < 2; i++)
#pragma unroll
        for (int j = 0; j < MT; j++) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    vec8<T> next[MT][2];
    auto request = [&](int s) {
        const int k = k0 + s * kStep;
        oy.request(py + (YC ? s * kStep * a.ldy : s * kStep), stage + (s & 1) * kFewStage, 0, lane, a.K - k);
#pragma unroll
        for (int j = 0; j < MT; j++)
#pragma unroll
            for (int ks = 0; ks < 2; ks++) {
                const int at = k + 32 * ks + 8 * quad;
                next[j][ks] = *reinterpret_cast<const vec8<T>*>(at < a.K ? px[j] + at : reinterpret_cast<const T*>(kZeros));
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
    const int lane_col = 16 * (quad & 1) + 8 * (quad >> 1), m = row0 + 16 * wave + (lane & 15), left = a.N - n0 - lane_col;
    if (m >= here.m_end || left <= 0) return;
    s16x8 early = {0, 0, 0, 0, 0, 0, 0, 0}, kept;
    if (kSlope) early = *reinterpret_cast<const s16x8*>(a.slope_at + (int64_t)m * a.ldz + n0 + lane_col);
    const vec8<T> bias = take8(!YC && a.bias != nullptr ? a.bias + (int64_t)here.expert * a.N + n0 + lane_col : nullptr, a.wide, left);
    way_out<YC, ACT>(a, v, bias, early, kept);
    if (kKeeps && a.slopes != nullptr) *reinterpret_cast<s16x8*>(a.slopes + (int64_t)m * a.ldz + n0 + lane_col) = kept;
    if constexpr (ACT == kWide) put8_wide(static_cast<float*>(a.out) + (int64_t)m * a.ldo + n0 + lane_col, v);
    else put8(static_cast<T*>(a.out) + (int64_t)m * a.ldo + n0 + lane_col, rounded<T>(v, left), a.wide_out, left);
}

// Many rows for each expert, a short contraction: the weights stay in registers (linear.hip's resident_kernel).  A workgroup of twelve waves keeps 384 columns of
// an expert's weights, 32 columns a wave, and takes its share of the rows through LDS, 32 at a time and two such tiles ahead; where the expert changes it takes
// in the next one's weights.  262144 rows 384 > 1536, us by card: GELU with slopes kept 535 to 573, back by the slopes 448 to 477 (in
// tiles of 128 x 128, with slopes in steps alone, 823 and 950 where this took 501 to 535 and 433 to 455).  Back it moves 1.9 GB at 4.0 to 4.3 TB/s; the forward writes 1.6 GB and issues a vector
// instruction for 0.58 of every four cycles of a SIMD (a kernel of nothing but fp32 fma: 0.9), most of them GELU, its slope and the slope's 16 bits.
constexpr int kResWaves = 12, kResColumns = 32 * kResWaves, kResRows = 32, kResStages = 3, kResOwn = 32 * kStep + 64;
struct Entry { int expert, begin, end, first, upto; };       // upto: number of the first tile behind its own
template <typename T, bool YC, int ACT, int STEPS>
__global__ __launch_bounds__(64 * kResWaves) void grouped_resident_kernel(const Grouped<T> a, int blocks, int slots) {
    typedef Operand<T, false, kResRows, 1> OperandX;          // of a step: 4 copies
    typedef Operand<T, YC, 32, 1> OperandY;
    constexpr int kStage = kResRows * kStep * STEPS;
    constexpr bool kSlope = YC && ACT == kBySlope;
    constexpr bool kKeeps = !YC && ACT != LLSA_ACT_NONE && ACT != kWide;
    static_assert(4 * STEPS <= 2 * kResWaves, "two copies of a wave take in a tile");
    HIP_DYNAMIC_SHARED(char, shared)
    T* const lds = reinterpret_cast<T*>(shared);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), quad = lane >> 4;
    // workgroups of an XCD: the blocks of columns of the same rows side by side
    const int xcd = blockIdx.x & 7, local = blockIdx.x >> 3, block = local % blocks, slot = (local / blocks) * 8 + xcd;
    if (slot >= slots) return;
    // begin, end and upto of every expert, and of the rows before the first and behind the last
    int* const table = reinterpret_cast<int*>(lds + kResStages * kStage + kResWaves * kResOwn);
    int tiles;
    {
        Runs runs;
        runs.load(a.offsets, a.experts, a.rows, kResRows, a.gaps != 0, lane);
        tiles = runs.total;
        if (wave == 0) {
#pragma unroll
            for (int i = 0; i < Runs::kLanes; i++)
                if (64 * i + lane < a.experts) {
                    int* const e = table + 3 * (64 * i + lane);
                    e[0] = runs.begin[i];
                    e[1] = runs.end[i];
                    e[2] = runs.upto[i];
                }
            if (lane < 2) {
                int* const e = table + 3 * (a.experts + lane);
                e[0] = lane ? runs.back : 0;
                e[1] = lane ? runs.rows : runs.front;
                e[2] = lane ? runs.total : runs.of_experts + (runs.front + kResRows - 1) / kResRows;
            }
        }
    }
    __syncthreads();
    const int t0 = (int)((int64_t)tiles * slot / slots), t1 = (int)((int64_t)tiles * (slot + 1) / slots);
    if (t0 >= t1) return;
    auto entry = [&](int e, int first) {
        const int* const p = table + 3 * e;
        return Entry{e, __builtin_amdgcn_readfirstlane(p[0]), __builtin_amdgcn_readfirstlane(p[1]), first, __builtin_amdgcn_readfirstlane(p[2])};
    };
    auto advance = [&](Entry& e, int t) {                     // to the entry of tile t < tiles
        while (t >= e.upto) e = entry(e.expert + 1, e.upto);
    };
    const int n0 = block * kResColumns + 32 * wave;
    const bool columns = n0 < a.N;                            // (a wave beyond the last column copies, and does no more)
    const int lane_col = 16 * (quad & 1) + 8 * (quad >> 1), lane_row = lane & 15;
    // LDS of the wave's own: its weights on their way, 64 of the contraction at a time; the bias of its columns
    T* const own = lds + kResStages * kStage + wave * kResOwn;
    T* const vectors = own + 32 * kStep;

    // (with slopes besides, the registers are 16 short of six steps' weights: the last step's stay in LDS, where they came through)
    constexpr int kHeld = kKeeps && STEPS == 6 ? STEPS - 1 : STEPS;
    vec8<T> fy[2 * kHeld][2];
    auto weights = [&](const T* w) {
        OperandY oy;
        oy.init(0, lane, a.ldy, 32);
#pragma unroll
        for (int s = 0; s < STEPS; s++) {
            oy.request(w + (YC ? s * kStep * a.ldy + n0 : n0 * a.ldy + s * kStep), own, 0, lane, kStep);
            wave_waits_for_copies();
            if (s >= kHeld) break;
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
    Entry ahead = entry(0, 0);
    auto request = [&](int t) {
        if (t >= t1 || wave >= 2 * STEPS) return;
        advance(ahead, t);
        if (ahead.expert >= a.experts) return;
        T* const stage = lds + (t % kResStages) * kStage;
        // (the last tile of all begins early enough to be whole)
        const T* const base = a.x + (int64_t)min(ahead.begin + (t - ahead.first) * kResRows, a.rows - kResRows) * a.ldx;
#pragma unroll
        for (int c = 0; c < 2; c++) copy_to_lds(base + off[c], stage + (2 * wave + c) * 512);
    };
    request(t0);
    request(t0 + 1);
    const unsigned at_out = (unsigned)(lane_row * a.ldo) + lane_col, at_z = (unsigned)(lane_row * a.ldz) + lane_col;
    Entry now = entry(0, 0);
    wait_vm0();
    for (int t = t0, have = -1; t < t1; t++) {
        advance(now, t);
        const int first = now.begin + (t - now.first) * kResRows, m0 = min(first, a.rows - kResRows);
        if (now.expert != have && columns && now.expert < a.experts) {
            weights(a.y + now.expert * a.y_expert);
            if (!YC && lane_row == 0) *reinterpret_cast<vec8<T>*>(vectors + lane_col) = take8(a.bias != nullptr ? a.bias + (int64_t)now.expert * a.N + n0 + lane_col : nullptr, a.wide, 8);
            have = now.expert;
        }
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
        if (now.expert >= a.experts) {                        // no expert's rows
            const float zeros[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int j = 0; j < 2; j++) {
                if (first + 16 * j + lane_row >= now.end) continue;
                const int64_t at = (int64_t)(first + 16 * j) * a.ldo + n0;
                if constexpr (ACT == kWide) put8_wide(static_cast<float*>(a.out) + at + at_out, zeros);
                else *reinterpret_cast<vec8<T>*>(static_cast<T*>(a.out) + at + at_out) = take8<T>(nullptr, true, 8);
            }
            wait_vm0();
            continue;
        }
        s16x8 early[2];                                       // what is read on the way out
#pragma unroll
        for (int j = 0; j < 2; j++) {
            const int64_t row = m0 + 16 * j;                  // (rows behind the expert's last are another's, or were never written: what comes of them is not kept)
            if (kSlope) early[j] = __builtin_nontemporal_load(reinterpret_cast<const s16x8*>(a.slope_at + (row * a.ldz + n0) + at_z));
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
                for (int j = 0; j < 2; j++) {
                    if (ks < 2 * kHeld) acc[i][j] = product16(fy[ks < 2 * kHeld ? ks : 0][i], fx[j], acc[i][j]);
                    else acc[i][j] = product16(OperandY::fragment(own, 16 * i, ks & 1, lane), fx[j], acc[i][j]);
                }
        }
        wait_vm0();
#pragma unroll
        for (int j = 0; j < 2; j++) {
            __builtin_amdgcn_sched_barrier(0);                // (the weights leave no registers for both at once, nor for the bias but here)
            vec8<T> bias = take8<T>(nullptr, true, 8);
            s16x8 kept;
            if (!YC) bias = *reinterpret_cast<const vec8<T>*>(vectors + lane_col);
            float v[8];
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const u32x2 w = __builtin_amdgcn_permlane16_swap(__float_as_uint(acc[0][j][e]), __float_as_uint(acc[1][j][e]), false, false);
                v[e] = __uint_as_float(w[0]);
                v[4 + e] = __uint_as_float(w[1]);
            }
            const int64_t row = m0 + 16 * j;
            const bool inside = (int)row + lane_row >= first && (int)row + lane_row < now.end;
            way_out<YC, ACT, true>(a, v, bias, early[j], kept);
            if (!inside) continue;
            if (kKeeps && a.slopes != nullptr) *reinterpret_cast<s16x8*>(a.slopes + (row * a.ldz + n0) + at_z) = kept;
            if constexpr (ACT == kWide) put8_wide(static_cast<float*>(a.out) + (row * a.ldo + n0) + at_out, v);
            else *reinterpret_cast<vec8<T>*>(static_cast<T*>(a.out) + (row * a.ldo + n0) + at_out) = rounded<T>(v, 8);
        }
    }
}

// ---------------------------------------------------------------------------------------
// dW: C_e[m][n] = sum over an expert's rows p of X[p][m] Y[p][n].  All rows are taken in chunks of one length, whatever the
// experts' are, so that the workgroups are alike; one that meets the end of an expert's rows writes its sums and goes on with the next expert's.  An expert
// within one chunk is written straight away, the sums of the others meet in a second launch, which also writes the zeros of an expert without rows.  A border of
// two chunks cuts one expert at most: its sums in front of border b (between chunks b and b + 1) are number 2 b, those behind it up to the next border number 2 b + 1.  Sums of
// the rows alone, which are small, have a place for every expert and chunk: c + e, as with every next one either grows.  us: 262144 rows of eight experts, 384 and 1536 channels, 376 to 390 (0.8 PFLOP/s, the matrix units
// at work 33 % of the time; a library's product of one weight 950 to 990), the sums 20; 16384 rows of 2048 and 2048 channels 180 to 203 and 12, where pieces of every
// expert's own took 303 and 70.
// ---------------------------------------------------------------------------------------
template <typename T>
struct GroupedWeights {
    const T *x, *y;
    int64_t ldx, ldy;
    const int32_t* offsets;
    int experts, rows, chunk;             // chunk: rows of one, a multiple of 64
    int M, N, nx, ny, tiles_m, tiles_n;
    T *out, *sums;                        // (experts, M, N), (experts, M) or NULL
    float *part, *part_sum;               // [cut][M][ld_part], [chunk + expert][tiles_n][M]
    int64_t ld_part;
    int wide_out;
};
// Rows first .. end - 1 of an expert; cut: number of their sums, -1 where they are all it has; number: of the rows' sums
template <typename T, int BM, int BN, int WAVES_M, int WAVES_N>
__device__ __forceinline__ void grouped_dw_piece(const GroupedWeights<T>& a, T* lds, int expert, int first, int end, int cut, int number, int m0, int n0, int lane, int wave) {
    constexpr int kWaves = WAVES_M * WAVES_N, WM = BM / WAVES_M, WN = BN / WAVES_N, MT = WM / 16, NT = WN / 16, kTileX = BM * kStep, kTileY = BN * kStep;
    typedef Operand<T, true, BM, kWaves> OperandX;
    typedef Operand<T, true, BN, kWaves> OperandY;
    const int quad = lane >> 4, wm = (wave % WAVES_M) * WM, wn = (wave / WAVES_M) * WN, rows = end - first, steps = (rows + kStep - 1) / kStep;
    OperandX ox;
    OperandY oy;
    ox.init(wave, lane, a.ldx, min(BM, a.nx - m0));
    oy.init(wave, lane, a.ldy, min(BN, a.ny - n0));
    const T *px = a.x + (first * a.ldx + m0), *py = a.y + (first * a.ldy + n0);
    // sums of x's rows: of every tiles_n-th step, the workgroups along a row of tiles take turns; each of the two waves that hold the same rows takes half of them
    static_assert(WAVES_N == 2 && MT % 2 == 0, "halves");
    const bool sums = a.part_sum != nullptr, upper = wave / WAVES_M != 0;
    constexpr int kHalf = MT / 2;
    const int tn = n0 / BN;
    auto request = [&](int s) {
        T* const t = lds + (s & 1) * (kTileX + kTileY);
        ox.request(px, t, wave, lane, rows - s * kStep);
        oy.request(py, t + kTileX, wave, lane, rows - s * kStep);
        px += kStep * a.ldx;
        py += kStep * a.ldy;
    };
    f32x4 acc[NT][MT], sum[kHalf];
#pragma unroll
    for (int i = 0; i < NT; i++)
#pragma unroll
        for (int j = 0; j < MT; j++) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < kHalf; j++) sum[j] = f32x4{0.f, 0.f, 0.f, 0.f};
    vec8<T> ones;
#pragma unroll
    for (int e = 0; e < 8; e++) ones[e] = (T)1.f;
    auto multiply = [&](int s) {
        const T* const tx = lds + (s & 1) * (kTileX + kTileY);
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
            if (sums && s % a.tiles_n == tn) {
#pragma unroll
                for (int j = 0; j < kHalf; j++) sum[j] = product16(ones, upper ? fx[j + kHalf] : fx[j], sum[j]);
            }
        }
    };
    request(0);
    for (int s = 0; s + 1 < steps; s++) {
        wait_vm0();
        __syncthreads();                                      // everyone's copies of this step are there, and everyone is done with the other buffer
        request(s + 1);
        multiply(s);
    }
    wait_vm0();
    __syncthreads();
    multiply(steps - 1);

    const int lane_row = lane & 15, lane_col = 16 * (quad & 1) + 8 * (quad >> 1);
#pragma unroll
    for (int c = 0; c < NT / 2; c++)
#pragma unroll
        for (int j = 0; j < MT; j++) {
            const int m = m0 + wm + 16 * j + lane_row, n = n0 + wn + 32 * c + lane_col, left = a.N - n;
            float v[8];
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const u32x2 w = __builtin_amdgcn_permlane16_swap(__float_as_uint(acc[2 * c][j][e]), __float_as_uint(acc[2 * c + 1][j][e]), false, false);
                v[e] = __uint_as_float(w[0]);
                v[4 + e] = __uint_as_float(w[1]);
            }
            if (m >= a.M || left <= 0) continue;
            if (cut < 0) {
                store8(a.out + ((int64_t)expert * a.M + m) * a.N + n, v, a.wide_out, left);
            } else {
                float* const o = a.part + ((int64_t)cut * a.M + m) * a.ld_part + n;
                *reinterpret_cast<f32x4*>(o) = f32x4{v[0], v[1], v[2], v[3]};
                *reinterpret_cast<f32x4*>(o + 4) = f32x4{v[4], v[5], v[6], v[7]};
            }
        }
    if (sums && quad == 0) {
#pragma unroll
        for (int j = 0; j < kHalf; j++) {
            const int m = m0 + wm + 16 * (j + (upper ? kHalf : 0)) + lane;
            if (m < a.M) a.part_sum[((int64_t)number * a.tiles_n + tn) * a.M + m] = sum[j][0];
        }
    }
}
template <typename T, int BM, int BN, int WAVES_M, int WAVES_N>
__global__ __launch_bounds__(64 * WAVES_M * WAVES_N, 2) void grouped_dw_kernel(const GroupedWeights<T> a) {
    HIP_DYNAMIC_SHARED(char, shared)
    T* const lds = reinterpret_cast<T*>(shared);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int per_chunk = a.tiles_m * a.tiles_n, at = xcd_order((int)blockIdx.x, (int)gridDim.x), chunk = at / per_chunk, tile = at - chunk * per_chunk, tn = tile / a.tiles_m;
    const int m0 = (tile - tn * a.tiles_m) * BM, n0 = tn * BN, chunk0 = chunk * a.chunk, chunk1 = min(a.rows, chunk0 + a.chunk);
    for (int first = chunk0; first < chunk1;) {
        Piece p;
        {                                                     // (looked up each time: where everyone's rows are does not stay in registers)
            Runs runs;
            runs.load(a.offsets, a.experts, a.rows, a.chunk, false, lane);
            p = runs.among(first, chunk1);
        }
        if (p.expert < 0) return;
        const int cut = p.begin < chunk0 ? 2 * chunk - 1 : p.end > chunk1 ? 2 * chunk : -1;
        grouped_dw_piece<T, BM, BN, WAVES_M, WAVES_N>(a, lds, p.expert, max(p.begin, chunk0), min(p.end, chunk1), cut, chunk + p.expert, m0, n0, fresh(lane), wave);
        first = p.end;
        __syncthreads();                                      // (everyone is done with what the next one's copies overwrite)
    }
}
// The sums of the experts that are more than one chunk's, or none's, added up, and those of all experts' rows.  `ways` waves take every so many-th chunk of the
// same places (of four elements): with few places a thread would wait for one chunk after another.
template <typename T>
__global__ __launch_bounds__(256) void grouped_join_kernel(const GroupedWeights<T> a, int ways) {
    __shared__ f32x4 rest[3][64];
    __shared__ int first[LLSA_MAX_EXPERTS], chunks[LLSA_MAX_EXPERTS], cut[LLSA_MAX_EXPERTS], cuts;      // first: chunk
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    {
        Runs runs;
        runs.load(a.offsets, a.experts, a.rows, a.chunk, false, lane);
        if (wave == 0) {
            int n = 0;
#pragma unroll
            for (int i = 0; i < Runs::kLanes; i++) {
                const int e = 64 * i + lane, c0 = runs.begin[i] / a.chunk, c = runs.end[i] > runs.begin[i] ? (runs.end[i] - 1) / a.chunk - c0 + 1 : 0;
                const bool joins = e < a.experts && c != 1;
                const uint64_t all = __ballot(joins);
                if (e < a.experts) {
                    first[e] = c0;
                    chunks[e] = c;
                }
                if (joins) cut[n + __popcll((unsigned long long)(all & (((uint64_t)1 << lane) - 1)))] = e;
                n += __popcll((unsigned long long)all);
            }
            if (lane == 0) cuts = n;
        }
    }
    __syncthreads();
    const int n4 = (int)(a.ld_part / 4), of_one = a.M * n4, at_once = 256 / ways, part = ways == 1 ? 0 : wave, mine = ways == 1 ? tid : lane, blocks = (of_one + at_once - 1) / at_once;
    auto join = [&](f32x4 v) {
        if (ways == 1) return v;
        if (wave > 0) rest[wave - 1][lane] = v;
        __syncthreads();
        if (wave == 0) {
#pragma unroll
            for (int w = 0; w < 3; w++) v += rest[w][lane];
        }
        __syncthreads();
        return v;
    };
    for (int c = 0, turn = 0; c < cuts; c++) {
        const int e = cut[c], from = first[e], count = chunks[e];
        // (each expert's places begin at another workgroup)
        for (int block = (int)((blockIdx.x + gridDim.x - (unsigned)turn) % gridDim.x); block < blocks; block += gridDim.x) {
            const int i = block * at_once + mine, m = min(i, of_one - 1) / n4, n = (min(i, of_one - 1) - m * n4) * 4;
            f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
            for (int s = part; s < count; s += ways) v += *reinterpret_cast<const f32x4*>(a.part + ((int64_t)(2 * (from + s) - (s > 0 ? 1 : 0)) * a.M + m) * a.ld_part + n);
            v = join(v);
            if (part > 0 || i >= of_one) continue;
            T* const out = a.out + ((int64_t)e * a.M + m) * a.N + n;
#pragma unroll
            for (int k = 0; k < 4; k++)
                if (n + k < a.N) out[k] = (T)v[k];
        }
        turn = (turn + blocks) % (int)gridDim.x;
    }
    if (a.part_sum == nullptr) return;
    const int rows = a.experts * a.M;
    for (int i0 = (int)blockIdx.x * at_once; i0 < rows; i0 += (int)gridDim.x * at_once) {
        const int i = min(i0 + mine, rows - 1), e = i / a.M, m = i - e * a.M;
        f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
        for (int s = part; s < chunks[e] * a.tiles_n; s += ways) v[0] += a.part_sum[((int64_t)(first[e] + e) * a.tiles_n + s) * a.M + m];
        v = join(v);
        if (part == 0 && i0 + mine < rows) a.sums[i] = (T)v[0];
    }
}

// ---------------------------------------------------------------------------------------
// Rows of tokens in the order of the places; with weights, multiplied by them (and by the gate of their sample) in fp32.  Bound by memory: 262144 rows of 384, 403 MB, 79 us.
// ---------------------------------------------------------------------------------------
template <typename T>
struct Gather {
    const T *x, *gate;
    T* out;
    const float* weights;
    Order order;
    int64_t ldx, ldo, s_gate, per_sample, first;              // first: workgroup of this launch
    int rows, N, pieces, wide, wide_gate;
};
template <typename T>
__global__ __launch_bounds__(256) void gather_kernel(const Gather<T> a) {
    const int64_t i = (a.first + blockIdx.x) * 256 + threadIdx.x, place = i / a.pieces;
    if (place >= a.rows) return;                              // (places behind the last expert's hold a row as well, whichever: it is not read)
    const int n = (int)(i - place * a.pieces) * 8, left = a.N - n, token = a.order.token((int)place);
    vec8<T> v = take8(a.x + token * a.ldx + n, a.wide, left);
    if (a.weights != nullptr) {
        const float w = a.weights[a.order.slot((int)place)];
        float f[8];
#pragma unroll
        for (int e = 0; e < 8; e++) f[e] = (float)v[e] * w;
        if (a.gate != nullptr) {
            const vec8<T> g = take8(a.gate + token / a.per_sample * a.s_gate + n, a.wide_gate, left);
#pragma unroll
            for (int e = 0; e < 8; e++) f[e] *= (float)g[e];
        }
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = (T)f[e];
    }
#pragma unroll
    for (int e = 0; e < 8; e++)
        if (e >= left) v[e] = (T)0.f;
    *reinterpret_cast<vec8<T>*>(a.out + place * a.ldo + n) = v;
}

// ---------------------------------------------------------------------------------------
// A token's rows added up: out = residual + gate * sum over j of w_j y[places[j]].  Bound by memory: 131072 tokens of 384, two experts each, 106 us with the residual (5.7 TB/s).
// ---------------------------------------------------------------------------------------
template <typename T>
struct Combine {
    const float* y;
    const T *gate, *residual;
    const int32_t* places;
    const float* weights;                 // or NULL: 1
    T* out;
    int64_t ldy, s_gate, ldr, ldo, tokens, per_sample, first;
    int k, rows, N, pieces, wide, wide_side, wide_out;       // pieces: of eight, of a row
};
template <typename T>
__global__ __launch_bounds__(256) void combine_kernel(const Combine<T> a) {
    const int64_t i = (a.first + blockIdx.x) * 256 + threadIdx.x, m = i / a.pieces;
    if (m >= a.tokens) return;
    const int n = (int)(i - m * a.pieces) * 8, left = a.N - n;
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; e++) v[e] = 0.f;
#pragma unroll 4
    for (int j = 0; j < a.k; j++) {
        const int p = a.places[m * a.k + j];
        if ((unsigned)p >= (unsigned)a.rows) continue;        // no expert
        const f32x4 y0 = *reinterpret_cast<const f32x4*>(a.y + p * a.ldy + n), y1 = *reinterpret_cast<const f32x4*>(a.y + p * a.ldy + n + 4);
        const float w = a.weights != nullptr ? a.weights[m * a.k + j] : 1.f;
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] = fmaf(w, y0[e], v[e]), v[4 + e] = fmaf(w, y1[e], v[4 + e]);
    }
    if (a.gate != nullptr) {
        const vec8<T> g = take8(a.gate + m / a.per_sample * a.s_gate + n, a.wide, left);
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] *= (float)g[e];
    }
    if (a.residual != nullptr) {
        const vec8<T> r = take8(a.residual + m * a.ldr + n, a.wide_side, left);
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] += (float)r[e];
    }
    store8(a.out + m * a.ldo + n, v, a.wide_out, left);
}

// dweights[m][j] = gate dout[m] . y of its place, 0 without one; pieces of dgate = sum over a sample's tokens of dout[m] * sum over j of w_j y.  A workgroup
// takes up to `piece` tokens of one sample, each of its waves every fourth, 512 columns at a time.  Bound by memory: dout and y are read once for both, 503 MB in 117 us.
template <typename T>
struct DWeights {
    const T *dout, *gate;
    const float *y, *weights;
    const int32_t* places;
    float *dweights, *part;               // either may be NULL; part: [sample][piece][N]
    int64_t ldd, ldy, s_gate, per_sample, first;
    int k, rows, N, wide, wide_gate, piece, pieces;
};
template <typename T>
__global__ __launch_bounds__(256) void dweights_kernel(const DWeights<T> a) {
    __shared__ float sums[4][512];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, block = (int)(a.first + blockIdx.x), sample = block / a.pieces, piece = block - sample * a.pieces;
    const int64_t t0 = sample * a.per_sample + (int64_t)piece * a.piece, t1 = min((int64_t)(sample + 1) * a.per_sample, t0 + a.piece);
    for (int n0 = 0; n0 < a.N; n0 += 512) {
        const int n = n0 + lane * 8, left = a.N - n;
        const bool inside = left > 0;
        const vec8<T> g = take8(a.gate != nullptr && inside ? a.gate + sample * a.s_gate + n : nullptr, a.wide_gate, left);
        float acc[8];
#pragma unroll
        for (int e = 0; e < 8; e++) acc[e] = 0.f;
        for (int64_t m = t0 + wave; m < t1; m += 4) {
            const vec8<T> dout = take8(inside ? a.dout + m * a.ldd + n : nullptr, a.wide, left);
            float d[8], s[8];
#pragma unroll
            for (int e = 0; e < 8; e++) d[e] = e >= left ? 0.f : (float)dout[e], s[e] = 0.f;
            for (int j0 = 0; j0 < a.k; j0 += 2) {             // (two at a time, their loads in flight together)
                f32x4 y[2][2];
                float w[2];
                bool there[2];
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const int64_t slot = m * a.k + min(j0 + h, a.k - 1);
                    const int p = a.places[slot];
                    there[h] = (unsigned)p < (unsigned)a.rows && j0 + h < a.k;
                    const float* const at = a.y + (there[h] ? p : 0) * a.ldy + (inside ? n : 0);
                    y[h][0] = *reinterpret_cast<const f32x4*>(at);
                    y[h][1] = *reinterpret_cast<const f32x4*>(at + 4);
                    w[h] = a.weights[slot];
                }
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    float dot = 0.f;
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        const float v = e >= left || !there[h] ? 0.f : y[h][e >> 2][e & 3];
                        s[e] = fmaf(there[h] ? w[h] : 0.f, v, s[e]);
                        dot = fmaf(a.gate != nullptr ? d[e] * (e >= left ? 0.f : (float)g[e]) : d[e], v, dot);
                    }
                    if (a.dweights != nullptr && j0 + h < a.k) {
                        dot = octet_sum(dot);
                        dot += across<8>(dot);
                        dot = quad_sum(dot);
                        if (lane == 0) a.dweights[m * a.k + j0 + h] = n0 == 0 ? dot : a.dweights[m * a.k + j0 + h] + dot;
                    }
                }
            }
#pragma unroll
            for (int e = 0; e < 8; e++) acc[e] = fmaf(d[e], s[e], acc[e]);
        }
        if (a.part == nullptr) continue;
#pragma unroll
        for (int e = 0; e < 8; e++) sums[wave][lane * 8 + e] = acc[e];
        __syncthreads();
        for (int c = threadIdx.x; c < 512; c += 256)
            if (n0 + c < a.N) a.part[(int64_t)block * a.N + n0 + c] = (sums[0][c] + sums[1][c]) + (sums[2][c] + sums[3][c]);
        __syncthreads();
    }
}
// The pieces of dgate added up: four waves take every fourth of the same 64 columns' (a thread alone would wait for one after another)
template <typename T>
__global__ __launch_bounds__(256) void expert_gate_kernel(const float* part, T* dgate, int N, int pieces, int groups, int64_t first) {
    __shared__ float rest[3][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, block = (int)(first + blockIdx.x), sample = block / groups, n = (block - sample * groups) * 64 + lane;
    float v = 0.f;
    if (n < N) {
#pragma unroll 8
        for (int p = wave; p < pieces; p += 4) v += part[((int64_t)sample * pieces + p) * N + n];
    }
    if (wave > 0) rest[wave - 1][lane] = v;
    __syncthreads();
    if (wave == 0 && n < N) dgate[(int64_t)sample * N + n] = (T)(v + rest[0][lane] + rest[1][lane] + rest[2][lane]);
}

// dz = dout * slope, of all rows.  Bound by memory.
template <typename T>
__global__ __launch_bounds__(256) void slope_rows_kernel(const T* dout, int64_t ldd, const int16_t* slopes, int64_t lds, T* dz, int64_t ldz, int64_t rows, int N, int pieces, int wide, int64_t first) {
    const int64_t i = (first + blockIdx.x) * 256 + threadIdx.x, m = i / pieces;
    if (m >= rows) return;
    const int n = (int)(i - m * pieces) * 8, left = N - n;
    const vec8<T> d = take8(dout + m * ldd + n, wide, left);
    const s16x8 k = *reinterpret_cast<const s16x8*>(slopes + m * lds + n);
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; e++) v[e] = (float)d[e] * slope_of(k[e]);
    *reinterpret_cast<vec8<T>*>(dz + m * ldz + n) = rounded<T>(v, left);
}

// ---------------------------------------------------------------------------------------
// launches
// ---------------------------------------------------------------------------------------
Order order_of(const int32_t* slots, int k, int64_t tokens, int64_t rows) {
    return Order{slots, k > 1 ? (unsigned)((((uint64_t)1 << 32) + k - 1) / k) : 0u, (int)tokens, (int)rows};
}
// Pieces there can be: the rows' whole ones, and one more for each expert (two more of rows that no expert has)
int64_t pieces_of(int64_t rows, int64_t experts, int64_t size) { return rows / size + std::min<int64_t>(experts + 2, rows); }

// Whether the weights stay in registers: a contraction of five or six steps, columns of which a wave has 32 or none and at most a quarter of the waves none (as
// linear.hip's resident() has it, with both sides' times), rows of out that take 16-byte stores, and tiles enough for each workgroup that they pay for the weights' way
// there, also where it meets the next expert.
bool resident(int64_t rows, int64_t experts, int64_t N, int64_t K, bool wide_out) {
    const int64_t blocks = ceil_div(N, kResColumns);
    if (!wide_out || (K != 5 * kStep && K != 6 * kStep) || N % 32 != 0 || 4 * N < 3 * kResColumns * blocks || blocks > kCus / 8) return false;
    const int64_t slots = kCus / 8 / blocks * 8;
    return rows >= 8 * kResRows * experts && rows >= 8 * kResRows * slots;
}
// Which tiles: few rows for each expert on the average (64 and less are one workgroup's), small tiles while there are few of them for each CU, large ones beyond.
// us, 16384 rows of eight experts 2048 > 2048: 256 x 256 181, 192 x 128 161 to 171; 262144 rows 1536 > 384: 128 x 128 425, 192 x 128 389; back 498 and 428 to 447.
enum GroupedTiles { kFew16, kFew32, kFew64, k64, k128, k192, k256, kResident = LLSA_EXPERTS_RESIDENT };
GroupedTiles grouped_tiles(int64_t rows, int64_t experts, int64_t N, int64_t K, bool dx, bool slope, bool wide_out) {
    const int64_t each = ceil_div(rows, experts);
    if (each <= 64 || (rows / 64 + experts) * ceil_div(N, kFewColumns) <= kCus) return each <= 12 ? kFew16 : each <= 28 ? kFew32 : kFew64;
    if (resident(rows, experts, N, K, wide_out)) return kResident;
    if ((rows / 64 + experts) * ceil_div(N, 64) <= 4 * kCus) return k64;
    // beyond, by linear.hip's lengths of a round, with half a tile more for each expert
    const auto rounds = [&](int bm, int bn, int slots) {
        const double n = ((double)rows / bm + 0.5 * (double)experts) * (double)ceil_div(N, bn) / slots;
        return n > 4 ? n + 0.5 : std::ceil(n);
    };
    const double t128 = rounds(128, 128, 2 * kCus), t192 = (dx ? 1.38 : 1.3) * rounds(192, 128, 2 * kCus), t256 = slope ? 1e30 : (dx ? 1.8 : 1.8 + 220. / (double)K) * rounds(256, 256, kCus);
    return t256 < std::min(t128, t192) ? k256 : t192 < t128 ? k192 : k128;      // (with act'(z) besides, 256 x 256 does not fit the registers)
}
template <typename T, bool YC, bool GATHERED, int BM, int BN, int WAVES_M, int WAVES_N, int ACT>
int launch_grouped_tiles(Grouped<T>& a, hipStream_t stream) {
    a.tiles_n = (int)ceil_div(a.N, BN);
    const int64_t grid = pieces_of(a.rows, a.experts, BM) * a.tiles_n;
    if (grid > kMaxGrid) return fail(-1, "experts: too many rows");
    constexpr int lds = 2 * (BM + BN) * kStep * (int)sizeof(T);
    auto kernel = grouped_kernel<T, YC, GATHERED, BM, BN, WAVES_M, WAVES_N, ACT>;
    if (lds > 64 * 1024) {
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, lds);
        if (e != hipSuccess) return fail(-101, "experts: %s", hipGetErrorString(e));
    }
    hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(64 * WAVES_M * WAVES_N), lds, stream, a);
    return 0;
}
template <typename T, bool YC, int ACT>
int launch_grouped_64(Grouped<T>& a, hipStream_t stream) {
    if constexpr (!YC && ACT != kWide) {
        if (a.order.slots != nullptr) return launch_grouped_tiles<T, YC, true, 64, 64, 2, 2, ACT>(a, stream);
    }
    return launch_grouped_tiles<T, YC, false, 64, 64, 2, 2, ACT>(a, stream);
}
template <typename T, bool YC, int MT, int ACT>
int launch_grouped_few(Grouped<T>& a, hipStream_t stream) {
    a.tiles_n = (int)ceil_div(a.N, kFewColumns);
    a.group = 1;
    const int64_t grid = pieces_of(a.rows, a.experts, 16 * MT) * a.tiles_n;
    if (grid > kMaxGrid) return fail(-1, "experts: too many rows");
    constexpr int lds = kFewWaves * 2 * kFewStage * (int)sizeof(T);                            // (the sums of up to 64 rows fit in it as well)
    hipLaunchKernelGGL(HIP_KERNEL_NAME(grouped_few_kernel<T, YC, MT, ACT>), dim3((unsigned)grid), dim3(64 * kFewWaves), lds, stream, a);
    return 0;
}
template <typename T, bool YC, int ACT, int STEPS>
int launch_grouped_resident(Grouped<T>& a, hipStream_t stream) {
    const int blocks = (int)ceil_div(a.N, kResColumns), slots = kCus / 8 / blocks * 8;
    constexpr int lds = (kResStages * kResRows * kStep * STEPS + kResWaves * kResOwn) * (int)sizeof(T) + 3 * (LLSA_MAX_EXPERTS + 2) * 4;
    auto kernel = grouped_resident_kernel<T, YC, ACT, STEPS>;
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, lds);
    if (e != hipSuccess) return fail(-101, "experts: %s", hipGetErrorString(e));
    hipLaunchKernelGGL(kernel, dim3(kCus), dim3(64 * kResWaves), lds, stream, a, blocks, slots);
    return 0;
}
template <typename T, bool YC, int ACT>
int launch_grouped(Grouped<T>& a, hipStream_t stream) {
    a.group = (int64_t)a.N * a.K <= (1 << 20) ? 1 : 8;        // (rows of tiles that share y while it does not fit the L2 beside them)
    const GroupedTiles t = grouped_tiles(a.rows, a.experts, a.N, a.K, YC, YC && ACT == kBySlope, a.wide_out != 0);
    switch (t) {
        case kFew16: return launch_grouped_few<T, YC, 1, ACT>(a, stream);
        case kFew32: return launch_grouped_few<T, YC, 2, ACT>(a, stream);
        case kFew64: return launch_grouped_few<T, YC, 4, ACT>(a, stream);
        case k64: return launch_grouped_64<T, YC, ACT>(a, stream);
        case k128: return launch_grouped_tiles<T, YC, false, 128, 128, 2, 2, ACT>(a, stream);
        case k192: return launch_grouped_tiles<T, YC, false, 192, 128, 2, 2, ACT>(a, stream);
        case kResident: return a.K == 5 * kStep ? launch_grouped_resident<T, YC, ACT, 5>(a, stream) : launch_grouped_resident<T, YC, ACT, 6>(a, stream);
        default:
            if constexpr (!YC || ACT != kBySlope) return launch_grouped_tiles<T, YC, false, 256, 256, 2, 4, ACT>(a, stream);
            else return fail(-1, "experts: no such tiles");
    }
}
template <typename T>
int launch_forward(Grouped<T>& a, int act, bool wide, hipStream_t stream) {
    if (wide) return launch_grouped<T, false, kWide>(a, stream);
    switch (act) {
        case LLSA_ACT_SILU: return launch_grouped<T, false, LLSA_ACT_SILU>(a, stream);
        case LLSA_ACT_GELU: return launch_grouped<T, false, LLSA_ACT_GELU>(a, stream);
        case LLSA_ACT_GELU_TANH: return launch_grouped<T, false, LLSA_ACT_GELU_TANH>(a, stream);
        default: return launch_grouped<T, false, LLSA_ACT_NONE>(a, stream);
    }
}
template <typename T>
int experts_fwd(const llsa_experts_args& q, hipStream_t stream) {
    Grouped<T> a{};
    a.x = (const T*)q.x; a.ldx = q.ldx; a.y = (const T*)q.w; a.ldy = q.ldw; a.y_expert = (int64_t)q.N * q.ldw;
    a.offsets = q.offsets; a.order = order_of(q.gather_x ? q.order : nullptr, q.k, q.tokens, q.rows);
    a.experts = q.E; a.rows = (int)q.rows; a.N = q.N; a.K = q.K; a.gaps = q.gaps;
    a.bias = (const T*)q.bias;
    a.out = q.out; a.ldo = q.ldo; a.slopes = (int16_t*)q.slopes; a.ldz = q.ldz;
    a.wide = q.N % 8 == 0 && wide8(q.bias, 0);
    a.wide_out = (q.N % 8 == 0 && wide8(q.out, q.ldo)) || q.padded;
    if (int rc = launch_forward<T>(a, q.act, q.wide, stream)) return rc;
    return launch_status("experts_fwd");
}
template <typename T>
int experts_dx(const llsa_experts_args& q, hipStream_t stream) {
    Grouped<T> a{};
    a.x = (const T*)q.dz; a.ldx = q.lddz; a.y = (const T*)q.w; a.ldy = q.ldw; a.y_expert = (int64_t)q.N * q.ldw;
    a.offsets = q.offsets;
    a.experts = q.E; a.rows = (int)q.rows; a.N = q.K; a.ny = (int)pad8(q.K); a.K = q.N; a.gaps = q.gaps;
    a.out = q.out; a.ldo = q.ldo; a.slope_at = (const int16_t*)q.slopes; a.ldz = q.ldz;
    a.wide_out = (q.K % 8 == 0 && wide8(q.out, q.ldo)) || q.padded;
    const int rc = q.wide ? launch_grouped<T, true, kWide>(a, stream) : q.slopes != nullptr ? launch_grouped<T, true, kBySlope>(a, stream) : launch_grouped<T, true, LLSA_ACT_NONE>(a, stream);
    if (rc != 0) return rc;
    return launch_status("experts_dx");
}

// Rows of a chunk.  More chunks fill the chip's workgroups more evenly, and are more sums to write and read (linear.hip's weight_pieces).  4593 rows of 777 and 333
// channels, tiles of 64 x 64: 19.6 us and the sums 10.
int grouped_rows(int64_t N) { return ceil_div(N, 192) * 192 <= ceil_div(N, 128) * 128 ? 192 : 128; }
bool small_tiles(int64_t rows, int64_t N, int64_t K) { return ceil_div(N, 128) * ceil_div(K, 128) * std::max<int64_t>(1, rows / 512) < kCus; }
int64_t chunk_rows(int64_t rows, int64_t N, int64_t K) {
    const bool small = small_tiles(rows, N, K);
    const int64_t bm = small ? 64 : grouped_rows(N), bn = small ? 64 : 128, tiles = ceil_div(N, bm) * ceil_div(K, bn), slots = (small ? 4 : 2) * kCus;
    const double all = 2. * (double)rows * N * K / 0.6e9, sums = 8. * (double)N * K / 4e6;     // us
    int64_t best = 1;
    double least = 0;
    for (int64_t p = 1; p <= std::max<int64_t>(1, rows / 256) && (p - 1) * tiles < 4 * slots; p++) {
        const double n = (double)(tiles * p) / (double)slots, t = all * std::ceil(n) / n + sums * (double)p;
        if (p == 1 || t < least) best = p, least = t;
    }
    return ceil_div(ceil_div(rows, best), kStep) * kStep;
}
int64_t cut_count(int64_t rows, int64_t N, int64_t K) { return 2 * (ceil_div(rows, chunk_rows(rows, N, K)) - 1); }
template <typename T, int BM, int BN>
int launch_grouped_dw(GroupedWeights<T>& a, hipStream_t stream) {
    a.tiles_m = (int)ceil_div(a.M, BM);
    a.tiles_n = (int)ceil_div(a.N, BN);
    const int64_t grid = ceil_div(a.rows, a.chunk) * a.tiles_m * a.tiles_n;
    if (grid > kMaxGrid) return fail(-1, "experts_dw: too many rows");
    constexpr int lds = 2 * (BM + BN) * kStep * (int)sizeof(T);
    auto kernel = grouped_dw_kernel<T, BM, BN, 2, 2>;
    if (lds > 64 * 1024) {
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, lds);
        if (e != hipSuccess) return fail(-101, "experts_dw: %s", hipGetErrorString(e));
    }
    hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(256), lds, stream, a);
    return 0;
}
template <typename T>
int experts_dw(const llsa_experts_args& q, hipStream_t stream) {
    GroupedWeights<T> a{};
    a.x = (const T*)q.dz; a.ldx = q.lddz; a.nx = (int)pad8(q.N);
    a.y = (const T*)q.x; a.ldy = q.ldx; a.ny = (int)pad8(q.K);
    a.offsets = q.offsets;
    a.experts = q.E; a.rows = (int)q.rows; a.M = q.N; a.N = q.K;
    a.chunk = (int)chunk_rows(q.rows, q.N, q.K);
    a.out = (T*)q.out; a.sums = (T*)q.dbias;
    a.ld_part = pad8(q.K);
    a.part = (float*)q.workspace;
    a.part_sum = q.dbias != nullptr ? a.part + cut_count(q.rows, q.N, q.K) * a.M * a.ld_part : nullptr;
    a.wide_out = q.K % 8 == 0 && aligned16(q.out);
    const bool small = small_tiles(q.rows, q.N, q.K);
    const int rc = small ? launch_grouped_dw<T, 64, 64>(a, stream) : grouped_rows(a.M) == 192 ? launch_grouped_dw<T, 192, 128>(a, stream) : launch_grouped_dw<T, 128, 128>(a, stream);
    if (rc != 0) return rc;
    const int64_t places = (int64_t)a.M * (a.ld_part / 4) * std::min<int64_t>(q.E, ceil_div(q.rows, a.chunk) + 1);
    const int ways = ceil_div(q.rows, a.chunk) >= 2 * q.E ? 4 : 1;       // (three chunks of an expert on the average)
    hipLaunchKernelGGL(HIP_KERNEL_NAME(grouped_join_kernel<T>), dim3((unsigned)std::min<int64_t>(8 * kCus, ceil_div(places, 256 / ways))), dim3(256), 0, stream, a, ways);
    return launch_status("experts_dw");
}
template <typename T>
int experts_gather(const llsa_experts_args& q, hipStream_t stream) {
    Gather<T> a{};
    a.x = (const T*)q.x; a.ldx = q.ldx; a.out = (T*)q.out; a.ldo = q.ldo; a.gate = (const T*)q.gate; a.s_gate = q.s_gate; a.per_sample = std::max<int64_t>(1, q.per_sample);
    a.weights = q.weights; a.order = order_of(q.order, q.k, q.tokens, q.rows);
    a.rows = (int)q.rows; a.N = q.N; a.pieces = (int)(pad8(q.N) / 8);
    a.wide = q.N % 8 == 0 && wide8(q.x, q.ldx);
    a.wide_gate = q.N % 8 == 0 && wide8(q.gate, q.s_gate);
    in_launches(ceil_div(q.rows * a.pieces, 256), [&](int64_t first, dim3 grid) {
        a.first = first;
        hipLaunchKernelGGL(HIP_KERNEL_NAME(gather_kernel<T>), grid, dim3(256), 0, stream, a);
    });
    return launch_status("experts_gather");
}
template <typename T>
int experts_combine(const llsa_experts_args& q, hipStream_t stream) {
    Combine<T> a{};
    a.y = (const float*)q.x; a.ldy = q.ldx; a.places = q.places; a.weights = q.weights; a.k = q.k; a.rows = (int)q.rows; a.N = q.N; a.tokens = q.tokens;
    a.per_sample = std::max<int64_t>(1, q.per_sample);
    a.gate = (const T*)q.gate; a.s_gate = q.s_gate; a.residual = (const T*)q.residual; a.ldr = q.ldr;
    a.out = (T*)q.out; a.ldo = q.ldo;
    a.pieces = (int)(pad8(q.N) / 8);
    a.wide = q.N % 8 == 0 && wide8(q.gate, q.s_gate);
    a.wide_side = q.N % 8 == 0 && wide8(q.residual, q.ldr);
    a.wide_out = q.N % 8 == 0 && wide8(q.out, q.ldo);
    in_launches(ceil_div(q.tokens * a.pieces, 256), [&](int64_t first, dim3 grid) {
        a.first = first;
        hipLaunchKernelGGL(HIP_KERNEL_NAME(combine_kernel<T>), grid, dim3(256), 0, stream, a);
    });
    return launch_status("experts_combine");
}
// About 1024 workgroups, each of at least 16 tokens
struct TokenPieces { int count, tokens; };
TokenPieces token_pieces(int64_t tokens, int64_t per_sample) {
    const int64_t samples = tokens / per_sample, want = std::max<int64_t>(1, 4 * kCus / samples), each = std::max<int64_t>(16, ceil_div(per_sample, want));
    return {(int)ceil_div(per_sample, each), (int)each};
}
template <typename T>
int experts_dweights(const llsa_experts_args& q, hipStream_t stream) {
    const int64_t per_sample = q.per_sample > 0 ? q.per_sample : q.tokens, samples = q.tokens / per_sample;
    const TokenPieces p = token_pieces(q.tokens, per_sample);
    DWeights<T> a{};
    a.dout = (const T*)q.dz; a.ldd = q.lddz; a.y = (const float*)q.x; a.ldy = q.ldx; a.gate = (const T*)q.gate; a.s_gate = q.s_gate; a.per_sample = per_sample;
    a.weights = q.weights; a.places = q.places; a.dweights = q.dweights; a.k = q.k; a.rows = (int)q.rows; a.N = q.N;
    a.part = q.dgate != nullptr ? (float*)q.workspace : nullptr;
    a.piece = p.tokens; a.pieces = p.count;
    a.wide = q.N % 8 == 0 && wide8(q.dz, q.lddz);
    a.wide_gate = q.N % 8 == 0 && wide8(q.gate, q.s_gate);
    const int64_t groups = ceil_div(q.N, 64);
    LLSA_REQUIRE(samples * p.count <= kMaxGrid && samples * groups <= kMaxGrid, "experts_dweights: too many samples");
    in_launches(samples * p.count, [&](int64_t first, dim3 grid) {
        a.first = first;
        hipLaunchKernelGGL(HIP_KERNEL_NAME(dweights_kernel<T>), grid, dim3(256), 0, stream, a);
    });
    if (q.dgate != nullptr)
        in_launches(samples * groups, [&](int64_t first, dim3 grid) {
            hipLaunchKernelGGL(HIP_KERNEL_NAME(expert_gate_kernel<T>), grid, dim3(256), 0, stream, a.part, (T*)q.dgate, q.N, p.count, (int)groups, first);
        });
    return launch_status("experts_dweights");
}
template <typename T>
int experts_dz(const llsa_experts_args& q, hipStream_t stream) {
    const int pieces = (int)(pad8(q.N) / 8);
    in_launches(ceil_div(q.rows * pieces, 256), [&](int64_t first, dim3 grid) {
        hipLaunchKernelGGL(HIP_KERNEL_NAME(slope_rows_kernel<T>), grid, dim3(256), 0, stream, (const T*)q.dz, q.lddz, (const int16_t*)q.slopes, q.ldz, (T*)q.out, q.ldo, q.rows, q.N,
                           pieces, q.N % 8 == 0 && wide8(q.dz, q.lddz), first);
    });
    return launch_status("experts_dz");
}

int check_experts(const char* what, const llsa_experts_args* a) {
    LLSA_REQUIRE(a != nullptr, "%s: no arguments", what);
    if (int rc = check_sizes(what, a->rows, a->N, a->K, a->dtype, a->act)) return rc;
    LLSA_REQUIRE(a->E >= 1 && a->E <= LLSA_MAX_EXPERTS && a->rows <= LLSA_MAX_SLOTS && a->tokens >= 0 && a->tokens <= LLSA_MAX_SLOTS, "%s: 1 to %d experts, at most %d rows", what,
                 LLSA_MAX_EXPERTS, LLSA_MAX_SLOTS);
    LLSA_REQUIRE(a->k >= 1 && a->k <= LLSA_MAX_CHOICES, "%s: 1 to %d experts a token", what, LLSA_MAX_CHOICES);
    LLSA_REQUIRE(a->rows == 0 || a->offsets != nullptr, "%s: offsets", what);
    LLSA_REQUIRE(!a->gather_x || a->rows == 0 || (a->order != nullptr && a->tokens > 0), "%s: gathered rows need the order and tokens", what);
    return 0;
}
}  // namespace
}  // namespace llsa

using namespace llsa;

#define BY_TYPE(fn) (a->dtype == LLSA_DTYPE_BF16 ? fn<bf16>(*a, (hipStream_t)stream) : fn<_Float16>(*a, (hipStream_t)stream))

extern "C" int64_t llsa_experts_dw_workspace_bytes(int64_t rows, int E, int N, int K) {
    if (rows <= 0 || E <= 0 || N <= 0 || K <= 0) return 0;
    const int64_t cuts = cut_count(rows, N, K);
    return 4 * N * (cuts * pad8(K) + (cuts / 2 + 1 + E) * ceil_div(K, 64));
}
extern "C" int llsa_experts_form(int64_t rows, int E, int N, int K, int back, int slopes, int stores16) {
    if (rows <= 0 || E <= 0 || N <= 0 || K <= 0) return -1;
    return grouped_tiles(rows, E, N, K, back != 0, back != 0 && slopes != 0, stores16 != 0);
}
extern "C" int llsa_experts_gathers(int64_t rows, int E, int N, int K) { return rows > 0 && E > 0 && N > 0 && K > 0 && grouped_tiles(rows, E, N, K, false, false, true) <= k64; }
extern "C" int llsa_experts_gather(const llsa_experts_args* a, void* stream) {
    if (int rc = check_experts("experts_gather", a)) return rc;
    if (a->rows == 0) return 0;
    LLSA_REQUIRE(a->order != nullptr && a->tokens > 0 && a->x != nullptr && rows16(a->out, a->ldo) && a->ldo >= pad8(a->N), "experts_gather: order, rows 16-byte aligned and padded to a multiple of 8");
    LLSA_REQUIRE(a->gate == nullptr || (a->weights != nullptr && a->per_sample > 0), "experts_gather: a gate goes with the weights");
    return BY_TYPE(experts_gather);
}
extern "C" int llsa_experts_fwd(const llsa_experts_args* a, void* stream) {
    if (int rc = check_experts("experts_fwd", a)) return rc;
    if (a->rows == 0) return 0;
    LLSA_REQUIRE(rows16(a->x, a->ldx) && rows16(a->w, a->ldw) && a->K % 8 == 0 && a->ldx >= a->K && a->ldw >= a->K,
                 "experts_fwd: rows of x and w must be 16-byte aligned and a multiple of 8 long (zeros beyond the end)");
    LLSA_REQUIRE(a->out != nullptr && offsets32(a->ldo) && (!a->padded || (rows16(a->out, a->ldo) && a->ldo >= pad8(a->N))), "experts_fwd: output, padded rows 16-byte aligned and a multiple of 8 long");
    LLSA_REQUIRE(a->slopes == nullptr || (rows16(a->slopes, a->ldz) && a->ldz >= pad8(a->N) && a->act != LLSA_ACT_NONE), "experts_fwd: rows of slopes must be 16-byte aligned and padded to a multiple of 8");
    LLSA_REQUIRE(!a->wide || (a->padded && a->act == LLSA_ACT_NONE && !a->gather_x), "experts_fwd: rows of fp32 are padded, without an activation or gathered rows");
    LLSA_REQUIRE(!a->gather_x || llsa_experts_gathers(a->rows, a->E, a->N, a->K), "experts_fwd: rows of this many tokens have to be gathered beforehand");
    return BY_TYPE(experts_fwd);
}
extern "C" int llsa_experts_dx(const llsa_experts_args* a, void* stream) {
    if (int rc = check_experts("experts_dx", a)) return rc;
    if (a->rows == 0) return 0;
    LLSA_REQUIRE(rows16(a->dz, a->lddz) && rows16(a->w, a->ldw) && a->lddz >= pad8(a->N) && a->ldw >= pad8(a->K), "experts_dx: rows of dz and w must be 16-byte aligned and padded to a multiple of 8");
    LLSA_REQUIRE(a->out != nullptr && offsets32(a->ldo) && (!a->padded || (rows16(a->out, a->ldo) && a->ldo >= pad8(a->K))), "experts_dx: output, padded rows 16-byte aligned and a multiple of 8 long");
    LLSA_REQUIRE(a->slopes == nullptr || (rows16(a->slopes, a->ldz) && a->ldz >= pad8(a->K)), "experts_dx: rows of slopes must be 16-byte aligned and padded to a multiple of 8");
    LLSA_REQUIRE(!a->wide || (a->padded && a->slopes == nullptr), "experts_dx: rows of fp32 are padded, without slopes");
    return BY_TYPE(experts_dx);
}
extern "C" int llsa_experts_dw(const llsa_experts_args* a, void* stream) {
    if (int rc = check_experts("experts_dw", a)) return rc;
    LLSA_REQUIRE(a->rows > 0, "experts_dw: no rows");
    LLSA_REQUIRE((int64_t)a->N * pad8(a->K) < (int64_t(1) << 31) && (int64_t)a->E * a->N < (int64_t(1) << 31), "experts_dw: too many weights of an expert");
    LLSA_REQUIRE(rows16(a->dz, a->lddz) && rows16(a->x, a->ldx) && a->lddz >= pad8(a->N) && a->ldx >= pad8(a->K), "experts_dw: rows of dz and x must be 16-byte aligned and padded to a multiple of 8");
    LLSA_REQUIRE(a->out != nullptr && a->workspace != nullptr && aligned16(a->workspace), "experts_dw: output and workspace (16-byte aligned)");
    return BY_TYPE(experts_dw);
}
extern "C" int llsa_experts_combine(const llsa_experts_args* a, void* stream) {
    if (int rc = check_experts("experts_combine", a)) return rc;
    if (a->tokens == 0) return 0;
    LLSA_REQUIRE(a->places != nullptr && a->out != nullptr && (a->rows == 0 || (rows16(a->x, a->ldx) && a->ldx >= pad8(a->N))), "experts_combine: rows 16-byte aligned and padded to a multiple of 8");
    LLSA_REQUIRE(a->gate == nullptr || (a->per_sample > 0 && a->tokens % a->per_sample == 0), "experts_combine: rows of a sample, whole samples");
    return BY_TYPE(experts_combine);
}
extern "C" int llsa_experts_dweights(const llsa_experts_args* a, void* stream) {
    if (int rc = check_experts("experts_dweights", a)) return rc;
    if (a->tokens == 0) return 0;
    LLSA_REQUIRE(a->places != nullptr && a->weights != nullptr && a->dz != nullptr && rows16(a->x, a->ldx) && a->ldx >= pad8(a->N), "experts_dweights: places, weights, dout, rows of fp32 16-byte aligned and padded to a multiple of 8");
    LLSA_REQUIRE(a->dgate == nullptr || (a->gate != nullptr && a->workspace != nullptr), "experts_dweights: dgate needs the gate and a workspace");
    LLSA_REQUIRE(a->gate == nullptr || (a->per_sample > 0 && a->tokens % a->per_sample == 0), "experts_dweights: rows of a sample, whole samples");
    return BY_TYPE(experts_dweights);
}
extern "C" int64_t llsa_experts_dweights_workspace_bytes(int64_t tokens, int64_t per_sample, int N) {
    if (tokens <= 0 || per_sample <= 0 || N <= 0) return 0;
    return 4 * (tokens / per_sample) * token_pieces(tokens, per_sample).count * N;
}
extern "C" int llsa_experts_dz(const llsa_experts_args* a, void* stream) {
    if (int rc = check_experts("experts_dz", a)) return rc;
    if (a->rows == 0) return 0;
    LLSA_REQUIRE(a->dz != nullptr && rows16(a->slopes, a->ldz) && rows16(a->out, a->ldo) && a->ldz >= pad8(a->N) && a->ldo >= pad8(a->N), "experts_dz: rows of slopes and dz must be 16-byte aligned and padded to a multiple of 8");
    return BY_TYPE(experts_dz);
}
