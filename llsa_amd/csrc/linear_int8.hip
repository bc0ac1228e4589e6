// The linear layer in 8-bit integers, for sampling: weights are kept as whole numbers q_n with a scale s_n for each channel out, the rows of x are
// brought to whole numbers q_m with a scale s_m each, and
//
//     s = max |x| / 127 (fp32),   q = x / s to the nearest whole number (halves to even),   out = residual + gate * act(s_m s_n sum_k q_m q_n + bias)
//
// The sum is exact: 127 * 128 * 131072 < 2^31.  Everything behind it is fp32, rounded once where out is written.  The matrix instructions of 8-bit
// integers take twice the contraction of 16-bit ones in the same time and from the same bytes, so the tiles are those of the 16-bit products, with
// pairs of integers in the place of an element.
#include "product_device.h"

namespace llsa {
namespace {

// ---------------------------------------------------------------------------------------
// rows to whole numbers
// ---------------------------------------------------------------------------------------
constexpr int kPads = 2;
struct Quantize {
    const void* x;
    int8_t* q;
    float* scale;
    int64_t ldx, ldq, rows;
    int K, wide_x, wide_q;                // wide_q: rows of q are 16-byte aligned and filled with zeros to a multiple of 16; else K numbers are written
    int64_t row_blocks, first;            // first: workgroup of this launch
    // rows of integers that are copied beside: to 16-byte aligned rows filled with zeros
    llsa_pad_job pad[kPads];
    int64_t pad_end[kPads];               // pieces of 16, of this and the one before it
};

template <typename T> struct Bits;
template <> struct Bits<bf16> { typedef uint16_t type; static constexpr unsigned kInf = 0x7f80u; };
template <> struct Bits<_Float16> { typedef uint16_t type; static constexpr unsigned kInf = 0x7c00u; };
template <> struct Bits<float> { typedef uint32_t type; static constexpr unsigned kInf = 0x7f800000u; };
template <typename T> using vec8any = __attribute__((ext_vector_type(8))) T;

__device__ __forceinline__ unsigned max_moved(unsigned v, unsigned o) { return v > o ? v : o; }
// the largest of LANES neighbouring lanes (16 or 64), in all of them
template <int LANES>
__device__ __forceinline__ unsigned lanes_max(unsigned v) {
    auto other = [](float x) { return __float_as_uint(x); };
    v = max_moved(v, other(across<1>(__uint_as_float(v))));
    v = max_moved(v, other(across<2>(__uint_as_float(v))));
    v = max_moved(v, other(across<7>(__uint_as_float(v))));
    v = max_moved(v, other(across<8>(__uint_as_float(v))));
    if (LANES > 16) {
        const u32x2 a = __builtin_amdgcn_permlane16_swap(v, v, false, false);
        v = max_moved(a[0], a[1]);
        const u32x2 b = __builtin_amdgcn_permlane32_swap(v, v, false, false);
        v = max_moved(b[0], b[1]);
    }
    return v;
}

// x / s to the nearest whole number, halves to even, of the real quotient: the guess is one off at most, and what is left of x is exact next to s / 2,
// where it is compared (multiples of half a step of s, below s).
__device__ __forceinline__ int nearest(float x, float s, float inverse, float half) {
    float q = __builtin_rintf(x * inverse);
    const float left = fmaf(-q, s, x);
    const bool odd = ((int)q & 1) != 0;
    if (left > half || (left == half && odd)) q += 1.f;
    if (left < -half || (left == -half && odd)) q -= 1.f;
    return (int)fmaxf(-127.f, fminf(127.f, q));
}

// A row's scale, out of its largest value's bits; NaN where that is no number
template <typename T>
__device__ __forceinline__ float step_of(unsigned top) {
    typedef typename Bits<T>::type B;
    const B bits = (B)top;
    T value;
    __builtin_memcpy(&value, &bits, sizeof(B));
    return top < Bits<T>::kInf ? (float)value / 127.f : __uint_as_float(0x7fc00000u);
}
// What a row's elements are divided by.  (Steps near the least numbers are multiplied by a power of two beforehand: their inverse would be an infinity.)
struct Steps { float lift, step, inverse, half; bool zero; };
__device__ __forceinline__ Steps steps_for(float s) {
    Steps t;
    t.zero = !(s > 0.f);
    t.lift = s < 0x1p-60f ? 0x1p80f : 1.f;
    t.step = t.zero ? 1.f : s * t.lift;
    t.inverse = __builtin_amdgcn_rcpf(t.step);
    t.half = 0.5f * t.step;
    return t;
}
template <typename T>
__device__ __forceinline__ int8_t whole_number(T x, const Steps& t) { return (int8_t)(t.zero ? 0 : nearest((float)x * t.lift, t.step, t.inverse, t.half)); }
// Eight of them.  Without the cases that hardly a row has (halves that are exact, steps near the least numbers, no numbers), which are looked at once more:
// with all of nearest() for each, more instructions and nothing else, 131072 rows of 1536 took 136 us instead of 106.
template <typename T>
__device__ __forceinline__ u32x2 whole_numbers(const vec8any<T>& x, const Steps& t) {
    union { int8_t b[8]; u32x2 w; } o;
    bool rare = t.zero || t.lift != 1.f;
#pragma unroll
    for (int e = 0; e < 8; e++) {
        const float v = (float)x[e], q = __builtin_rintf(v * t.inverse), left = fmaf(-q, t.step, v), size = fabsf(left);
        rare |= size == t.half;
        o.b[e] = (int8_t)(int)(size > t.half ? q + __builtin_copysignf(1.f, left) : q);
    }
    if (rare) {
#pragma unroll
        for (int e = 0; e < 8; e++) o.b[e] = whole_number(x[e], t);
    }
    return o.w;
}

// LANES lanes hold a row, PIECES pieces of 8 elements each; longer rows (256 lanes only) are read a second time.  Bound by memory (131072 rows of
// 1536 106 to 128 us by card, 5.7 to 4.7 TB/s) and near what the vector units issue: one instruction for every four cycles of a SIMD, where a kernel of nothing but fp32 fma issues 0.9
// and one of integer operations or conversions 1.6.
template <typename T, int LANES, int PIECES>
__global__ __launch_bounds__(256) void quantize_kernel(const Quantize a) {
    typedef typename Bits<T>::type B;
    constexpr int kRows = 256 / LANES;
    __shared__ unsigned most[4];
    const int tid = threadIdx.x;
    const int64_t block = a.first + blockIdx.x;
    if (block >= a.row_blocks) {                              // (uniform) the copies beside
        int64_t i = (block - a.row_blocks) * 256 + tid;
        int k = 0;
        while (k < kPads && i >= a.pad_end[k]) k++;
        if (k == kPads) return;
        if (k > 0) i -= a.pad_end[k - 1];
        const llsa_pad_job p = a.pad[k];
        const int64_t per = p.ldy / 16, r = i / per;
        const int c = (int)(i - r * per) * 16;
        const int8_t* const x = static_cast<const int8_t*>(p.x) + r * p.ldx;
        typedef __attribute__((ext_vector_type(16))) int8_t i8x16;
        i8x16 v;
#pragma unroll
        for (int e = 0; e < 16; e++) {
            const int8_t t = x[min(c + e, p.cols - 1)];
            v[e] = c + e < p.cols ? t : (int8_t)0;
        }
        *reinterpret_cast<i8x16*>(static_cast<int8_t*>(p.y) + r * p.ldy + c) = v;
        return;
    }
    const int lane = tid % LANES;
    const int64_t row = block * kRows + tid / LANES;
    const bool there = row < a.rows;
    const T* const x = static_cast<const T*>(a.x) + (there ? row : a.rows - 1) * a.ldx;
    const int pieces = (a.K + 7) / 8, runs = LANES < 256 ? 1 : (pieces + LANES * PIECES - 1) / (LANES * PIECES);
    vec8any<T> v[PIECES];
    auto read = [&](int run) {
#pragma unroll
        for (int i = 0; i < PIECES; i++) {
            const int c = ((run * PIECES + i) * LANES + lane) * 8;
            if (a.wide_x && c < a.K) {
                v[i] = *reinterpret_cast<const vec8any<T>*>(x + c);
            } else {
#pragma unroll
                for (int e = 0; e < 8; e++) v[i][e] = c + e < a.K ? x[c + e] : (T)0.f;
            }
        }
    };
    unsigned top = 0;
    for (int run = 0; run < runs; run++) {
        read(run);
#pragma unroll
        for (int i = 0; i < PIECES; i++)
#pragma unroll
            for (int e = 0; e < 8; e++) {
                constexpr unsigned kNoSign = sizeof(B) == 2 ? 0x7fffu : 0x7fffffffu;
                const T t = v[i][e];
                B b;
                __builtin_memcpy(&b, &t, sizeof(B));
                top = max_moved(top, (unsigned)b & kNoSign);  // (as integers: in the order of the sizes, infinities and NaN behind all of them)
            }
    }
    top = lanes_max<(LANES < 64 ? 16 : 64)>(top);
    if (LANES == 256) {
        if ((tid & 63) == 0) most[tid >> 6] = top;
        __syncthreads();
        top = max_moved(max_moved(most[0], most[1]), max_moved(most[2], most[3]));
    }
    if (!there) return;
    const float s = step_of<T>(top);
    if (lane == 0) a.scale[row] = s;
    const Steps st = steps_for(s);
    for (int run = 0; run < runs; run++) {
        if (runs > 1) read(run);
#pragma unroll
        for (int i = 0; i < PIECES; i++) {
            const int c = ((run * PIECES + i) * LANES + lane) * 8;
            union { int8_t b[8]; u32x2 w; } o;
            o.w = whole_numbers<T>(v[i], st);
            int8_t* const q = a.q + row * a.ldq + c;
            if (a.wide_q) {
                if (c < (a.K + 15) / 16 * 16) *reinterpret_cast<u32x2*>(q) = o.w;
            } else {
#pragma unroll
                for (int e = 0; e < 8; e++)
                    if (c + e < a.K) q[e] = o.b[e];
            }
        }
    }
}

// ---------------------------------------------------------------------------------------
// the product
// ---------------------------------------------------------------------------------------
typedef _Float16 Pair;                    // two integers, in the place of an element of the 16-bit products: only moved

__device__ __forceinline__ i32x4 product8(vec8<Pair> a, vec8<Pair> b, i32x4 c) {
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, a), __builtin_bit_cast(i32x4, b), c, 0, 0, 0);
}

template <typename T>
struct Product8 {
    const Pair *x, *y;                    // rows of q_m and q_n
    int64_t ldx, ldy;                     // in pairs
    int M, N, K;                          // K in pairs, a multiple of 8
    int tiles_m, tiles_n, group;
    const float *x_scale, *y_scale;
    const T *bias, *gate, *residual;
    int64_t s_gate, ldr, ldo;
    T* out;
    int per_sample, act;
    int wide, wide_side, wide_out;        // whether 16-byte accesses are allowed: to bias, gate and y_scale; to the residual; to out
};

// Eight values of a row: columns n .. n + 7, `left` of them inside the matrix
template <int WAY, typename T>
__device__ __forceinline__ vec8<T> way_out8(const Product8<T>& a, const int (&sum)[8], float sx, const float (&sy)[8], const vec8<T>& bias, const vec8<T>& gate, const vec8<T>& side) {
    const int act = WAY < 0 ? a.act : WAY;
    vec8<T> o;
#pragma unroll
    for (int e = 0; e < 8; e++) {
        float v = activate(act, (float)sum[e] * sx * sy[e] + (float)bias[e]);       // (the scales one after another: their product may be out of range)
        if (a.gate != nullptr) v *= (float)gate[e];
        if (a.residual != nullptr) v += (float)side[e];
        o[e] = (T)v;
    }
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
template <typename T>
__device__ __forceinline__ void scales8(float (&v)[8], const float* p, bool wide, int n) {
    if (wide) {
        const f32x4 a = *reinterpret_cast<const f32x4*>(p), b = *reinterpret_cast<const f32x4*>(p + 4);
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] = a[e], v[4 + e] = b[e];
    } else {
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = p[min(e, n - 1)];
    }
}
// WAY: the activation, everything in pieces of 16 bytes; -1: any activation and alignment.  8192 x 4096 x 4096 129 to 136 us by card (2.0 to 2.1 POP/s; a library's product without
// scales 129), 131072 x 1536 x 384 with gate and residual 122 to 138 (a library's plain one 159; 168 here in tiles of 256 x 256 before the residual was read ahead and whole
// lines stored).  Bound by the operands' way and the wait for it at every step, as the 16-bit products are: the matrix units work 40 % and 25 % of the time.
template <typename T, int BM, int BN, int WAVES_M, int WAVES_N, int WAY>
__global__ __launch_bounds__(64 * WAVES_M * WAVES_N, 2) void product8_kernel(const Product8<T> a) {
    constexpr int kWaves = WAVES_M * WAVES_N, WM = BM / WAVES_M, WN = BN / WAVES_N, MT = WM / 16, NT = WN / 16, kTileX = BM * kStep, kTileY = BN * kStep;
    typedef Operand<Pair, false, BM, kWaves> OperandX;
    typedef Operand<Pair, false, BN, kWaves> OperandY;
    HIP_DYNAMIC_SHARED(char, shared)
    Pair* const lds = reinterpret_cast<Pair*>(shared);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), quad = lane >> 4;
    const int wm = (wave % WAVES_M) * WM, wn = (wave / WAVES_M) * WN;
    const int at = xcd_order((int)blockIdx.x, (int)gridDim.x), in_group = a.group * a.tiles_n, g = at / in_group, rest = at - g * in_group;
    const int rows_here = min(a.group, a.tiles_m - g * a.group), tn = rest / rows_here, m0 = (g * a.group + rest - tn * rows_here) * BM, n0 = tn * BN;
    OperandX ox;
    OperandY oy;
    ox.init(wave, lane, a.ldx, min(BM, a.M - m0));
    oy.init(wave, lane, a.ldy, min(BN, a.N - n0));
    const Pair *px = a.x + (int64_t)m0 * a.ldx, *py = a.y + (int64_t)n0 * a.ldy;
    int k_left = a.K;
    auto request = [&](int buffer) {
        Pair* const t = lds + buffer * (kTileX + kTileY);
        ox.request(px, t, wave, lane, k_left);
        oy.request(py, t + kTileX, wave, lane, k_left);
        px += kStep;
        py += kStep;
        k_left -= kStep;
    };
    i32x4 acc[NT][MT];
#pragma unroll
    for (int i = 0; i < NT; i++)
#pragma unroll
        for (int j = 0; j < MT; j++) acc[i][j] = i32x4{0, 0, 0, 0};
    auto multiply = [&](int buffer) {
        const Pair* const tx = lds + buffer * (kTileX + kTileY);
        const Pair* const ty = tx + kTileX;
#pragma unroll
        for (int ks = 0; ks < kStep / 32; ks++) {
            vec8<Pair> fx[MT], fy[NT];
#pragma unroll
            for (int j = 0; j < MT; j++) fx[j] = OperandX::fragment(tx, wm + 16 * j, ks, lane);
#pragma unroll
            for (int i = 0; i < NT; i++) fy[i] = OperandY::fragment(ty, wn + 16 * i, ks, lane);
#pragma unroll
            for (int i = 0; i < NT; i++)
#pragma unroll
                for (int j = 0; j < MT; j++) acc[i][j] = product8(fy[i], fx[j], acc[i][j]);
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

    // Lane l holds columns 4 (l/16) .. +3 of every 16, of row l%16; swapped between sixteens of lanes, a pair of tiles gives it eight neighbouring ones, and
    // where the tile is whole two pairs leave as whole lines (linear.hip).  The residual is on its way during the last step's products.
    const int lane_row = lane & 15, lane_col = 16 * (quad & 1) + 8 * (quad >> 1), row0 = m0 + wm, col0 = n0 + wn, rows_left = a.M - row0 - lane_row, cols_left = a.N - col0 - lane_col;
    const unsigned at_out = (unsigned)(lane_row * a.ldo) + lane_col, at_side = (unsigned)(lane_row * a.ldr) + lane_col;
    constexpr int kPair = NT % 4 == 0 ? 2 : 1;
    const bool whole = kPair == 2 && WAY >= 0 && m0 + BM <= a.M && n0 + BN <= a.N;
    constexpr bool kAhead = BM * BN < 256 * 256;              // (256 x 256 leave no registers for it: row by row)
    constexpr int kEarly = kAhead ? MT : 1;
    vec8<T> early[kPair][kEarly];
    auto read_side = [&](int p0, int first) {
        if (WAY < 0 || a.residual == nullptr) return;
        if constexpr (kPair == 2) {
            if (whole) {
#pragma unroll
                for (int i = 0, j = first; i < kEarly; i++, j++)
                    request_lines(early[0][i], early[1][i], a.residual + ((int64_t)(row0 + 16 * j) * a.ldr + (col0 + 32 * p0)), at_side, (unsigned)(8 * a.ldr), lane);
                return;
            }
        }
#pragma unroll
        for (int i = 0, j = first; i < kEarly; i++, j++)
#pragma unroll
            for (int h = 0; h < kPair; h++)
                if (16 * j < rows_left && 32 * (p0 + h) < cols_left)
                    early[h][i] = *reinterpret_cast<const vec8<T>*>(a.residual + ((int64_t)(row0 + 16 * j) * a.ldr + (col0 + 32 * (p0 + h))) + at_side);
    };
    if (kAhead) read_side(0, 0);
    float sx[MT];
#pragma unroll
    for (int j = 0; j < MT; j++) sx[j] = a.x_scale[min(row0 + lane_row + 16 * j, a.M - 1)];
    multiply((steps - 1) & 1);
    const int sample = a.gate != nullptr ? m0 / a.per_sample : 0;
    const bool one_sample = a.gate != nullptr && min(m0 + BM, a.M) <= (int64_t)(sample + 1) * a.per_sample;
#pragma unroll
    for (int p0 = 0; p0 < NT / 2; p0 += kPair) {
        vec8<T> bias[kPair], gate[kPair];
        float sy[kPair][8];
#pragma unroll
        for (int h = 0; h < kPair; h++) {
            const int n = col0 + lane_col + 32 * (p0 + h), left = cols_left - 32 * (p0 + h);
            if (left > 0) scales8<T>(sy[h], a.y_scale + n, a.wide, left);
            bias[h] = take8(a.bias != nullptr && left > 0 ? a.bias + n : nullptr, a.wide, left);
            gate[h] = take8(one_sample && left > 0 ? a.gate + sample * a.s_gate + n : nullptr, a.wide, left);
        }
#pragma unroll
        for (int j = 0; j < MT; j++) {
            const int64_t row = row0 + 16 * j;
            vec8<T> o[kPair];
            const int i = kAhead ? j : 0;
            if (!kAhead) read_side(p0, j);
            if constexpr (kPair == 2) {
                if (whole && a.residual != nullptr) arrange_lines<T>(early[0][i], early[1][i], lane);
            }
#pragma unroll
            for (int h = 0; h < kPair; h++) {
                const int p = p0 + h, col = col0 + 32 * p, left = cols_left - 32 * p;
                int v[8];
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const u32x2 w = __builtin_amdgcn_permlane16_swap((unsigned)acc[2 * p][j][e], (unsigned)acc[2 * p + 1][j][e], false, false);
                    v[e] = (int)w[0];
                    v[4 + e] = (int)w[1];
                }
                if (16 * j >= rows_left || left <= 0) continue;      // (not before the swap, which takes all lanes)
                if (a.gate != nullptr && !one_sample) gate[h] = take8(a.gate + (int)(row + lane_row) / a.per_sample * a.s_gate + col + lane_col, a.wide, left);
                if (WAY < 0 && a.residual != nullptr) early[h][i] = take8(a.residual + (row + lane_row) * a.ldr + col + lane_col, a.wide_side && left >= 8, left);
                o[h] = way_out8<WAY>(a, v, sx[j], sy[h], bias[h], gate[h], early[h][i]);
                if (!whole) put8(a.out + (row * a.ldo + col) + at_out, o[h], WAY >= 0 || (a.wide_out && left >= 8), left);
            }
            if constexpr (kPair == 2) {
                if (whole) store_lines(a.out + (row * a.ldo + (col0 + 32 * p0)), at_out, (unsigned)(8 * a.ldo), o[0], o[1], lane);
            }
            __builtin_amdgcn_sched_barrier(0);                // (rows one after another: all at once do not fit the registers)
        }
        if (kAhead && p0 + kPair < NT / 2) read_side(p0 + kPair, 0);
    }
}

// Few rows: a workgroup takes 32 columns of up to 64 rows, its eight waves an eighth of the contraction each, through two stages of LDS of their own; the
// sums meet at the end.
constexpr int kFewWaves = 8, kFewColumns = 32, kFewStage = kFewColumns * kStep, kFewRows = 64;
template <typename T, int MT, int WAY>
__global__ __launch_bounds__(64 * kFewWaves, 2) void few_rows8_kernel(const Product8<T> a) {
    typedef Operand<Pair, false, kFewColumns, 1> OperandY;
    HIP_DYNAMIC_SHARED(char, shared)
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), quad = lane >> 4;
    Pair* const stage = reinterpret_cast<Pair*>(shared) + wave * 2 * kFewStage;
    const int n0 = (int)blockIdx.x * kFewColumns, row0 = (int)blockIdx.y * 16 * MT;
    const int all = (a.K + kStep - 1) / kStep, each = (all + kFewWaves - 1) / kFewWaves, first = min(all, wave * each), steps = min(all - first, each);
    OperandY oy;
    oy.init(0, lane, a.ldy, min(kFewColumns, a.N - n0));
    const int k0 = first * kStep;
    const Pair* const py = a.y + (int64_t)n0 * a.ldy + k0;
    const Pair* px[MT];
#pragma unroll
    for (int j = 0; j < MT; j++) px[j] = a.x + min(row0 + 16 * j + (lane & 15), a.M - 1) * a.ldx;
    i32x4 acc[2][MT];
#pragma unroll
    for (int i = 0; i < 2; i++)
#pragma unroll
        for (int j = 0; j < MT; j++) acc[i][j] = i32x4{0, 0, 0, 0};
    vec8<Pair> next[MT][2];
    auto request = [&](int s) {
        const int k = k0 + s * kStep;
        oy.request(py + s * kStep, stage + (s & 1) * kFewStage, 0, lane, a.K - k);
#pragma unroll
        for (int j = 0; j < MT; j++)
#pragma unroll
            for (int ks = 0; ks < 2; ks++) {
                const int at = k + 32 * ks + 8 * quad;
                next[j][ks] = *reinterpret_cast<const vec8<Pair>*>(at < a.K ? px[j] + at : reinterpret_cast<const Pair*>(kZeros));
            }
    };
    if (steps > 0) request(0);
    for (int s = 0; s < steps; s++) {
        vec8<Pair> fx[MT][2];
        wave_waits_for_copies();
#pragma unroll
        for (int j = 0; j < MT; j++)
#pragma unroll
            for (int ks = 0; ks < 2; ks++) fx[j][ks] = next[j][ks];
        if (s + 1 < steps) request(s + 1);
        const Pair* const ty = stage + (s & 1) * kFewStage;
#pragma unroll
        for (int ks = 0; ks < 2; ks++)
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const vec8<Pair> fy = OperandY::fragment(ty, 16 * i, ks, lane);
#pragma unroll
                for (int j = 0; j < MT; j++) acc[i][j] = product8(fy, fx[j][ks], acc[i][j]);
            }
        wave_waits_for_reads();                               // (done, before the next request but one writes there)
    }
    __syncthreads();
    i32x4* const sums = reinterpret_cast<i32x4*>(shared);     // [wave][tile][half][lane]
#pragma unroll
    for (int j = 0; j < MT; j++)
#pragma unroll
        for (int i = 0; i < 2; i++) sums[((wave * MT + j) * 2 + i) * 64 + lane] = acc[i][j];
    __syncthreads();
    if (wave >= MT) return;
    i32x4 t[2];
#pragma unroll
    for (int i = 0; i < 2; i++) {
        t[i] = sums[(wave * 2 + i) * 64 + lane];
#pragma unroll
        for (int w = 1; w < kFewWaves; w++) t[i] += sums[((w * MT + wave) * 2 + i) * 64 + lane];
    }
    int v[8];
#pragma unroll
    for (int e = 0; e < 4; e++) {
        const u32x2 w = __builtin_amdgcn_permlane16_swap((unsigned)t[0][e], (unsigned)t[1][e], false, false);
        v[e] = (int)w[0];
        v[4 + e] = (int)w[1];
    }
    const int n = n0 + 16 * (quad & 1) + 8 * (quad >> 1), m = row0 + 16 * wave + (lane & 15), left = a.N - n;
    if (m >= a.M || left <= 0) return;
    float sy[8];
    scales8<T>(sy, a.y_scale + n, a.wide, left);
    const vec8<T> bias = take8(a.bias != nullptr ? a.bias + n : nullptr, a.wide, left);
    const vec8<T> gate = take8(a.gate != nullptr ? a.gate + m / a.per_sample * a.s_gate + n : nullptr, a.wide, left);
    const vec8<T> side = take8(a.residual != nullptr ? a.residual + (int64_t)m * a.ldr + n : nullptr, WAY >= 0 || (a.wide_side && left >= 8), left);
    put8(a.out + (int64_t)m * a.ldo + n, way_out8<WAY>(a, v, a.x_scale[m], sy, bias, gate, side), WAY >= 0 || (a.wide_out && left >= 8), left);
}

// Up to sixteen rows of 16-bit elements, single tokens of a batch: brought to whole numbers here, by every workgroup for itself, in one launch with the product (8 rows
// 384 > 2304: 6.2 us, in two launches 10.3).
// Each of the eight waves finds the largest values of two rows, and the rows' steps meet in LDS; the fragments are made of 32 bytes of a row as they are read.
template <typename T, int WAY>
__global__ __launch_bounds__(64 * kFewWaves, 2) void few_rows_direct8_kernel(const Product8<T> a, const T* rows, int64_t ld) {
    typedef Operand<Pair, false, kFewColumns, 1> OperandY;
    __shared__ float steps_of[16];
    HIP_DYNAMIC_SHARED(char, shared)
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), quad = lane >> 4, lane_row = lane & 15;
    Pair* const stage = reinterpret_cast<Pair*>(shared) + wave * 2 * kFewStage;
    const int n0 = (int)blockIdx.x * kFewColumns;
    const int all = (a.K + kStep - 1) / kStep, each = (all + kFewWaves - 1) / kFewWaves, first = min(all, wave * each), steps = min(all - first, each);
    OperandY oy;
    oy.init(0, lane, a.ldy, min(kFewColumns, a.N - n0));
    const int k0 = first * kStep;                             // in pairs
    const Pair* const py = a.y + (int64_t)n0 * a.ldy + k0;
    auto request = [&](int s) { oy.request(py + s * kStep, stage + (s & 1) * kFewStage, 0, lane, a.K - k0 - s * kStep); };
    if (steps > 0) request(0);                                // (weights on their way meanwhile)
#pragma unroll
    for (int h = 0; h < 2; h++) {
        const int r = 2 * wave + h;
        const T* const x = rows + min(r, a.M - 1) * ld;
        unsigned top = 0;
        for (int c = lane * 8; c < 2 * a.K; c += 512) {
            const vec8<T> v = *reinterpret_cast<const vec8<T>*>(x + c);
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const T t = v[e];
                uint16_t b;
                __builtin_memcpy(&b, &t, 2);
                top = max_moved(top, b & 0x7fffu);
            }
        }
        top = lanes_max<64>(top);
        if (lane == 0) steps_of[r] = step_of<T>(top);
    }
    __syncthreads();
    const float own = steps_of[lane_row];
    const Steps st = steps_for(own);
    const T* const px = rows + min(lane_row, a.M - 1) * ld;
    i32x4 acc[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
    for (int s = 0; s < steps; s++) {
        vec8<T> raw[2][2];
#pragma unroll
        for (int ks = 0; ks < 2; ks++) {
            const int at = 2 * (k0 + s * kStep + 32 * ks + 8 * quad);         // (a multiple of 16 elements, as K is)
#pragma unroll
            for (int h = 0; h < 2; h++) raw[ks][h] = take8(at < 2 * a.K ? px + at + 8 * h : nullptr, true, 8);
        }
        wave_waits_for_copies();
        if (s + 1 < steps) request(s + 1);
        const Pair* const ty = stage + (s & 1) * kFewStage;
#pragma unroll
        for (int ks = 0; ks < 2; ks++) {
            const u32x2 lo = whole_numbers<T>(raw[ks][0], st), hi = whole_numbers<T>(raw[ks][1], st);
            const vec8<Pair> fx = __builtin_bit_cast(vec8<Pair>, u32x4{lo[0], lo[1], hi[0], hi[1]});
#pragma unroll
            for (int i = 0; i < 2; i++) acc[i] = product8(OperandY::fragment(ty, 16 * i, ks, lane), fx, acc[i]);
        }
        wave_waits_for_reads();
    }
    __syncthreads();
    i32x4* const sums = reinterpret_cast<i32x4*>(shared);     // [wave][half][lane]
#pragma unroll
    for (int i = 0; i < 2; i++) sums[(wave * 2 + i) * 64 + lane] = acc[i];
    __syncthreads();
    if (wave > 0) return;
    i32x4 t[2];
#pragma unroll
    for (int i = 0; i < 2; i++) {
        t[i] = sums[i * 64 + lane];
#pragma unroll
        for (int w = 1; w < kFewWaves; w++) t[i] += sums[(w * 2 + i) * 64 + lane];
    }
    int v[8];
#pragma unroll
    for (int e = 0; e < 4; e++) {
        const u32x2 w = __builtin_amdgcn_permlane16_swap((unsigned)t[0][e], (unsigned)t[1][e], false, false);
        v[e] = (int)w[0];
        v[4 + e] = (int)w[1];
    }
    const int n = n0 + 16 * (quad & 1) + 8 * (quad >> 1), m = lane_row, left = a.N - n;
    if (m >= a.M || left <= 0) return;
    float sy[8];
    scales8<T>(sy, a.y_scale + n, a.wide, left);
    const vec8<T> bias = take8(a.bias != nullptr ? a.bias + n : nullptr, a.wide, left);
    const vec8<T> gate = take8(a.gate != nullptr ? a.gate + m / a.per_sample * a.s_gate + n : nullptr, a.wide, left);
    const vec8<T> side = take8(a.residual != nullptr ? a.residual + (int64_t)m * a.ldr + n : nullptr, WAY >= 0 || (a.wide_side && left >= 8), left);
    put8(a.out + (int64_t)m * a.ldo + n, way_out8<WAY>(a, v, own, sy, bias, gate, side), WAY >= 0 || (a.wide_out && left >= 8), left);
}

// ---------------------------------------------------------------------------------------
// launches
// ---------------------------------------------------------------------------------------
template <typename T, int LANES, int PIECES>
void launch_quantize(Quantize& a, int64_t pads, hipStream_t stream) {
    a.row_blocks = ceil_div(a.rows, 256 / LANES);
    in_launches(a.row_blocks + ceil_div(pads, 256), [&](int64_t first, dim3 grid) {
        a.first = first;
        hipLaunchKernelGGL(HIP_KERNEL_NAME(quantize_kernel<T, LANES, PIECES>), grid, dim3(256), 0, stream, a);
    });
}
template <typename T>
void quantize(Quantize& a, int64_t pads, hipStream_t stream) {
    const int64_t pieces = ceil_div(a.K, 8);
    if (pieces <= 16) launch_quantize<T, 16, 1>(a, pads, stream);
    else if (pieces <= 32) launch_quantize<T, 16, 2>(a, pads, stream);
    else if (pieces <= 48) launch_quantize<T, 16, 3>(a, pads, stream);
    else if (pieces <= 64) launch_quantize<T, 64, 1>(a, pads, stream);
    else if (pieces <= 128) launch_quantize<T, 64, 2>(a, pads, stream);
    else if (pieces <= 192) launch_quantize<T, 64, 3>(a, pads, stream);
    else launch_quantize<T, 256, 2>(a, pads, stream);
}

template <typename T, int BM, int BN, int WAVES_M, int WAVES_N, int WAY>
int launch_tiles8(Product8<T>& a, hipStream_t stream) {
    const int64_t tm = ceil_div(a.M, BM), tn = ceil_div(a.N, BN);
    if (tm * tn > kMaxGrid) return fail(-1, "linear_int8: too many rows");
    a.tiles_m = (int)tm;
    a.tiles_n = (int)tn;
    constexpr int lds = 2 * (BM + BN) * kStep * (int)sizeof(Pair);
    auto kernel = product8_kernel<T, BM, BN, WAVES_M, WAVES_N, WAY>;
    if (lds > 64 * 1024) {
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, lds);
        if (e != hipSuccess) return fail(-101, "linear_int8: %s", hipGetErrorString(e));
    }
    hipLaunchKernelGGL(kernel, dim3((unsigned)(tm * tn)), dim3(64 * WAVES_M * WAVES_N), lds, stream, a);
    return 0;
}
template <typename T, int WAY>
int launch_few8(const Product8<T>& a, hipStream_t stream) {
    const dim3 grid((unsigned)ceil_div(a.N, kFewColumns), (unsigned)ceil_div(a.M, kFewRows)), block(64 * kFewWaves);
    constexpr int lds = kFewWaves * 2 * kFewStage * (int)sizeof(Pair);
    if (a.M <= 16) hipLaunchKernelGGL(HIP_KERNEL_NAME(few_rows8_kernel<T, 1, WAY>), grid, block, lds, stream, a);
    else if (a.M <= 32) hipLaunchKernelGGL(HIP_KERNEL_NAME(few_rows8_kernel<T, 2, WAY>), grid, block, lds, stream, a);
    else hipLaunchKernelGGL(HIP_KERNEL_NAME(few_rows8_kernel<T, 4, WAY>), grid, block, lds, stream, a);
    return 0;
}
template <typename T, int WAY>
int launch_way8(Product8<T>& a, const void* rows, int64_t ld, hipStream_t stream) {
    if (rows != nullptr) {
        constexpr int lds = kFewWaves * 2 * kFewStage * (int)sizeof(Pair);
        hipLaunchKernelGGL(HIP_KERNEL_NAME(few_rows_direct8_kernel<T, WAY>), dim3((unsigned)ceil_div(a.N, kFewColumns)), dim3(64 * kFewWaves), lds, stream, a, (const T*)rows, ld);
        return 0;
    }
    a.group = (int64_t)a.N * a.K <= (1 << 20) ? 1 : 8;        // (rows of tiles that share y while it does not fit the L2 beside them)
    if (a.M <= kFewRows || ceil_div(a.M, kFewRows) * ceil_div(a.N, kFewColumns) <= kCus) return launch_few8<T, WAY>(a, stream);
    if (ceil_div(a.M, 64) * ceil_div(a.N, 64) <= 4 * kCus) return launch_tiles8<T, 64, 64, 2, 2, WAY>(a, stream);
    // (pairs of integers are half as many elements: linear.hip's lengths of a round, the way out weighing twice)
    const auto rounds = [&](int bm, int bn, int slots) {
        const double n = (double)(ceil_div(a.M, bm) * ceil_div(a.N, bn)) / slots;
        return n > 4 ? n + 0.5 : std::ceil(n);
    };
    const double t128 = rounds(128, 128, 2 * kCus), t192 = 1.3 * rounds(192, 128, 2 * kCus), t256 = (1.8 + 220. / (double)a.K) * rounds(256, 256, kCus);
    if (t256 < std::min(t128, t192)) return launch_tiles8<T, 256, 256, 2, 4, WAY>(a, stream);
    if (t192 < t128) return launch_tiles8<T, 192, 128, 2, 2, WAY>(a, stream);
    return launch_tiles8<T, 128, 128, 2, 2, WAY>(a, stream);
}
template <typename T>
int linear_int8(const llsa_int8_args& q, hipStream_t stream) {
    Product8<T> a{};
    a.x = (const Pair*)q.q; a.ldx = q.ldq / 2; a.x_scale = q.q_scale;
    a.y = (const Pair*)q.w; a.ldy = q.ldw / 2; a.y_scale = q.w_scale;
    a.M = (int)q.M; a.N = q.N; a.K = (q.K + 15) / 16 * 8;
    a.bias = (const T*)q.bias; a.gate = (const T*)q.gate; a.s_gate = q.s_gate; a.per_sample = (int)std::max<int64_t>(1, q.per_sample);
    a.residual = (const T*)q.residual; a.ldr = q.ldr; a.out = (T*)q.out; a.ldo = q.ldo; a.act = q.act;
    a.wide = q.N % 8 == 0 && wide8(q.bias, 0) && wide8(q.gate, q.s_gate) && aligned16(q.w_scale);
    a.wide_side = wide8(q.residual, q.ldr);
    a.wide_out = wide8(q.out, q.ldo);
    int rc;
    if (!a.wide || !a.wide_side || !a.wide_out) rc = launch_way8<T, -1>(a, q.x, q.ldx, stream);
    else if (a.act == LLSA_ACT_SILU) rc = launch_way8<T, LLSA_ACT_SILU>(a, q.x, q.ldx, stream);
    else if (a.act == LLSA_ACT_GELU) rc = launch_way8<T, LLSA_ACT_GELU>(a, q.x, q.ldx, stream);
    else if (a.act == LLSA_ACT_GELU_TANH) rc = launch_way8<T, LLSA_ACT_GELU_TANH>(a, q.x, q.ldx, stream);
    else rc = launch_way8<T, LLSA_ACT_NONE>(a, q.x, q.ldx, stream);
    return rc != 0 ? rc : launch_status("linear_int8");
}
bool rows8(const void* p, int64_t ld, int64_t K) { return p != nullptr && aligned16(p) && ld % 16 == 0 && ld >= K && ld <= kMaxLd; }
}  // namespace
}  // namespace llsa

using namespace llsa;

extern "C" int llsa_quantize_rows(const llsa_quantize_args* a, void* stream) {
    LLSA_REQUIRE(a != nullptr, "quantize_rows: no arguments");
    LLSA_REQUIRE(a->rows >= 0 && a->rows <= kMaxRows && a->K > 0 && a->K < (1 << 23), "quantize_rows: bad sizes (%lld rows of %d)", (long long)a->rows, a->K);
    LLSA_REQUIRE(a->dtype == LLSA_DTYPE_BF16 || a->dtype == LLSA_DTYPE_F16 || a->dtype == LLSA_DTYPE_F32, "quantize_rows: bf16, fp16 or fp32 only");
    LLSA_REQUIRE(a->rows == 0 || (a->x != nullptr && a->q != nullptr && a->scale != nullptr), "quantize_rows: x, q and scales");
    LLSA_REQUIRE(!a->padded || rows8(a->q, a->ldq, (a->K + 15) / 16 * 16), "quantize_rows: padded rows of q must be 16-byte aligned and a multiple of 16 long");
    LLSA_REQUIRE(a->pads >= 0 && a->pads <= kPads, "quantize_rows: at most %d copies", kPads);
    Quantize q{};
    q.x = a->x; q.ldx = a->ldx; q.q = (int8_t*)a->q; q.ldq = a->ldq; q.scale = a->scale; q.rows = a->rows; q.K = a->K;
    const int per = a->dtype == LLSA_DTYPE_F32 ? 4 : 8;
    q.wide_x = a->K % 8 == 0 && aligned16(a->x) && a->ldx % per == 0;
    q.wide_q = a->padded;
    int64_t pads = 0;
    for (int i = 0; i < kPads; i++) {
        if (i < a->pads) {
            const llsa_pad_job& p = a->pad[i];
            LLSA_REQUIRE(p.rows >= 0 && p.cols > 0 && p.ldy >= p.cols && rows8(p.y, p.ldy, p.cols) && (p.rows == 0 || p.x != nullptr), "quantize_rows: bad copies");
            q.pad[i] = p;
            pads += p.rows * (p.ldy / 16);
        }
        q.pad_end[i] = pads;
    }
    if (q.rows == 0 && pads == 0) return 0;
    if (a->dtype == LLSA_DTYPE_BF16) quantize<bf16>(q, pads, (hipStream_t)stream);
    else if (a->dtype == LLSA_DTYPE_F16) quantize<_Float16>(q, pads, (hipStream_t)stream);
    else quantize<float>(q, pads, (hipStream_t)stream);
    return launch_status("quantize_rows");
}
extern "C" int llsa_linear_int8(const llsa_int8_args* a, void* stream) {
    LLSA_REQUIRE(a != nullptr, "linear_int8: no arguments");
    if (int rc = check_sizes("linear_int8", a->M, a->N, a->K, a->dtype, a->act)) return rc;
    LLSA_REQUIRE(a->K <= LLSA_INT8_MAX_K, "linear_int8: at most %d channels in (sums of 32 bits)", LLSA_INT8_MAX_K);
    if (a->M == 0) return 0;
    const int64_t K = (a->K + 15) / 16 * 16;
    LLSA_REQUIRE(rows8(a->w, a->ldw, K) && (a->x != nullptr || rows8(a->q, a->ldq, K)), "linear_int8: rows of q and w must be 16-byte aligned and filled with zeros to a multiple of 16");
    LLSA_REQUIRE(a->x == nullptr || (a->M <= LLSA_INT8_DIRECT_ROWS && a->K % 16 == 0 && rows16(a->x, a->ldx) && a->ldx >= a->K),
                 "linear_int8: at most %d rows of x itself, 16-byte aligned and a multiple of 16 long", LLSA_INT8_DIRECT_ROWS);
    LLSA_REQUIRE((a->x != nullptr || a->q_scale != nullptr) && a->w_scale != nullptr && a->out != nullptr, "linear_int8: scales and output");
    LLSA_REQUIRE(a->gate == nullptr || (a->per_sample > 0 && a->M % a->per_sample == 0), "linear_int8: rows of a sample, whole samples");
    LLSA_REQUIRE(offsets32(a->ldo) && (a->residual == nullptr || offsets32(a->ldr)), "linear_int8: rows of out and residual at most %lld apart", (long long)kMaxLd);
    return a->dtype == LLSA_DTYPE_BF16 ? linear_int8<bf16>(*a, (hipStream_t)stream) : linear_int8<_Float16>(*a, (hipStream_t)stream);
}
