// What the kernels of the linear layers share (products of a long matrix of rows with a weight matrix): 16-bit types and their matrix instructions,
// activations, operands in LDS, accesses of eight elements and of whole lines, and the checks of their entry points.
#pragma once
#include <algorithm>
#include <cmath>
#include <type_traits>

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

// Waits of a single wave that nothing is moved across: for its copies into LDS (vmcnt(0)), for its reads of LDS (lgkmcnt(0))
__device__ __forceinline__ void wave_waits_for_copies() {
    asm volatile("" ::: "memory");
    wait_vm0();
    __builtin_amdgcn_wave_barrier();
    asm volatile("" ::: "memory");
}
__device__ __forceinline__ void wave_waits_for_reads() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0xC07F);
    asm volatile("" ::: "memory");
}

// ---------------------------------------------------------------------------------------
// activations, in fp32.  Written with the logistic function: 0.5 (1 + tanh u) = s(2u), which saturates to 0 and 1 without an
// overflow.  The derivatives are taken at z held to +-128, where they are 0 and 1 in fp32 (SiLU's 128 e^-128 is below its smallest number), so that a large z
// does not multiply an infinite inner derivative by zero.
// ---------------------------------------------------------------------------------------
constexpr float kGeluC = 0.7978845608028654f, kGeluA = 0.044715f, kRsqrt2 = 0.7071067811865476f, kRsqrt2Pi = 0.3989422804014327f;

// e^u and 1 / (1 + e^-u) with the hardware's exponential and reciprocal, one step off each
__device__ __forceinline__ float logistic2(float u) { return __builtin_amdgcn_rcpf(1.f + exp2_fast(-u)); }      // of u ln 2
// 0.5 erfc(-z / sqrt 2), by the rational approximation 7.1.26 of Abramowitz and Stegun (absolute error 1.5e-7)
__device__ __forceinline__ float normal_cdf(float z) {
    const float x = fabsf(z) * kRsqrt2, t = __builtin_amdgcn_rcpf(fmaf(0.3275911f, x, 1.f));
    const float p = t * fmaf(t, fmaf(t, fmaf(t, fmaf(t, 1.061405429f, -1.453152027f), 1.421413741f), -0.284496736f), 0.254829592f);
    const float tail = 0.5f * p * exp2_fast(-0.5f * kLog2e * z * z);
    return z > 0.f ? 1.f - tail : tail;
}
constexpr float kTanh1 = 2.f * kGeluC * kLog2e, kTanh3 = kTanh1 * kGeluA;     // 2 u log2 e = z (kTanh1 + kTanh3 z^2)

__device__ __forceinline__ float activate(int act, float z) {
    switch (act) {
        case LLSA_ACT_SILU: return z * logistic2(kLog2e * z);
        case LLSA_ACT_GELU: return z * normal_cdf(z);
        case LLSA_ACT_GELU_TANH: return z * logistic2(z * fmaf(kTanh3, z * z, kTanh1));
        default: return z;
    }
}
__device__ __forceinline__ float activate_slope(int act, float z) {
    if (act == LLSA_ACT_NONE) return 1.f;
    z = z > 128.f ? 128.f : z < -128.f ? -128.f : z;            // (a NaN stays one)
    switch (act) {
        case LLSA_ACT_SILU: {
            const float s = logistic2(kLog2e * z);
            return fmaf(z * s, 1.f - s, s);
        }
        case LLSA_ACT_GELU: return fmaf(z * kRsqrt2Pi, exp2_fast(-0.5f * kLog2e * z * z), normal_cdf(z));
        default: {
            const float q = z * z, s = logistic2(z * fmaf(kTanh3, q, kTanh1));
            return fmaf(z * fmaf(6.f * kGeluC * kGeluA, q, 2.f * kGeluC) * s, 1.f - s, s);
        }
    }
}

// Both at once, with one exponential and one reciprocal.  The slope is that of a number: whoever keeps it looks at z for a NaN
__device__ __forceinline__ void activate_both(int act, float z, float& value, float& slope) {
    const float t = __builtin_amdgcn_fmed3f(z, -128.f, 128.f);        // (of a NaN some number: the slope is then no number's)
    switch (act) {
        case LLSA_ACT_SILU: {
            const float s = logistic2(kLog2e * t);
            value = z * s;
            slope = fmaf(t * s, 1.f - s, s);
            break;
        }
        case LLSA_ACT_GELU: {
            const float x = fabsf(t) * kRsqrt2, r = __builtin_amdgcn_rcpf(fmaf(0.3275911f, x, 1.f)), bell = exp2_fast(-0.5f * kLog2e * t * t);
            const float p = r * fmaf(r, fmaf(r, fmaf(r, fmaf(r, 1.061405429f, -1.453152027f), 1.421413741f), -0.284496736f), 0.254829592f), tail = 0.5f * p * bell;
            const float cdf = t > 0.f ? 1.f - tail : tail;
            value = z * cdf;
            slope = fmaf(t * kRsqrt2Pi, bell, cdf);
            break;
        }
        case LLSA_ACT_GELU_TANH: {
            const float q = t * t, s = logistic2(t * fmaf(kTanh3, q, kTanh1));
            value = z * s;
            slope = fmaf(t * fmaf(6.f * kGeluC * kGeluA, q, 2.f * kGeluC) * s, 1.f - s, s);
            break;
        }
        default: value = z, slope = 1.f;
    }
}

// ---------------------------------------------------------------------------------------
// operands in LDS
//
// A step takes 64 of the contraction.  Copies go straight into LDS, 16 bytes a lane and 1 KB an instruction, so a tile's layout is
// the order of its source pieces; it is the source address that is permuted, never the place in LDS.
//   rows     ROWS rows of 64 elements.  Piece p (8 elements) of row r holds the row's piece p ^ ((r >> 1) & 7): the 16 rows a fragment read touches then lie in 16 different 16-byte columns of the 256 bytes that all banks hold.
//   columns  64 rows of ROWS elements.  32-byte granule g of row k holds the row's granule g ^ f(k), f out of bits 0, 1 and 3 of k
//            (64 or 192 elements: 1 and 3, 32: 3): the transposing read takes granules of 4 neighbouring rows in each group of 16 lanes and of
//            rows 8 further in the next, which then lie in different banks.
// What lies outside the matrix: rows are clamped (their results are not stored), and beyond the end of the contraction zeros are fetched.
// ---------------------------------------------------------------------------------------
constexpr int kStep = 64;                 // of the contraction
__device__ const u32x4 kZeros[1] = {{0u, 0u, 0u, 0u}};

template <typename T>
__device__ __forceinline__ void copy_to_lds(const T* g_lane, T* lds_wave_base) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)g_lane, (__attribute__((address_space(3))) void*)lds_wave_base, 16, 0, 0);
}

template <typename T, bool COLUMNS, int ROWS, int WAVES>
struct Operand {
    static constexpr int kCopies = ROWS * kStep / 512 / WAVES; // instructions of a wave for one step
    static constexpr int kPerRow = ROWS / 8;                  // columns: 16-byte pieces of a row
    static constexpr int kPieces = kStep / 8;                  // rows: pieces of a row
    static_assert(kCopies * 512 * WAVES == ROWS * kStep, "a step is whole copies of every wave");
    unsigned off[kCopies];                                    // elements from the step's first, of this lane's pieces

    static __device__ __forceinline__ int swap(int r) { return (r >> 1) & 7; }
    static __device__ __forceinline__ int turn(int k) {
        return ROWS == 32 ? (k >> 3) & 1 : ROWS % 128 == 64 ? ((k >> 1) & 1) | ((k >> 3) & 1) << 1 : (k & 3) | ((k >> 3) & 1) << 2;
    }
    // of the lane's piece of copy i: its row and its first element along the row, in the tile
    static __device__ __forceinline__ int row_of(int i, int lane) { return COLUMNS ? (i * 64 + lane) / kPerRow : i * (64 / kPieces) + lane / kPieces; }
    static __device__ __forceinline__ int place_of(int i, int row, int lane) {
        if (!COLUMNS) return ((lane % kPieces) ^ swap(row)) * 8;
        const int unit = i * 64 + lane - row * kPerRow;
        return (((unit >> 1) ^ turn(row)) * 2 + (unit & 1)) * 8;
    }

    // left: rows (columns: elements of a row, a multiple of 8) from the tile's first to the matrix's last
    __device__ __forceinline__ void init(int wave, int lane, int64_t ld, int left) {
#pragma unroll
        for (int j = 0; j < kCopies; j++) {
            const int i = wave * kCopies + j, r = row_of(i, lane), e = place_of(i, r, lane);
            off[j] = COLUMNS ? (unsigned)(r * ld) + (unsigned)min(e, left - 8) : (unsigned)(min(r, left - 1) * ld) + (unsigned)e;
        }
    }
    // k_left: what is left of the contraction from this step on
    __device__ __forceinline__ void request(const T* base, T* tile, int wave, int lane, int k_left) const {
        if (k_left >= kStep) {
#pragma unroll
            for (int j = 0; j < kCopies; j++) copy_to_lds(base + off[j], tile + (wave * kCopies + j) * 512);
        } else {
#pragma unroll
            for (int j = 0; j < kCopies; j++) {
                const int i = wave * kCopies + j, r = row_of(i, lane), k = COLUMNS ? r : place_of(i, r, lane);
                copy_to_lds(k < k_left ? base + off[j] : reinterpret_cast<const T*>(kZeros), tile + (wave * kCopies + j) * 512);
            }
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
            const int r = row + (lane & 15), piece = (4 * ks + (lane >> 4)) ^ swap(lane & 15);
            return *reinterpret_cast<const vec8<T>*>(tile + r * kStep + piece * 8);
        }
    }
};

// Workgroups go round the eight XCDs: each XCD gets a run of consecutive tiles, which share rows of x and y in its L2.
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
        for (int e = 0; e < 8; e++) v[e] = (float)p[min(e, n - 1)];          // (the last one again beyond the end: a branch for each would wait for each)
    }
}
// the same as they are; zeros of no memory
template <typename T>
__device__ __forceinline__ vec8<T> take8(const T* p, bool wide, int n) {
    vec8<T> v;
    if (p != nullptr && wide) return *reinterpret_cast<const vec8<T>*>(p);
#pragma unroll
    for (int e = 0; e < 8; e++) v[e] = (T)0.f;
    if (p != nullptr) {
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = p[min(e, n - 1)];
    }
    return v;
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

// The value of lane l ^ 8
__device__ __forceinline__ u32x4 from_other_half(u32x4 v) {
    u32x4 r;
#pragma unroll
    for (int e = 0; e < 4; e++) r[e] = __float_as_uint(across<8>(__uint_as_float(v[e])));
    return r;
}
// Two pieces of sixteen rows, 64 bytes of each row in either, stored as eight whole lines of 128 bytes twice: lanes l and l ^ 8 exchange a piece, so that
// the first store takes rows 0 .. 7 and the second rows 8 .. 15.  lane_at: elements from `base` to the lane's first piece; the other one is 32 elements further.
template <typename T>
__device__ __forceinline__ void store_lines(T* base, unsigned lane_at, unsigned ld8, const vec8<T>& first, const vec8<T>& second, int lane) {
    const bool upper = lane & 8;
    const u32x4 f = __builtin_bit_cast(u32x4, first), s = __builtin_bit_cast(u32x4, second), theirs = from_other_half(upper ? f : s);
    const u32x4 low = upper ? theirs : f, high = upper ? s : theirs;
    T* const to = base + (upper ? lane_at - ld8 + 32 : lane_at);
    __builtin_nontemporal_store(low, reinterpret_cast<u32x4*>(to));
    __builtin_nontemporal_store(high, reinterpret_cast<u32x4*>(to + ld8));
}
// The same pieces read: requested as lines, and once they are there put back where the lanes want them
template <typename T>
__device__ __forceinline__ void request_lines(vec8<T>& low, vec8<T>& high, const T* base, unsigned lane_at, unsigned ld8, int lane) {
    const T* const from = base + ((lane & 8) ? lane_at - ld8 + 32 : lane_at);
    low = __builtin_nontemporal_load(reinterpret_cast<const vec8<T>*>(from));
    high = __builtin_nontemporal_load(reinterpret_cast<const vec8<T>*>(from + ld8));
}
template <typename T>
__device__ __forceinline__ void arrange_lines(vec8<T>& first, vec8<T>& second, int lane) {
    const bool upper = lane & 8;
    const u32x4 low = __builtin_bit_cast(u32x4, first), high = __builtin_bit_cast(u32x4, second), theirs = from_other_half(upper ? low : high);
    first = __builtin_bit_cast(vec8<T>, upper ? theirs : low);
    second = __builtin_bit_cast(vec8<T>, upper ? high : theirs);
}

// ---------------------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------------------
constexpr int64_t kMaxGrid = (int64_t(1) << 31) - 1;
int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Workgroups of 256 threads in launches that have fewer than 2^32 threads each, all that a launch takes: f(first, count)
constexpr int64_t kMaxBlocks = ((int64_t(1) << 32) - 1) / 256;
template <typename F>
void in_launches(int64_t blocks, F f) {
    for (int64_t first = 0; first < blocks; first += kMaxBlocks) f(first, dim3((unsigned)std::min(kMaxBlocks, blocks - first)));
}

constexpr int kCus = 256;
bool wide8(const void* p, int64_t ld) { return p == nullptr || (aligned16(p) && ld % 8 == 0); }

int64_t pad8(int64_t n) { return (n + 7) / 8 * 8; }

constexpr int64_t kMaxRows = (int64_t(1) << 31) - (1 << 16);
constexpr int64_t kMaxLd = int64_t(1) << 23;                  // 128 rows of 16 bits then lie within 2^32 bytes
bool offsets32(int64_t ld) { return ld >= 0 && ld <= kMaxLd; }
bool rows16(const void* p, int64_t ld) { return p != nullptr && aligned16(p) && ld % 8 == 0 && ld > 0 && ld <= kMaxLd; }

int check_sizes(const char* what, int64_t M, int N, int K, int dtype, int act) {
    LLSA_REQUIRE(M >= 0 && M <= kMaxRows && N > 0 && K > 0 && N < (1 << 23) && K < (1 << 23), "%s: bad sizes (M %lld, N %d, K %d)", what, (long long)M, N, K);
    LLSA_REQUIRE(dtype == LLSA_DTYPE_BF16 || dtype == LLSA_DTYPE_F16, "%s: bf16 or fp16 only", what);
    LLSA_REQUIRE(act >= LLSA_ACT_NONE && act <= LLSA_ACT_GELU_TANH, "%s: unknown activation %d", what, act);
    return 0;
}
}  // namespace
}  // namespace llsa
