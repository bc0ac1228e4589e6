// Layer norm over the channels of token rows, with the weight and bias of a layer norm and the scale and shift of an adaLN block in the
// same pass, and its backward.
//
//     h = (x - mean) * rstd,   y = (h * weight + bias) * (1 + scale_b) + shift_b
//     g = dy * (1 + scale_b) * weight,   dx = rstd * (g - mean(g) - h * mean(g * h))
//
// The gradients of all four vectors come out of two sums per sample and channel, S1 = sum of dy and S2 = sum of dy * h.
//
// A row is held in registers by LANES lanes, up to CHUNKS pieces of 8 channels each: it is read once, the variance is that of the
// differences from the mean (no cancellation; fp32 rows are centred twice), and everything is fp32 in between.  Bound by memory: 131072 x 384 in bf16, forward 39.5 us (201 MB, 5.1 TB/s;
// a large copy 5.2), backward 62.6 (302 MB, 4.8 TB/s), the sums of its pieces 4.6; 32768 x 768 in fp32 46.6 and 67.1 (46.1 and 68.0 centred
// once).
#include <algorithm>
#include <type_traits>

#include "llsa_device.h"
#include "llsa_host.h"

namespace llsa {
namespace {

template <typename T> struct Eight { typedef __attribute__((ext_vector_type(8))) T type; };

// Where a row's channels are held.  WIDE (rows are 16-byte aligned and whole pieces of eight): piece j of a lane is channels (j LANES + lane) 8 .. + 7, read
// and written in pieces.  Otherwise value e of piece j is channel (j 8 + e) LANES + lane, so that what the lanes read one by one lies side by side too.
template <bool WIDE, int LANES>
__device__ __forceinline__ int channel(int j, int e, int lane) { return WIDE ? (j * LANES + lane) * 8 + e : (j * 8 + e) * LANES + lane; }

template <bool WIDE, int LANES, int CHUNKS, typename T>
struct Row {
    typename Eight<T>::type piece[CHUNKS];                    // as they are in memory; zeros beyond the row
    __device__ __forceinline__ void load(const T* row, int C, int lane) {
#pragma unroll
        for (int j = 0; j < CHUNKS; j++) {
            if (WIDE) {
                const int c = channel<WIDE, LANES>(j, 0, lane);
                if (c < C) {
                    piece[j] = __builtin_nontemporal_load(reinterpret_cast<const typename Eight<T>::type*>(row + c));
                } else {
#pragma unroll
                    for (int e = 0; e < 8; e++) piece[j][e] = (T)0.f;
                }
            } else {
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const int c = channel<WIDE, LANES>(j, e, lane);
                    piece[j][e] = c < C ? row[c] : (T)0.f;
                }
            }
        }
    }
};
template <bool WIDE, int LANES, typename T>
__device__ __forceinline__ void store8(T* row, int j, int lane, int C, const float (&v)[8]) {
    if (WIDE) {
        const int c = channel<WIDE, LANES>(j, 0, lane);
        if (c < C) {
            typename Eight<T>::type a;
#pragma unroll
            for (int e = 0; e < 8; e++) a[e] = (T)v[e];
            __builtin_nontemporal_store(a, reinterpret_cast<typename Eight<T>::type*>(row + c));
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const int c = channel<WIDE, LANES>(j, e, lane);
            if (c < C) row[c] = (T)v[e];
        }
    }
}
// A small vector, of the rows' type or fp32, in pieces if it allows them: `otherwise` where there is none or beyond the row
template <bool WIDE, int LANES, typename T>
__device__ __forceinline__ void load_vector(float (&v)[8], const void* p, bool f32, int j, int lane, int C, float otherwise = 0.f) {
    const int first = channel<WIDE, LANES>(j, 0, lane);
    const bool aligned = WIDE && (reinterpret_cast<uintptr_t>(p) & 15) == 0;
    if (p != nullptr && aligned && first < C) {
        if (f32) {
            const Eight<float>::type a = *reinterpret_cast<const Eight<float>::type*>(static_cast<const float*>(p) + first);
#pragma unroll
            for (int e = 0; e < 8; e++) v[e] = a[e];
        } else {
            const typename Eight<T>::type a = *reinterpret_cast<const typename Eight<T>::type*>(static_cast<const T*>(p) + first);
#pragma unroll
            for (int e = 0; e < 8; e++) v[e] = (float)a[e];
        }
        return;
    }
#pragma unroll
    for (int e = 0; e < 8; e++) {
        const int c = channel<WIDE, LANES>(j, e, lane);
        v[e] = p == nullptr || c >= C ? otherwise : f32 ? static_cast<const float*>(p)[c] : (float)static_cast<const T*>(p)[c];
    }
}
__device__ __forceinline__ const void* row_of(const void* p, int64_t elements, int size) {
    return p == nullptr ? nullptr : static_cast<const char*>(p) + elements * size;
}

// Sum over the LANES lanes of a row, the same bits in all of them.  Up to 64 lanes inside a wave; more go through LDS, one slot a wave.
template <int LANES>
__device__ __forceinline__ float row_sum(float v, float* slots) {
    v += across<1>(v);
    v += across<2>(v);
    v += across<7>(v);
    v += across<8>(v);
    if constexpr (LANES >= 64) {
        const u32x2 a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
        const u32x2 b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = __uint_as_float(b[0]) + __uint_as_float(b[1]);
    }
    if constexpr (LANES > 64) {
        constexpr int kWaves = LANES / 64;
        __syncthreads();                                      // the sum before is read by everyone
        if ((threadIdx.x & 63) == 0) slots[threadIdx.x >> 6] = v;
        __syncthreads();
        v = 0.f;
#pragma unroll
        for (int w = 0; w < kWaves; w++) v += slots[w];
    }
    return v;
}

// The row's values v become their differences from `mean`, zeros beyond the row.  Of fp32 rows far from zero the mean is off by a part of their size, which
// may be more than their spread: the differences, exact or nearly, are then centred a second time (`again`).  Returns what that adds to the mean.
template <bool WIDE, int LANES, int CHUNKS>
__device__ __forceinline__ float centre(float (&v)[CHUNKS][8], float mean, int C, int lane, float* slots, bool again) {
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < CHUNKS; j++)
#pragma unroll
        for (int e = 0; e < 8; e++) {
            v[j][e] = channel<WIDE, LANES>(j, e, lane) < C ? v[j][e] - mean : 0.f;
            s += v[j][e];
        }
    if (!again) return 0.f;
    const float more = row_sum<LANES>(s, slots) / (float)C;
#pragma unroll
    for (int j = 0; j < CHUNKS; j++)
#pragma unroll
        for (int e = 0; e < 8; e++) v[j][e] = channel<WIDE, LANES>(j, e, lane) < C ? v[j][e] - more : 0.f;
    return more;
}

struct Norm {
    const void *x, *dy;
    void *y, *dx;
    const void *weight, *bias, *scale, *shift;
    float *stats, *part;
    int64_t ldx, ldy, lddy, lddx, s_scale, s_shift;
    int64_t rows, per_sample;
    int C, pieces, piece_rows;            // a workgroup: piece_rows rows of one sample
    bool f32;                             // the small vectors are fp32
    float eps;
};

constexpr int kThreads = 256, kCus = 256;

// rows first .. last - 1 of the workgroup's sample
struct Share { int64_t first, last; int64_t sample; };
__device__ __forceinline__ Share share_of(const Norm& a) {
    const int64_t sample = (int)blockIdx.x / a.pieces, piece = (int)blockIdx.x - sample * a.pieces, base = sample * a.per_sample;
    const int64_t end = min(a.per_sample, (piece + 1) * a.piece_rows);
    return {base + piece * a.piece_rows, base + end, sample};
}

template <typename T, int LANES, int CHUNKS, bool WIDE>
__global__ __launch_bounds__(kThreads) void norm_fwd_kernel(const Norm a) {
    constexpr int kRows = kThreads / LANES;
    __shared__ float slots[LANES > 64 ? LANES / 64 : 1];
    const int lane = threadIdx.x % LANES, row = threadIdx.x / LANES;
    const Share share = share_of(a);
    Row<WIDE, LANES, CHUNKS, T> next;                         // a row on its way while the one before is worked on
    auto request = [&](int64_t first) { next.load(static_cast<const T*>(a.x) + min(first + row, share.last - 1) * a.ldx, a.C, lane); };
    request(share.first);
    float up[CHUNKS][8], add[CHUNKS][8];                      // y = h * up + add
    const int es = a.f32 ? 4 : (int)sizeof(T);
    const void *scale = row_of(a.scale, share.sample * a.s_scale, es), *shift = row_of(a.shift, share.sample * a.s_shift, es);
#pragma unroll
    for (int j = 0; j < CHUNKS; j++) {
        float t[8], u[8];
        load_vector<WIDE, LANES, T>(up[j], a.weight, a.f32, j, lane, a.C, 1.f);
        load_vector<WIDE, LANES, T>(add[j], a.bias, a.f32, j, lane, a.C);
        load_vector<WIDE, LANES, T>(t, scale, a.f32, j, lane, a.C);
        load_vector<WIDE, LANES, T>(u, shift, a.f32, j, lane, a.C);
#pragma unroll
        for (int e = 0; e < 8; e++) {
            up[j][e] *= 1.f + t[e];
            add[j][e] = fmaf(add[j][e], 1.f + t[e], u[e]);
        }
    }
    const float C = (float)a.C;
    for (int64_t first = share.first; first < share.last; first += kRows) {       // (the same count for all lanes: row sums may meet at barriers)
        const int64_t r = first + row;
        float v[CHUNKS][8], s = 0.f;
#pragma unroll
        for (int j = 0; j < CHUNKS; j++)
#pragma unroll
            for (int e = 0; e < 8; e++) {
                v[j][e] = (float)next.piece[j][e];
                s += v[j][e];
            }
        if (first + kRows < share.last) request(first + kRows);
        float mean = row_sum<LANES>(s, slots) / C;           // (divided: the mean of equal values of 16 bits, whose sums are exact, is that value)
        mean += centre<WIDE, LANES>(v, mean, a.C, lane, slots, std::is_same_v<T, float>);
        s = 0.f;
#pragma unroll
        for (int j = 0; j < CHUNKS; j++)
#pragma unroll
            for (int e = 0; e < 8; e++) s = fmaf(v[j][e], v[j][e], s);
        const float rstd = rsqrtf(row_sum<LANES>(s, slots) / C + a.eps);
        if (r >= share.last) continue;
        if (a.stats != nullptr && lane == 0) {
            a.stats[2 * r] = mean;
            a.stats[2 * r + 1] = rstd;
        }
        T* const y = static_cast<T*>(a.y) + r * a.ldy;
#pragma unroll
        for (int j = 0; j < CHUNKS; j++) {
#pragma unroll
            for (int e = 0; e < 8; e++) v[j][e] = fmaf(v[j][e] * rstd, up[j][e], add[j][e]);
            store8<WIDE, LANES>(y, j, lane, a.C, v[j]);
        }
    }
}

// dx, and the workgroup's share of S1 and S2 ([sample][piece][2][C])
template <typename T, int LANES, int CHUNKS, bool WIDE>
__global__ __launch_bounds__(kThreads) void norm_bwd_kernel(const Norm a) {
    constexpr int kRows = kThreads / LANES;
    __shared__ float slots[LANES > 64 ? LANES / 64 : 1];
    __shared__ float sums[kRows > 1 ? kThreads * 8 : 1];
    const int lane = threadIdx.x % LANES, row = threadIdx.x / LANES;
    const Share share = share_of(a);
    Row<WIDE, LANES, CHUNKS, T> next_x, next_dy;
    float next_mean, next_rstd;
    auto request = [&](int64_t first) {
        const int64_t r = min(first + row, share.last - 1);
        next_x.load(static_cast<const T*>(a.x) + r * a.ldx, a.C, lane);
        next_dy.load(static_cast<const T*>(a.dy) + r * a.lddy, a.C, lane);
        next_mean = a.stats[2 * r];
        next_rstd = a.stats[2 * r + 1];
    };
    request(share.first);
    float up[CHUNKS][8], s1[CHUNKS][8], s2[CHUNKS][8];
    const void* scale = row_of(a.scale, share.sample * a.s_scale, a.f32 ? 4 : (int)sizeof(T));
#pragma unroll
    for (int j = 0; j < CHUNKS; j++) {
        float t[8];
        load_vector<WIDE, LANES, T>(up[j], a.weight, a.f32, j, lane, a.C, 1.f);
        load_vector<WIDE, LANES, T>(t, scale, a.f32, j, lane, a.C);
#pragma unroll
        for (int e = 0; e < 8; e++) up[j][e] *= 1.f + t[e], s1[j][e] = 0.f, s2[j][e] = 0.f;
    }
    const float per = 1.f / (float)a.C;
    for (int64_t first = share.first; first < share.last; first += kRows) {
        const int64_t r = first + row;
        const bool there = r < share.last;
        const float mean = next_mean, rstd = next_rstd;
        float h[CHUNKS][8], d[CHUNKS][8], sg = 0.f, sgh = 0.f;
#pragma unroll
        for (int j = 0; j < CHUNKS; j++)
#pragma unroll
            for (int e = 0; e < 8; e++) {
                h[j][e] = std::is_same_v<T, float> ? (float)next_x.piece[j][e] : ((float)next_x.piece[j][e] - mean) * rstd;
                d[j][e] = there ? (float)next_dy.piece[j][e] : 0.f;         // (beyond the row d is zero, and so is all that h enters)
            }
        if (first + kRows < share.last) request(first + kRows);
        if constexpr (std::is_same_v<T, float>) {             // (the mean that the forward left is rounded to fp32)
            centre<WIDE, LANES>(h, mean, a.C, lane, slots, true);
#pragma unroll
            for (int j = 0; j < CHUNKS; j++)
#pragma unroll
                for (int e = 0; e < 8; e++) h[j][e] *= rstd;
        }
#pragma unroll
        for (int j = 0; j < CHUNKS; j++)
#pragma unroll
            for (int e = 0; e < 8; e++) {
                s1[j][e] += d[j][e];
                s2[j][e] = fmaf(d[j][e], h[j][e], s2[j][e]);
                d[j][e] *= up[j][e];
                sg += d[j][e];
                sgh = fmaf(d[j][e], h[j][e], sgh);
            }
        if (a.dx == nullptr) continue;
        sg = row_sum<LANES>(sg, slots) * per;
        sgh = row_sum<LANES>(sgh, slots) * per;
        if (!there) continue;
        T* const dx = static_cast<T*>(a.dx) + r * a.lddx;
#pragma unroll
        for (int j = 0; j < CHUNKS; j++) {
#pragma unroll
            for (int e = 0; e < 8; e++) d[j][e] = rstd * (d[j][e] - sg - h[j][e] * sgh);
            store8<WIDE, LANES>(dx, j, lane, a.C, d[j]);
        }
    }
    if (a.part == nullptr) return;
    float* const part = a.part + (int64_t)blockIdx.x * 2 * a.C;
#pragma unroll
    for (int which = 0; which < 2; which++)
#pragma unroll
        for (int j = 0; j < CHUNKS; j++) {
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; e++) v[e] = which == 0 ? s1[j][e] : s2[j][e];
            if constexpr (kRows > 1) {                        // the rows of the workgroup, added in their order
                __syncthreads();
#pragma unroll
                for (int e = 0; e < 8; e++) sums[e * kThreads + threadIdx.x] = v[e];
                __syncthreads();
                if (row > 0) continue;
#pragma unroll 1
                for (int i = 1; i < kRows; i++)
#pragma unroll
                    for (int e = 0; e < 8; e++) v[e] += sums[e * kThreads + i * LANES + lane];
            }
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const int c = channel<WIDE, LANES>(j, e, lane);
                if (c < a.C) part[(int64_t)which * a.C + c] = v[e];
            }
        }
}

struct Join {
    const float* part;
    float* per_sample;                    // [sample][2][C]: what a sample adds to dbias and dweight, or NULL
    const void *weight, *bias, *scale;
    void *dscale, *dshift, *dweight, *dbias;
    int64_t s_scale;
    int C, pieces, samples, groups;       // groups: of sixteen channels
    bool f32;
};
template <typename T>
__device__ __forceinline__ float entry(const void* p, bool f32, int64_t i) { return f32 ? static_cast<const float*>(p)[i] : (float)static_cast<const T*>(p)[i]; }
template <typename T>
__device__ __forceinline__ void put(void* p, bool f32, int64_t i, float v) {
    if (f32) static_cast<float*>(p)[i] = v;
    else static_cast<T*>(p)[i] = (T)v;
}
// S1 and S2 of a sample out of its pieces: 16 channels a workgroup, sixteen threads for each, which take every sixteenth piece
constexpr int kJoinChannels = 16, kJoinLanes = 16;
template <typename T>
__global__ __launch_bounds__(256) void norm_join_kernel(const Join a) {
    __shared__ float sums[2][kJoinLanes][kJoinChannels];
    const int k = threadIdx.x % kJoinChannels, lane = threadIdx.x / kJoinChannels, sample = (int)blockIdx.x / a.groups, c = ((int)blockIdx.x - sample * a.groups) * kJoinChannels + k;
    float s1 = 0.f, s2 = 0.f;
    if (c < a.C) {
        const float* const part = a.part + (int64_t)sample * a.pieces * 2 * a.C + c;
#pragma unroll 8
        for (int p = lane; p < a.pieces; p += kJoinLanes) {
            s1 += part[(int64_t)p * 2 * a.C];
            s2 += part[(int64_t)p * 2 * a.C + a.C];
        }
    }
    sums[0][lane][k] = s1;
    sums[1][lane][k] = s2;
    __syncthreads();
    if (lane > 0 || c >= a.C) return;
#pragma unroll
    for (int i = 1; i < kJoinLanes; i++) s1 += sums[0][i][k], s2 += sums[1][i][k];
    const int64_t at = (int64_t)sample * a.C + c;
    if (a.dshift != nullptr) put<T>(a.dshift, a.f32, at, s1);
    if (a.dscale != nullptr) {
        const float w = a.weight != nullptr ? entry<T>(a.weight, a.f32, c) : 1.f, b = a.bias != nullptr ? entry<T>(a.bias, a.f32, c) : 0.f;
        put<T>(a.dscale, a.f32, at, w * s2 + b * s1);
    }
    if (a.samples == 1) {                                     // (their sum over the samples already)
        const float up = a.scale != nullptr ? 1.f + entry<T>(a.scale, a.f32, c) : 1.f;
        if (a.dbias != nullptr) put<T>(a.dbias, a.f32, c, up * s1);
        if (a.dweight != nullptr) put<T>(a.dweight, a.f32, c, up * s2);
    } else if (a.per_sample != nullptr) {
        const float up = a.scale != nullptr ? 1.f + entry<T>(a.scale, a.f32, sample * a.s_scale + c) : 1.f;
        a.per_sample[(int64_t)sample * 2 * a.C + c] = up * s1;
        a.per_sample[(int64_t)sample * 2 * a.C + a.C + c] = up * s2;
    }
}
template <typename T>
__global__ __launch_bounds__(256) void norm_join_samples_kernel(const Join a) {
    const int c = (int)blockIdx.x * 256 + threadIdx.x;
    if (c >= a.C) return;
    float s1 = 0.f, s2 = 0.f;
    for (int b = 0; b < a.samples; b++) {
        s1 += a.per_sample[(int64_t)b * 2 * a.C + c];
        s2 += a.per_sample[(int64_t)b * 2 * a.C + a.C + c];
    }
    if (a.dbias != nullptr) put<T>(a.dbias, a.f32, c, s1);
    if (a.dweight != nullptr) put<T>(a.dweight, a.f32, c, s2);
}

// ---------------------------------------------------------------------------------------
// launches
// ---------------------------------------------------------------------------------------
constexpr int64_t kMaxGrid = (int64_t(1) << 31) - 1;
int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Lanes and pieces of eight channels a lane: as few idle lanes as there can be with at most three pieces (backward: two, whose sums take registers from the
// waves that hide the loads), then as few lanes.  us, forward + backward of 131072 x 384: 16 lanes of 3 pieces 39.5 + 80.8, 64 of 1 42.0 + 65.1; 8192 x 2048:
// 64 of 4 18.9 + 44.0, 256 of 1 15.5 + 37.0.
struct Shape { int lanes, chunks; };
Shape shape_for(int C, bool backward) {
    const int pieces = (int)ceil_div(C, 8);
    Shape best{256, 4};
    for (int lanes : {16, 64, 256})
        for (int chunks = 1; chunks <= (backward ? 2 : 3); chunks++)
            if (lanes * chunks >= pieces && (lanes * chunks < best.lanes * best.chunks)) best = {lanes, chunks};
    return best.chunks == 4 && 3 * 256 >= pieces ? Shape{256, 3} : best;
}
// The split of the rows over workgroups, each of one sample's rows.  A workgroup first reads the vectors, so it gets several rows for every one that it holds
// at a time.  The backward's leave sums that are added up in a launch of their own: 64 rows each, but 512 to 768 workgroups (us, 512 / 768 / 1536: 131072 x
// 384 72 / 65 / 72, 32768 x 1024 49.6 / 51.5 / 54.9, 8192 x 2048 34.0 / 37.0 / 47.1).
struct Split { int pieces, rows; };
Split split_rows(int64_t rows, int64_t per_sample, int C, bool backward) {
    const Shape s = shape_for(C, backward);
    const int64_t at_once = std::max(1, kThreads / s.lanes), samples = rows / per_sample;
    const int64_t most = backward ? std::min<int64_t>(768, std::max<int64_t>(512, rows / 64)) : 2048;
    const int64_t wanted = std::max<int64_t>(1, most / samples);
    int64_t each = ceil_div(ceil_div(per_sample, wanted), at_once) * at_once;
    each = std::max(each, std::min<int64_t>(2, ceil_div(rows, at_once * kCus)) * at_once);      // (twice as many rows as at a time, if that leaves a workgroup for each CU)
    return {(int)ceil_div(per_sample, each), (int)each};
}

template <typename T, int LANES, int CHUNKS>
void launch_fwd(const Norm& a, int64_t grid, bool wide, hipStream_t stream) {
    const dim3 g((unsigned)grid), b(kThreads);
    if (wide) hipLaunchKernelGGL(HIP_KERNEL_NAME(norm_fwd_kernel<T, LANES, CHUNKS, true>), g, b, 0, stream, a);
    else hipLaunchKernelGGL(HIP_KERNEL_NAME(norm_fwd_kernel<T, LANES, CHUNKS, false>), g, b, 0, stream, a);
}
template <typename T, int LANES, int CHUNKS>
void launch(const Norm& a, int64_t grid, bool backward, bool wide, hipStream_t stream) {
    const dim3 g((unsigned)grid), b(kThreads);
    if (!backward) return launch_fwd<T, LANES, CHUNKS>(a, grid, wide, stream);
    if (wide) hipLaunchKernelGGL(HIP_KERNEL_NAME(norm_bwd_kernel<T, LANES, CHUNKS, true>), g, b, 0, stream, a);
    else hipLaunchKernelGGL(HIP_KERNEL_NAME(norm_bwd_kernel<T, LANES, CHUNKS, false>), g, b, 0, stream, a);
}
template <typename T, int LANES>
void launch_chunks(const Norm& a, int chunks, int64_t grid, bool backward, bool wide, hipStream_t stream) {
    if (chunks == 1) return launch<T, LANES, 1>(a, grid, backward, wide, stream);
    if (chunks == 2) return launch<T, LANES, 2>(a, grid, backward, wide, stream);
    if constexpr (LANES == 256) {
        if (chunks == 3) return launch<T, LANES, 3>(a, grid, backward, wide, stream);
        return launch<T, LANES, 4>(a, grid, backward, wide, stream);
    } else {
        return launch_fwd<T, LANES, 3>(a, grid, wide, stream);
    }
}
template <typename T>
int launch_norm(const Norm& a, bool backward, bool wide, hipStream_t stream) {
    const Shape s = shape_for(a.C, backward);
    const int64_t grid = a.rows / a.per_sample * a.pieces;
    if (grid > kMaxGrid) return fail(-1, "layer_norm: too many samples");
    switch (s.lanes) {
        case 16: launch_chunks<T, 16>(a, s.chunks, grid, backward, wide, stream); break;
        case 64: launch_chunks<T, 64>(a, s.chunks, grid, backward, wide, stream); break;
        default: launch_chunks<T, 256>(a, s.chunks, grid, backward, wide, stream); break;
    }
    return 0;
}

int check(const char* what, const llsa_layer_norm_args* a) {
    LLSA_REQUIRE(a != nullptr, "%s: no arguments", what);
    LLSA_REQUIRE(a->C > 0 && a->C <= LLSA_NORM_MAX_CHANNELS, "%s: 1 to %d channels (got %d)", what, LLSA_NORM_MAX_CHANNELS, a->C);
    LLSA_REQUIRE(a->rows >= 0 && a->per_sample > 0 && a->rows % a->per_sample == 0, "%s: rows of a sample", what);
    LLSA_REQUIRE(a->dtype == LLSA_DTYPE_BF16 || a->dtype == LLSA_DTYPE_F16 || a->dtype == LLSA_DTYPE_F32, "%s: bf16, fp16 or fp32", what);
    LLSA_REQUIRE(a->vtype == a->dtype || a->vtype == LLSA_DTYPE_F32, "%s: weight, bias, scale and shift have the rows' type or fp32", what);
    LLSA_REQUIRE(a->rows == 0 || a->x != nullptr, "%s: no rows", what);
    return 0;
}
Norm common(const llsa_layer_norm_args* a, bool backward) {
    Norm n{};
    const Split s = split_rows(a->rows, a->per_sample, a->C, backward);
    n.x = a->x; n.ldx = a->ldx;
    n.weight = a->weight; n.bias = a->bias; n.scale = a->scale; n.shift = a->shift; n.s_scale = a->s_scale; n.s_shift = a->s_shift;
    n.stats = a->stats;
    n.rows = a->rows; n.per_sample = a->per_sample; n.C = a->C; n.pieces = s.pieces; n.piece_rows = s.rows;
    n.f32 = a->vtype == LLSA_DTYPE_F32;
    n.eps = a->eps;
    return n;
}
// pieces of eight channels are whole and 16-byte aligned
bool wide_rows(const void* p, int64_t ld) { return p == nullptr || (aligned16(p) && ld % 8 == 0); }

template <typename T>
int backward(const llsa_layer_norm_args* a, hipStream_t stream) {
    Norm n = common(a, true);
    n.dy = a->dy; n.lddy = a->lddy; n.dx = a->dx; n.lddx = a->lddx;
    const bool sums = a->dweight != nullptr || a->dbias != nullptr || a->dscale != nullptr || a->dshift != nullptr;
    n.part = sums ? static_cast<float*>(a->workspace) : nullptr;
    const bool wide = a->C % 8 == 0 && wide_rows(a->x, a->ldx) && wide_rows(a->dy, a->lddy) && wide_rows(a->dx, a->lddx);
    if (int rc = launch_norm<T>(n, true, wide, stream)) return rc;
    if (sums) {
        Join j{};
        const int64_t samples = a->rows / a->per_sample;
        j.part = n.part; j.pieces = n.pieces; j.samples = (int)samples; j.groups = (int)ceil_div(a->C, kJoinChannels); j.C = a->C; j.f32 = n.f32;
        j.weight = a->weight; j.bias = a->bias; j.scale = a->scale; j.s_scale = a->s_scale;
        j.dscale = a->dscale; j.dshift = a->dshift; j.dweight = a->dweight; j.dbias = a->dbias;
        if (samples > 1 && (a->dweight != nullptr || a->dbias != nullptr)) j.per_sample = n.part + samples * n.pieces * 2 * a->C;
        hipLaunchKernelGGL(HIP_KERNEL_NAME(norm_join_kernel<T>), dim3((unsigned)(samples * j.groups)), dim3(256), 0, stream, j);
        if (j.per_sample != nullptr) hipLaunchKernelGGL(HIP_KERNEL_NAME(norm_join_samples_kernel<T>), dim3((unsigned)ceil_div(a->C, 256)), dim3(256), 0, stream, j);
    }
    return launch_status("layer_norm_bwd");
}
}  // namespace
}  // namespace llsa

using namespace llsa;

extern "C" int64_t llsa_layer_norm_bwd_workspace_bytes(int64_t rows, int64_t per_sample, int C) {
    if (rows <= 0 || per_sample <= 0 || C <= 0 || C > LLSA_NORM_MAX_CHANNELS) return 0;
    return 4 * (rows / per_sample) * (split_rows(rows, per_sample, C, true).pieces + 1) * 2 * C;
}
extern "C" int llsa_layer_norm_fwd(const llsa_layer_norm_args* a, void* stream) {
    if (int rc = check("layer_norm_fwd", a)) return rc;
    if (a->rows == 0) return 0;
    LLSA_REQUIRE(a->y != nullptr, "layer_norm_fwd: no output");
    Norm n = common(a, false);
    n.y = a->y; n.ldy = a->ldy;
    const bool wide = a->C % 8 == 0 && wide_rows(a->x, a->ldx) && wide_rows(a->y, a->ldy);
    const hipStream_t s = (hipStream_t)stream;
    int rc = a->dtype == LLSA_DTYPE_BF16 ? launch_norm<bf16>(n, false, wide, s) : a->dtype == LLSA_DTYPE_F16 ? launch_norm<_Float16>(n, false, wide, s) : launch_norm<float>(n, false, wide, s);
    return rc != 0 ? rc : launch_status("layer_norm_fwd");
}
extern "C" int llsa_layer_norm_bwd(const llsa_layer_norm_args* a, void* stream) {
    if (int rc = check("layer_norm_bwd", a)) return rc;
    LLSA_REQUIRE(a->rows > 0, "layer_norm_bwd: no rows");
    LLSA_REQUIRE(a->dy != nullptr && a->stats != nullptr, "layer_norm_bwd: dy and the statistics are needed");
    LLSA_REQUIRE(a->workspace != nullptr || (a->dweight == nullptr && a->dbias == nullptr && a->dscale == nullptr && a->dshift == nullptr), "layer_norm_bwd: workspace");
    LLSA_REQUIRE(a->rows / a->per_sample <= kMaxGrid / ceil_div(a->C, kJoinChannels), "layer_norm_bwd: too many samples (%lld)", (long long)(a->rows / a->per_sample));
    const hipStream_t s = (hipStream_t)stream;
    return a->dtype == LLSA_DTYPE_BF16 ? backward<bf16>(a, s) : a->dtype == LLSA_DTYPE_F16 ? backward<_Float16>(a, s) : backward<float>(a, s);
}
