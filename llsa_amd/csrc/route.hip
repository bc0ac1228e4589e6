// The router in front of the experts: the k largest logits of every token, their weights, and the order in which the experts' products take the rows.
//
//     w_j = exp(l_j - max l) / sum,  the sum over the chosen ones or over all;     back  dl_i = p_i ([chosen] g_i - [chosen, or sum over all] sum_j g_j w_j)
//
// Equal logits go to the lowest index, a logit of -inf is never chosen, a NaN counts as the largest number (and makes the row's weights NaN, as a softmax does).
// The order is a counting sort by expert that keeps the slots (token * k + choice) in turn: integer counts, no order of atomics in the result.  fp32 throughout.
// Up to 4096 slots in one workgroup and one launch (1024 tokens, two of eight: 7.5 us), beyond in a launch that chooses and counts and one that places.  131072 tokens,
// eight of 64 (33 MB of logits): 29 + 12 us, back 29.
#include "experts_device.h"

namespace llsa {
namespace {

struct Route {
    const void* logits;
    float* weights;
    int32_t *experts, *order, *offsets, *places, *counts;     // counts: [chunk][E]
    int64_t ld;
    int M, E, k, normalize, wide, chunks, per;                // per: tokens of a chunk
    const float* dweights;
    void* dlogits;
    int64_t first;                                            // back: workgroup of this launch
};
constexpr int kRouteThreads = 1024, kRouteSlots = 4096, kRouteChunks = 256;

// Numbers that sort like the logits: 0 for one that cannot be chosen, all bits for a NaN; +0 and -0 are one.
__device__ __forceinline__ unsigned route_key(float f) {
    const unsigned b = __float_as_uint(f + 0.f);
    if (f != f) return ~0u;
    return b == 0xff800000u ? 0u : (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float logit_of(unsigned key) { return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key); }
template <int XOR>
__device__ __forceinline__ unsigned bits_across(unsigned v) { return __float_as_uint(across<XOR>(__uint_as_float(v))); }

template <typename T, int PER>
__device__ __forceinline__ void take_logits(float (&v)[PER], const T* p, int first, int E, bool wide) {
#pragma unroll
    for (int i = 0; i < PER; i += 8) {
        typedef __attribute__((ext_vector_type(8))) T Eight;
        if (wide && first + i < E) {
            const Eight a = *reinterpret_cast<const Eight*>(p + first + i);
#pragma unroll
            for (int e = 0; e < 8; e++) v[i + e] = (float)a[e];
        } else {
#pragma unroll
            for (int e = 0; e < 8; e++) v[i + e] = first + i + e < E ? (float)p[first + i + e] : -__builtin_inff();
        }
    }
}
template <int LANES>
__device__ __forceinline__ float lanes_add(float v) {
    if (LANES > 1) v += across<1>(v);
    if (LANES > 1) v += across<2>(v);
    if (LANES > 4) v += across<7>(v);
    if (LANES > 4) v += across<8>(v);
    return v;
}

// LANES neighbouring lanes hold a token's logits, PER each.  The largest is looked for k times, in the registers and then across the lanes.
template <typename T, int LANES, int PER>
__device__ __forceinline__ void choose(const Route& a, int m, int part, bool there, int* hist) {
    float v[PER];
    unsigned key[PER];
    take_logits<T, PER>(v, static_cast<const T*>(a.logits) + m * a.ld, part * PER, a.E, a.wide);
#pragma unroll
    for (int i = 0; i < PER; i++) key[i] = route_key(v[i]);
    unsigned best[LLSA_MAX_CHOICES];
    int index[LLSA_MAX_CHOICES];
    float top = 0.f, sum = 0.f;
#pragma unroll
    for (int j = 0; j < LLSA_MAX_CHOICES; j++) {
        best[j] = 0;
        index[j] = -1;
        if (j < a.k) {
            unsigned b = 0;
            int at = 0;
#pragma unroll
            for (int i = 0; i < PER; i++)
                if (key[i] > b) b = key[i], at = i;
            at += part * PER;
            auto meet = [&](unsigned other, int there) {
                if (other > b || (other == b && there < at)) b = other, at = there;
            };
            if (LANES > 1) meet(bits_across<1>(b), (int)bits_across<1>((unsigned)at));
            if (LANES > 1) meet(bits_across<2>(b), (int)bits_across<2>((unsigned)at));
            if (LANES > 4) meet(bits_across<7>(b), (int)bits_across<7>((unsigned)at));
            if (LANES > 4) meet(bits_across<8>(b), (int)bits_across<8>((unsigned)at));
#pragma unroll
            for (int i = 0; i < PER; i++)
                if (at == part * PER + i) key[i] = 0;         // (taken; one that cannot be chosen is 0 already)
            best[j] = b;
            index[j] = b != 0 ? at : -1;
            if (j == 0) top = logit_of(b);
            if (b != 0) sum += expf(logit_of(b) - top);
        }
    }
    if (!a.normalize) {
        sum = 0.f;
#pragma unroll
        for (int i = 0; i < PER; i++) sum += part * PER + i < a.E && best[0] != 0 ? expf(v[i] - top) : 0.f;
        sum = lanes_add<LANES>(sum);
    }
    if (part != 0 || !there) return;
#pragma unroll
    for (int j = 0; j < LLSA_MAX_CHOICES; j++) {
        if (j < a.k) {
            a.experts[(int64_t)m * a.k + j] = index[j];
            a.weights[(int64_t)m * a.k + j] = best[j] != 0 ? expf(logit_of(best[j]) - top) / sum : 0.f;
            if (best[j] != 0) atomicAdd(hist + index[j], 1);
        }
    }
}

// The slots of a chunk to their places: run[e] is where the next one of expert e goes.
__device__ __forceinline__ void place_slots(const Route& a, int chunk, int* run, int (*in_wave)[LLSA_MAX_EXPERTS]) {
    constexpr int kWaves = kRouteThreads / 64;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int first = chunk * a.per * a.k, end = min(a.M, (chunk + 1) * a.per) * a.k;
    for (int s0 = first; s0 < end; s0 += kRouteThreads) {
        const int slot = s0 + tid, e = slot < end ? a.experts[slot] : -1;
        uint64_t same = __ballot(e >= 0);
#pragma unroll
        for (int bit = 0; bit < 8; bit++) {
            const uint64_t set = __ballot((e >> bit) & 1);
            same &= (e >> bit) & 1 ? set : ~set;
        }
        const int before = __popcll((unsigned long long)(same & (((uint64_t)1 << lane) - 1)));
        for (int i = lane; i < a.E; i += 64) in_wave[wave][i] = 0;
        __builtin_amdgcn_wave_barrier();
        if (e >= 0 && before == 0) in_wave[wave][e] = __popcll((unsigned long long)same);
        __syncthreads();
        if (e >= 0) {
            int at = run[e] + before;
            for (int w = 0; w < wave; w++) at += in_wave[w][e];
            a.order[at] = slot;
            a.places[slot] = at;
        } else if (slot < end) {
            a.places[slot] = -1;
        }
        __syncthreads();
        if (tid < a.E) {
            int n = run[tid];
            for (int w = 0; w < kWaves; w++) n += in_wave[w][tid];
            run[tid] = n;
        }
        __syncthreads();
    }
}
// Where the experts begin: total[e] of each becomes the sum of those before it, in `run` (and run[E], in all)
__device__ __forceinline__ void begin_runs(int E, const int* total, int* run) {
    if (threadIdx.x >= 64) return;
    int sum = 0;
    for (int e0 = 0; e0 < E; e0 += 64) {
        const int e = e0 + (int)threadIdx.x, n = e < E ? total[e] : 0, upto = sum + lanes_sum_up(n);
        if (e < E) run[e] = upto - n;
        sum = __builtin_amdgcn_readlane(upto, 63);
    }
    if (threadIdx.x == 0) run[E] = sum;
}
__device__ __forceinline__ void fill_tail(const Route& a, int chunk, int all) {
    const int first = max(chunk * a.per * a.k, all), end = min(a.M, (chunk + 1) * a.per) * a.k;
    for (int i = first + (int)threadIdx.x; i < end; i += kRouteThreads) a.order[i] = -1;
}

// ONE: all tokens in this workgroup, which goes on to place them
template <typename T, int LANES, int PER, bool ONE>
__global__ __launch_bounds__(kRouteThreads) void route_kernel(const Route a) {
    __shared__ int hist[LLSA_MAX_EXPERTS], run[LLSA_MAX_EXPERTS + 1], in_wave[kRouteThreads / 64][LLSA_MAX_EXPERTS];
    const int tid = threadIdx.x, chunk = blockIdx.x, end = min(a.M, (chunk + 1) * a.per);
    if (tid < a.E) hist[tid] = 0;
    __syncthreads();
    for (int m0 = chunk * a.per; m0 < end; m0 += kRouteThreads / LANES) {
        const int m = m0 + tid / LANES;
        choose<T, LANES, PER>(a, min(m, end - 1), tid % LANES, m < end, hist);      // (all lanes: they ask one another)
    }
    __syncthreads();
    if constexpr (ONE) {
        begin_runs(a.E, hist, run);
        __syncthreads();
        const int all = run[a.E];
        if (tid <= a.E) a.offsets[tid] = run[tid];
        __syncthreads();
        place_slots(a, 0, run, in_wave);
        fill_tail(a, 0, all);
    } else {
        if (tid < a.E) a.counts[chunk * a.E + tid] = hist[tid];
    }
}
// The counts of all chunks, added up by every workgroup for itself (at most 256 KB out of L2, a launch less)
__global__ __launch_bounds__(kRouteThreads) void place_kernel(const Route a) {
    __shared__ int total[LLSA_MAX_EXPERTS], before[LLSA_MAX_EXPERTS], run[LLSA_MAX_EXPERTS + 1], in_wave[kRouteThreads / 64][LLSA_MAX_EXPERTS];
    const int tid = threadIdx.x, chunk = blockIdx.x;
    if (tid < a.E) total[tid] = before[tid] = 0;
    __syncthreads();
    const int groups = kRouteThreads / a.E, e = tid % a.E, group = tid / a.E;
    if (group < groups) {
        int all = 0, mine = 0;
#pragma unroll 8
        for (int c = group; c < a.chunks; c += groups) {
            const int n = a.counts[c * a.E + e];
            all += n;
            mine += c < chunk ? n : 0;
        }
        atomicAdd(total + e, all);
        atomicAdd(before + e, mine);
    }
    __syncthreads();
    begin_runs(a.E, total, run);
    __syncthreads();
    const int all = run[a.E];
    if (chunk == 0 && tid <= a.E) a.offsets[tid] = run[tid];
    __syncthreads();
    if (tid < a.E) run[tid] += before[tid];
    __syncthreads();
    place_slots(a, chunk, run, in_wave);
    fill_tail(a, chunk, all);
}

// Bound by memory: logits in, their gradient out.
template <typename T, int LANES, int PER>
__global__ __launch_bounds__(256) void route_bwd_kernel(const Route a) {
    const int part = (int)threadIdx.x % LANES;
    const int64_t at = ((a.first + blockIdx.x) * 256 + threadIdx.x) / LANES, m = min(at, (int64_t)a.M - 1);      // (all lanes: they ask one another)
    const T* const logits = static_cast<const T*>(a.logits) + m * a.ld;
    float v[PER], g[PER];
    bool chosen[PER];
    take_logits<T, PER>(v, logits, part * PER, a.E, a.wide);
#pragma unroll
    for (int i = 0; i < PER; i++) g[i] = 0.f, chosen[i] = false;
    // (all loads in flight together)
    int e[LLSA_MAX_CHOICES];
    float d[LLSA_MAX_CHOICES], l[LLSA_MAX_CHOICES];
#pragma unroll
    for (int j = 0; j < LLSA_MAX_CHOICES; j++) e[j] = j < a.k ? a.experts[m * a.k + j] : -1;
#pragma unroll
    for (int j = 0; j < LLSA_MAX_CHOICES; j++) {
        const bool there = (unsigned)e[j] < (unsigned)a.E;
        d[j] = there ? a.dweights[m * a.k + j] : 0.f;
        l[j] = there ? (float)logits[e[j]] : 0.f;
    }
    float top = 0.f, sum = 0.f, dot = 0.f;
    bool any = false;
#pragma unroll
    for (int j = 0; j < LLSA_MAX_CHOICES; j++) {
        if ((unsigned)e[j] < (unsigned)a.E) {
            if (!any) top = l[j];                             // (the largest is the first)
            any = true;
            const float x = expf(l[j] - top);
            sum += x;
            dot += d[j] * x;
#pragma unroll
            for (int i = 0; i < PER; i++)
                if (e[j] == part * PER + i) g[i] = d[j], chosen[i] = true;
        }
    }
    if (!a.normalize && any) {
        sum = 0.f;
#pragma unroll
        for (int i = 0; i < PER; i++) sum += part * PER + i < a.E ? expf(v[i] - top) : 0.f;
        sum = lanes_add<LANES>(sum);
    }
    const float inverse = 1.f / sum;
    dot *= inverse;
    T o[PER];
#pragma unroll
    for (int i = 0; i < PER; i++) {
        const float p = expf(v[i] - top) * inverse;
        const bool counts = any && v[i] != -__builtin_inff() && (chosen[i] || !a.normalize);
        o[i] = (T)(counts ? p * (g[i] - dot) : 0.f);
    }
    if (at >= a.M) return;
    T* const out = static_cast<T*>(a.dlogits) + m * a.E + part * PER;
#pragma unroll
    for (int i = 0; i < PER; i += 8) {
        if (a.E % 8 == 0 && part * PER + i < a.E) {
            typedef __attribute__((ext_vector_type(8))) T Eight;
            Eight w;
#pragma unroll
            for (int e = 0; e < 8; e++) w[e] = o[i + e];
            *reinterpret_cast<Eight*>(out + i) = w;
        } else {
#pragma unroll
            for (int e = 0; e < 8; e++)
                if (part * PER + i + e < a.E) out[i + e] = o[i + e];
        }
    }
}

int route_chunks(int64_t M, int64_t k) { return (int)std::max<int64_t>(1, std::min<int64_t>(kRouteChunks, ceil_div(M * k, kRouteSlots))); }

template <typename T, int LANES, int PER>
void launch_route(Route& a, hipStream_t stream) {
    if (a.dlogits != nullptr) {
        in_launches(ceil_div((int64_t)a.M * LANES, 256), [&](int64_t first, dim3 grid) {
            a.first = first;
            hipLaunchKernelGGL(HIP_KERNEL_NAME(route_bwd_kernel<T, LANES, PER>), grid, dim3(256), 0, stream, a);
        });
    } else if (a.chunks == 1) {
        hipLaunchKernelGGL(HIP_KERNEL_NAME(route_kernel<T, LANES, PER, true>), dim3(1), dim3(kRouteThreads), 0, stream, a);
    } else {
        hipLaunchKernelGGL(HIP_KERNEL_NAME(route_kernel<T, LANES, PER, false>), dim3((unsigned)a.chunks), dim3(kRouteThreads), 0, stream, a);
        hipLaunchKernelGGL(place_kernel, dim3((unsigned)a.chunks), dim3(kRouteThreads), 0, stream, a);
    }
}
template <typename T>
void route(Route& a, hipStream_t stream) {
    if (a.E <= 8) launch_route<T, 1, 8>(a, stream);
    else if (a.E <= 16) launch_route<T, 1, 16>(a, stream);
    else if (a.E <= 64) launch_route<T, 4, 16>(a, stream);
    else launch_route<T, 16, 16>(a, stream);
}
int route_call(const char* what, const llsa_route_args* a, bool back, hipStream_t stream) {
    LLSA_REQUIRE(a != nullptr, "%s: no arguments", what);
    LLSA_REQUIRE(a->E >= 1 && a->E <= LLSA_MAX_EXPERTS && a->k >= 1 && a->k <= a->E && a->k <= LLSA_MAX_CHOICES, "%s: 1 to %d experts, of which a token takes 1 to %d", what, LLSA_MAX_EXPERTS,
                 LLSA_MAX_CHOICES);
    LLSA_REQUIRE(a->M >= 0 && a->M * a->k <= LLSA_MAX_SLOTS, "%s: too many tokens (%lld)", what, (long long)a->M);
    LLSA_REQUIRE(a->dtype == LLSA_DTYPE_BF16 || a->dtype == LLSA_DTYPE_F16 || a->dtype == LLSA_DTYPE_F32, "%s: bf16, fp16 or fp32 only", what);
    LLSA_REQUIRE(a->M == 0 || (a->logits != nullptr && a->experts != nullptr && a->ld >= 0), "%s: logits and experts", what);
    Route r{};
    r.logits = a->logits; r.ld = a->ld; r.weights = a->weights; r.experts = a->experts; r.order = a->order; r.offsets = a->offsets; r.places = a->places;
    r.counts = (int32_t*)a->workspace;
    r.M = (int)a->M; r.E = a->E; r.k = a->k; r.normalize = a->normalize;
    r.wide = a->E % 8 == 0 && aligned16(a->logits) && a->ld % (a->dtype == LLSA_DTYPE_F32 ? 4 : 8) == 0;
    r.chunks = route_chunks(a->M, a->k);
    r.per = (int)ceil_div(a->M, r.chunks);
    if (back) {
        if (a->M == 0) return 0;
        LLSA_REQUIRE(a->dweights != nullptr && a->dlogits != nullptr && aligned16(a->dlogits), "%s: gradients (16-byte aligned)", what);
        r.dweights = a->dweights; r.dlogits = a->dlogits;
    } else {
        LLSA_REQUIRE(a->offsets != nullptr && (a->M == 0 || (a->weights != nullptr && a->order != nullptr && a->places != nullptr)), "%s: results", what);
        LLSA_REQUIRE(r.chunks == 1 || a->workspace != nullptr, "%s: workspace", what);
    }
    if (a->dtype == LLSA_DTYPE_BF16) route<bf16>(r, stream);
    else if (a->dtype == LLSA_DTYPE_F16) route<_Float16>(r, stream);
    else route<float>(r, stream);
    return launch_status(what);
}
}  // namespace
}  // namespace llsa

using namespace llsa;

extern "C" int64_t llsa_route_workspace_bytes(int64_t M, int E, int k) {
    if (M <= 0 || E <= 0 || k <= 0) return 0;
    const int chunks = route_chunks(M, k);
    return chunks > 1 ? 4 * (int64_t)chunks * E : 0;
}
extern "C" int llsa_route_tokens(const llsa_route_args* a, void* stream) { return route_call("route_tokens", a, false, (hipStream_t)stream); }
extern "C" int llsa_route_tokens_bwd(const llsa_route_args* a, void* stream) { return route_call("route_tokens_bwd", a, true, (hipStream_t)stream); }
