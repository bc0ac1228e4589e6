// Runs of rows that belong to one expert each, as the kernels find their work in them, and operands whose rows are gathered.
#pragma once
#include "product_device.h"

namespace llsa {
namespace {

// Inclusive sums and maxima over the lanes of a wave, of values that are not negative: moves inside vector instructions (rows of 16 lanes shifted, the
// last lane of a row handed on), where a shuffle goes through the LDS unit.
#ifndef LLSA_CPU_EMU_BUILD
#define LLSA_SCAN(op)                                                                     \
    op(__builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, true));  /* row_shr:1 */        \
    op(__builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, true));                         \
    op(__builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, true));                         \
    op(__builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, true));                         \
    op(__builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false)); /* row_bcast:15 */     \
    op(__builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false)); /* row_bcast:31 */
#else
#define LLSA_SCAN(op)                                                                     \
    for (int step = 1; step < 64; step *= 2) {                                            \
        const int below = __shfl_up(v, step);                                             \
        op(emu::lane_id() >= step ? below : 0);                                           \
    }
#endif
__device__ __forceinline__ int lanes_sum_up(int v) {
#define LLSA_ADD(x) v += x
    LLSA_SCAN(LLSA_ADD)
#undef LLSA_ADD
    return v;
}
__device__ __forceinline__ int lanes_max_up(int v) {
#define LLSA_MAX(x) do { const int o = (x); v = o > v ? o : v; } while (0)
    LLSA_SCAN(LLSA_MAX)
#undef LLSA_MAX
    return v;
}
#undef LLSA_SCAN

// The rows of expert e are offsets[e] .. offsets[e + 1] - 1.  The offsets are a caller's: they are held to 0 .. rows and made not to fall, so that no
// two experts share a row.  Cut into pieces of `size` rows, and the pieces numbered expert by expert, then those of the rows that no expert has (`gaps`).
// Every wave works this out for itself, a lane an expert: one load of latency, like a table of pieces, and no launch that writes one.
struct Piece { int expert, first, begin, end, count; };      // first: number of the expert's first piece; count: its pieces.  expert < 0: no expert's rows
struct Runs {
    static constexpr int kLanes = LLSA_MAX_EXPERTS / 64;
    int begin[kLanes], end[kLanes], upto[kLanes], of_experts, total, front, back;
    int size, rows;

    __device__ __forceinline__ void load(const int32_t* offsets, int experts, int rows_, int size_, bool gaps, int lane) {
        size = size_;
        rows = rows_;
        int most = 0, sum = 0, first = 0;
#pragma unroll
        for (int i = 0; i < kLanes; i++) {
            begin[i] = end[i] = upto[i] = 0;
            if (64 * i >= experts) continue;
            const int e = 64 * i + lane;
            const int from = e < experts ? clampi(offsets[e], 0, rows) : 0, to = e < experts ? clampi(offsets[e + 1], 0, rows) : 0;
            begin[i] = max(most, lanes_max_up(from));
            end[i] = max(begin[i], to);
            if (e >= experts) end[i] = begin[i];
            upto[i] = sum + lanes_sum_up((end[i] - begin[i] + size - 1) / size);
            if (i == 0) first = __builtin_amdgcn_readlane(begin[0], 0);
            sum = __builtin_amdgcn_readlane(upto[i], 63);
            most = __builtin_amdgcn_readlane(end[i], min(experts - 64 * i, 64) - 1);
        }
        of_experts = total = sum;
        front = first;
        back = most;
        if (gaps) total += (front + size - 1) / size + (rows - back + size - 1) / size;
    }
    __device__ __forceinline__ Piece of_expert(int i, int lane_) const {
        const int b = __builtin_amdgcn_readlane(begin[i], lane_), e = __builtin_amdgcn_readlane(end[i], lane_), u = __builtin_amdgcn_readlane(upto[i], lane_);
        const int n = (e - b + size - 1) / size;
        return {64 * i + lane_, u - n, b, e, n};
    }
    // the first expert with rows among first .. last - 1; -1: none
    __device__ __forceinline__ Piece among(int first, int last) const {
        Piece p = {-1, 0, last, last, 0};
#pragma unroll
        for (int i = 0; i < kLanes; i++) {
            const uint64_t them = __ballot(end[i] > begin[i] && begin[i] < last && end[i] > first);
            if (p.expert < 0 && them != 0) p = of_expert(i, __ffsll((unsigned long long)them) - 1);
        }
        return p;
    }
    // piece t < total: its expert, and that expert's rows
    __device__ __forceinline__ Piece find(int t) const {
        if (t >= of_experts) {
            const int g = t - of_experts, n = (front + size - 1) / size;
            return g < n ? Piece{-1, of_experts, 0, front, n} : Piece{-1, of_experts + n, back, rows, (rows - back + size - 1) / size};
        }
        Piece p = {0, 0, 0, 0, 0};
        bool found = false;
#pragma unroll
        for (int i = 0; i < kLanes; i++) {
            if (found) continue;
            const uint64_t beyond = __ballot(upto[i] > t);
            if (beyond != 0) {
                p = of_expert(i, __ffsll((unsigned long long)beyond) - 1);
                found = true;
            }
        }
        return p;
    }
};

// A copy that the compiler takes for a new value: what is computed from it inside a loop is not kept in registers around the loop.
__device__ __forceinline__ int fresh(int v) {
#ifndef LLSA_CPU_EMU_BUILD
    asm volatile("" : "+v"(v));
#endif
    return v;
}

// Which row of tokens stands at a place of the sorted order: slots are numbered token * per_token + choice
struct Order {
    const int32_t* slots;                 // or NULL: rows are where they are
    unsigned inverse;                     // 2^32 / per_token, rounded up; 0: one choice
    int tokens, count;                    // rows of tokens, places
    __device__ __forceinline__ int slot(int place) const { return clampi(slots[place], 0, count - 1); }      // (a caller's numbers)
    __device__ __forceinline__ int token(int place) const {
        const unsigned s = (unsigned)slot(place);
        return min(inverse == 0 ? (int)s : (int)(((uint64_t)s * inverse) >> 32), tokens - 1);
    }
};

// Rows of x as Operand<rows> lays them out in LDS.  GATHERED: of tokens in the order
template <typename T, int ROWS, int WAVES, bool GATHERED>
struct RowsAlong {
    typedef Operand<T, false, ROWS, WAVES> Plain;
    static constexpr int kCopies = Plain::kCopies;
    Plain plain;
    const T* x;
    const T* from[GATHERED ? kCopies : 1];
    __device__ __forceinline__ void init(const T* x_, int64_t ld, const Order& order, int first, int left, int wave, int lane) {
        if constexpr (GATHERED) {
#pragma unroll
            for (int j = 0; j < kCopies; j++) {
                const int i = wave * kCopies + j, r = Plain::row_of(i, lane);
                from[j] = x_ + order.token(first + min(r, left - 1)) * ld + Plain::place_of(i, r, lane);
            }
        } else {
            x = x_ + first * ld;
            plain.init(wave, lane, ld, left);
        }
    }
    __device__ __forceinline__ void request(T* tile, int wave, int lane, int k_left) {
        if constexpr (GATHERED) {
#pragma unroll
            for (int j = 0; j < kCopies; j++) {
                const int i = wave * kCopies + j;
                const bool inside = k_left >= kStep || Plain::place_of(i, Plain::row_of(i, lane), lane) < k_left;
                copy_to_lds(inside ? from[j] : reinterpret_cast<const T*>(kZeros), tile + i * 512);
                from[j] += kStep;
            }
        } else {
            plain.request(x, tile, wave, lane, k_left);
            x += kStep;
        }
    }
};
}  // namespace
}  // namespace llsa
