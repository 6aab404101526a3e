// What the sampling kernels share: walks over a row of logits, its best token, and the thresholds that keep the most likely of a set of weights.
#pragma once

#include "common.h"

namespace egpt {

constexpr int kSampleThreads = 1024;

// Calls f(index, value) for every element of p[0..n) once, spread over the workgroup's threads (thread `tid` of
// `n_threads`).  The body reads 16 bytes per thread and keeps eight such loads in flight: a pass over a row is a
// chain of dependent loads otherwise, and its time is their latency, not the row's size.
template <int kAhead = 8, typename F>
__device__ __forceinline__ void for_each_in_row(const float* __restrict__ p, int n, int tid, int n_threads, F f) {
    const int head = min(n, static_cast<int>((4u - ((reinterpret_cast<uintptr_t>(p) >> 2) & 3u)) & 3u));
    for (int j = tid; j < head; j += n_threads) f(j, p[j]);
    const float4* p4 = reinterpret_cast<const float4*>(p + head);
    const int n4 = (n - head) / 4;
    // eight loads issued before the first value is used (the compiler does not do this by itself across calls of f
    // that hold ballots or atomic additions)
    int i = tid;
    for (; i + (kAhead - 1) * n_threads < n4; i += kAhead * n_threads) {
        float4 v[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) v[u] = p4[i + u * n_threads];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int j = head + 4 * (i + u * n_threads);
            f(j, v[u].x);
            f(j + 1, v[u].y);
            f(j + 2, v[u].z);
            f(j + 3, v[u].w);
        }
    }
    for (; i < n4; i += n_threads) {
        const float4 v = p4[i];
        const int j = head + 4 * i;
        f(j, v.x);
        f(j + 1, v.y);
        f(j + 2, v.z);
        f(j + 3, v.w);
    }
    for (int j = head + 4 * n4 + tid; j < n; j += n_threads) f(j, p[j]);
}

// lowest index among equal maxima (/root/reference/src/sampler.cpp:13-20: std::max_element)
__device__ __forceinline__ void argmax_combine(float& v, int& i, float ov, int oi) {
    if (ov > v || (ov == v && oi < i)) {
        v = ov;
        i = oi;
    }
}

// The row's best token and its value (every thread); kNoToken and -infinity where there is nothing but NaN.
struct BestToken {
    int index;
    float value;
};
constexpr int kNoToken = 0x7fffffff;
__device__ BestToken block_argmax(const float* __restrict__ row, int vocab, float* s_val, int* s_idx) {
    float best = -INFINITY;
    int best_i = kNoToken;
    for_each_in_row(row, vocab, threadIdx.x, blockDim.x, [&](int j, float v) {
        if (v > best || (v == best && j < best_i)) {
            best = v;
            best_i = j;
        }
    });
#pragma unroll
    for (int o = kWave / 2; o > 0; o >>= 1) {
        const float ov = __shfl_xor(best, o, kWave);
        const int oi = __shfl_xor(best_i, o, kWave);
        argmax_combine(best, best_i, ov, oi);
    }
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    __syncthreads();
    if (lane == 0) {
        s_val[wave] = best;
        s_idx[wave] = best_i;
    }
    __syncthreads();
    const int n_waves = (blockDim.x + kWave - 1) / kWave;
    best = s_val[0];
    best_i = s_idx[0];
    for (int w = 1; w < n_waves; ++w) argmax_combine(best, best_i, s_val[w], s_idx[w]);
    return {best_i, best};
}

// weight of token j: exp((x_j - max) / T), in [0, 1]
__device__ __forceinline__ float weight_of(float x, float mx, float inv_t) { return expf((x - mx) * inv_t); }

// Fixed-point image of a weight in [0, 1] (40 fractional bits, what is below them cut off): sums of these are integers, so a sum over the
// row does not depend on the order in which threads add, and neither does any decision taken from it.
__device__ __forceinline__ unsigned long long fixed_of(float w) {
    const uint32_t bits = __float_as_uint(w), exponent = bits >> 23;         // (127: a weight of 1)
    return (static_cast<unsigned long long>(bits & 0x007fffffu | 0x00800000u) << 17) >> min(63u, 127u - exponent);
}

// The largest bit pattern tau with count(w >= tau) >= need (non-negative floats order like their bits): radix
// selection, eight bits a level, histogram in LDS.  The weights of a row crowd into a few exponents, so the
// lanes of a wavefront that hit the same bin first agree on one addition (a ballot and a population count).
// The weights come from each(f), which calls f(index, weight) once for everyone of them, spread over the workgroup's threads.
template <typename Each>
__device__ uint32_t select_by_count(Each each, unsigned int need, unsigned int* hist, uint32_t* shared_prefix, unsigned int* shared_need) {
    uint32_t prefix = 0u, mask = 0u;
    const int lane = threadIdx.x % kWave;
    int first_level = 3;
    {
        // The highest digit of a weight's pattern is its exponent (two exponents a bin), and the k-th largest
        // weight is almost always within 2^-15 of the largest (1.0, digit 0x3f): count those eight bins in
        // registers.  If the k-th weight is smaller still, the general histogram below takes over.
        unsigned int c[8] = {0u, 0u, 0u, 0u, 0u, 0u, 0u, 0u};
        each([&](int, float wj) {
            const uint32_t bits = __float_as_uint(wj);
            if (bits >= 0x38000000u) {
                const uint32_t d = 0x3fu - (bits >> 24);
#pragma unroll
                for (int i = 0; i < 8; ++i) c[i] += d == static_cast<uint32_t>(i) ? 1u : 0u;
            }
        });
        for (int i = threadIdx.x; i < 8; i += blockDim.x) hist[i] = 0u;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            unsigned int v = c[i];
#pragma unroll
            for (int o = kWave / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, kWave);
            if (lane == 0 && v) atomicAdd(&hist[i], v);          // integer sums: order does not matter
        }
        __syncthreads();
        if (threadIdx.x == 0) {
            unsigned int cum = 0u;
            int found = -1;
            for (int i = 0; i < 8; ++i) {
                if (cum + hist[i] >= need) {
                    found = i;
                    break;
                }
                cum += hist[i];
            }
            *shared_prefix = found >= 0 ? (0x3fu - found) << 24 : 0xffffffffu;
            *shared_need = found >= 0 ? need - cum : need;
        }
        __syncthreads();
        if (*shared_prefix != 0xffffffffu) {
            prefix = *shared_prefix;
            need = *shared_need;
            mask = 255u << 24;
            first_level = 2;
        }
        __syncthreads();
    }
    for (int level = first_level; level >= 0; --level) {
        const int shift = 8 * level;
        for (int i = threadIdx.x; i < 256; i += blockDim.x) hist[i] = 0u;
        __syncthreads();
        each([&](int, float wj) {
            const uint32_t bits = __float_as_uint(wj);
            const uint32_t bin = (bits & mask) == prefix ? (bits >> shift) & 255u : 0xffffffffu;
            unsigned long long todo = __ballot(bin != 0xffffffffu);      // over the lanes that are here
            while (todo) {
                const int leader = __ffsll(static_cast<long long>(todo)) - 1;
                const uint32_t b0 = __shfl(bin, leader, kWave);
                const unsigned long long same = __ballot(bin == b0);
                if (lane == leader) atomicAdd(&hist[b0], static_cast<unsigned int>(__popcll(same)));
                todo &= ~same;
            }
        });
        __syncthreads();
        if (threadIdx.x == 0) {
            unsigned int cum = 0u;
            int bin = 255;
            for (; bin > 0; --bin) {
                if (cum + hist[bin] >= need) break;
                cum += hist[bin];
            }
            *shared_prefix = prefix | (static_cast<uint32_t>(bin) << shift);
            *shared_need = need - cum;
        }
        __syncthreads();
        prefix = *shared_prefix;
        need = *shared_need;
        mask |= 255u << shift;
        __syncthreads();
    }
    return prefix;
}

// Among the weights >= lo, the largest bit pattern tau with mass(w >= tau) >= need: the smallest set of most likely tokens whose
// mass reaches need, ties at tau included whole.  In between, mass(w >= lo) >= need and mass(w >= hi) = above < need.  Each pass
// divides [lo, hi): weights that crowd into a few exponents by fifteen pivots, whose masses every thread sums in registers;
// after that by 64 bins in LDS (152,000 weights of a row that top-p alone cuts, four such passes: 540 -> 170 us a row, where
// seven passes of pivots walked it).  Masses are fixed-point integers, whose sums depend on no order.
template <typename Each>
__device__ uint32_t select_by_mass(Each each, uint32_t lo, uint32_t hi, unsigned long long above, unsigned long long need,
                                   unsigned long long* sums /* [16][15] */, uint32_t* shared_lo, uint32_t* shared_hi,
                                   unsigned long long* shared_above) {
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave, n_waves = blockDim.x / kWave;
    if (lo + 1u < hi && hi == 0x3f800001u && lo < 0x38000000u) {
        // pivots on exponent boundaries near 1.0, where the mass is
        const uint32_t base = 0x37000000u, step = 0x01000000u;       // pivot i = base + (i + 1) * step
        unsigned long long acc[15];
#pragma unroll
        for (int i = 0; i < 15; ++i) acc[i] = 0ull;
        each([&](int, float wj) {
            const uint32_t bits = __float_as_uint(wj);
            if (bits > base && bits < hi && bits >= lo) {             // only these can lie at or above a pivot
                const unsigned long long f = fixed_of(wj);
#pragma unroll
                for (int i = 0; i < 15; ++i) acc[i] += bits >= base + (i + 1) * step ? f : 0ull;
            }
        });
#pragma unroll
        for (int i = 0; i < 15; ++i) {
            unsigned long long v = acc[i];
#pragma unroll
            for (int o = kWave / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, kWave);
            if (lane == 0) sums[wave * 15 + i] = v;
        }
        __syncthreads();
        if (threadIdx.x == 0) {
            uint32_t new_lo = lo, new_hi = hi;
            unsigned long long new_above = above;
            for (int i = 0; i < 15; ++i) {
                const uint32_t pivot = base + (i + 1) * step;
                if (pivot >= hi) break;
                if (pivot <= lo) continue;
                unsigned long long mass = above;
                for (int wv = 0; wv < n_waves; ++wv) mass += sums[wv * 15 + i];
                if (mass >= need) {
                    new_lo = pivot;
                } else {
                    new_hi = pivot;
                    new_above = mass;
                    break;
                }
            }
            *shared_lo = new_lo;
            *shared_hi = new_hi;
            *shared_above = new_above;
        }
        __syncthreads();
        lo = *shared_lo;
        hi = *shared_hi;
        above = *shared_above;
        __syncthreads();
    }
    while (lo + 1u < hi) {                           // (every pass leaves at most 1 / 32 of the range, and one pattern in the end)
        const int width = 32 - __clz(static_cast<int>(hi - lo - 1u));
        const int shift = width > 6 ? width - 6 : 0;
        if (threadIdx.x < kWave) sums[threadIdx.x] = 0ull;
        __syncthreads();
        each([&](int, float wj) {
            const uint32_t bits = __float_as_uint(wj);
            if (bits >= lo && bits < hi) atomicAdd(&sums[(bits - lo) >> shift], fixed_of(wj));
        });
        __syncthreads();
        if (threadIdx.x < kWave) {
            const int bin = kWave - 1 - lane;        // from the greatest weights down
            const unsigned long long mine = sums[bin];
            unsigned long long incl = mine;
#pragma unroll
            for (int o = 1; o < kWave; o <<= 1) {
                const unsigned long long up = __shfl_up(incl, o, kWave);
                if (lane >= o) incl += up;
            }
            const unsigned long long reached = __ballot(above + incl >= need);
            const int holder = reached ? __ffsll(static_cast<long long>(reached)) - 1 : kWave - 1;
            if (lane == holder) {
                *shared_lo = lo + (static_cast<uint32_t>(bin) << shift);
                *shared_hi = min(hi, lo + (static_cast<uint32_t>(bin + 1) << shift));
                *shared_above = above + incl - mine;
            }
        }
        __syncthreads();
        lo = *shared_lo;
        hi = *shared_hi;
        above = *shared_above;
        __syncthreads();
    }
    return lo;
}

}  // namespace egpt
