// Sampling with min-p: of what top-k and top-p keep, the tokens at least min_p times as likely as the most likely one.
//
// With weights w_j = exp((x_j - max) / T), which are at most 1, a token passes iff w_j >= min_p: a bound on the logit, max + T ln min_p,
// that needs no search and leaves a few dozen tokens of a model's distribution.  So the row is read once: a workgroup takes it in parts of 1,024
// threads' registers, knows the greatest logit so far behind one barrier a part, and lists the tokens that reach the bound below it (the
// bound only rises: what is listed holds every token of the end).  Top-k needs the k-th largest weight: the k-th largest of
// the threads' own maxima of the first part is no larger, and stands in the same comparison.  Top-p without top-k refers to the mass of the whole
// row: added up along the way, scaled to the greatest logit so far.  All cuts and the draw then run on the list, as searches for the bin that holds a
// count or a mass.  Rows that leave too long a list (nearly flat ones; top-p alone with a min_p of 0) are walked again for each threshold.
//
// What bounds it: for many rows the one pass over the logits; for a few the part's chain of load, maximum, barrier, comparison on the one unit that has the row.
#include "api.h"
#include "common.h"
#include "sampling.h"

namespace egpt {

constexpr int kListed = 4096;                      // tokens that a row's list holds
constexpr int kWaves = kSampleThreads / kWave;

// A part of a row, kQuads * 4 logits a thread; NaN where there is none.
template <int kQuads>
__device__ __forceinline__ void load_part(const float* __restrict__ row, int before /* floats between 16 bytes and the row */, int vocab, int part,
                                          float4 (&v)[kQuads]) {
    const float4* quads = reinterpret_cast<const float4*>(row - before);
#pragma unroll
    for (int i = 0; i < kQuads; ++i) {
        const int first = (part * kQuads + i) * kSampleThreads, q = first + threadIdx.x, j = 4 * q - before;
        if ((4 * first >= before && 4 * (first + kSampleThreads) - before <= vocab) || (j >= 0 && j + 4 <= vocab)) {
            v[i] = quads[q];
        } else {
            auto at = [&](int t) { return static_cast<unsigned>(t) < static_cast<unsigned>(vocab) ? row[t] : NAN; };
            v[i] = float4{at(j), at(j + 1), at(j + 2), at(j + 3)};
        }
    }
}

constexpr int kBins = 256;

struct LeastSpace {
    uint32_t w[kListed];                             // the list, in no order: logits, then the patterns of their weights
    int token[kListed];
    float share[kSampleThreads], max[2][kWaves];
    unsigned long long mass[2][kBins];
    unsigned int count[2][kBins];
    double row_mass[kWaves];
    unsigned long long sums[kWaves * 15], above, need;
    unsigned int hist[256], bound, needed;
    float best_val[kWaves];
    int best_idx[kWaves], listed, best, pick, done;
    uint32_t lo, hi;
};

// The k-th largest of the maxima of shares of the threads (at least 2 k shares where there are as many threads), or -infinity: no larger than the row's k-th
// largest logit.
__device__ __forceinline__ float bound_by_count(float mine, int k, LeastSpace& s) {
    const int t = threadIdx.x;
    const int together = k <= 64 ? 8 : k <= 128 ? 4 : k <= 256 ? 2 : 1, shares = kSampleThreads / together;
    for (int o = 1; o < together; o <<= 1) mine = fmaxf(mine, __shfl_xor(mine, o, kWave));
    if (t % together == 0) s.share[t / together] = mine;
    if (t == 0) s.bound = 0xffffffffu;
    __syncthreads();
    if (t < shares) {
        mine = s.share[t];
        int greater = 0;
        for (int i = 0; i < shares / 4; ++i) {
            const float4 v = reinterpret_cast<const float4*>(s.share)[i];
            greater += (v.x > mine) + (v.y > mine) + (v.z > mine) + (v.w > mine);
        }
        const unsigned int bits = __float_as_uint(mine), order = bits & 0x80000000u ? ~bits : bits | 0x80000000u;
        if (greater < k) atomicMin(&s.bound, order);     // the least of those that fewer than k exceed
    }
    __syncthreads();
    const unsigned int order = s.bound;
    return __uint_as_float(order & 0x80000000u ? order & 0x7fffffffu : ~order);
}

// The sum over a wavefront's lanes up to each: rows of 16 lanes by shifts, then the rows before (vector instructions; a shuffle goes through LDS).
template <int CTRL, int ROWS>
__device__ __forceinline__ unsigned long long moved(unsigned long long v) {
    const int lo = __builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, ROWS, 0xf, ROWS == 0xf);
    const int hi = __builtin_amdgcn_update_dpp(0, static_cast<int>(v >> 32), CTRL, ROWS, 0xf, ROWS == 0xf);
    return static_cast<unsigned long long>(static_cast<uint32_t>(hi)) << 32 | static_cast<uint32_t>(lo);
}
__device__ __forceinline__ unsigned long long sum_up_to(unsigned long long v) {
    v += moved<0x111, 0xf>(v);
    v += moved<0x112, 0xf>(v);
    v += moved<0x114, 0xf>(v);
    v += moved<0x118, 0xf>(v);
    v += moved<0x142, 0xa>(v);
    v += moved<0x143, 0xc>(v);
    return v;
}

// Among the list's entries the greatest key of [lo, hi) whose mass with that of all greater keys reaches what need_of makes of the mass of all; lo if none
// does.  entry(j, key, mass): whether the j-th takes part (asked by the thread that has it, j modulo the threads).  Masses are integers, whose
// sums depend on no order.  Left in lo and hi: the bin of the last pass, which holds that key and no other.  Every pass counts 256 bins; few
// entries need more than two.  One set of bins is cleared while the other is looked at: `turn`, the one that is clear.
template <typename Entry, typename Need>
__device__ __forceinline__ void bound_in_list(int n, Entry entry, uint32_t& lo, uint32_t& hi, Need need_of, int& turn, LeastSpace& s) {
    const int lane = threadIdx.x % kWave;
    unsigned long long above = 0ull;
    for (bool first = true;; first = false) {
        const int width = 32 - __clz(static_cast<int>(hi - lo - 1u)), shift = width > 8 ? width - 8 : 0;
        unsigned long long* masses = s.mass[turn];
        unsigned int* counts = s.count[turn];
        turn ^= 1;
        for (int j = threadIdx.x; j < n; j += kSampleThreads) {
            uint32_t key;
            unsigned long long mass;
            if (entry(j, key, mass) && key >= lo && key < hi) {
                atomicAdd(&masses[(key - lo) >> shift], mass);
                atomicAdd(&counts[(key - lo) >> shift], 1u);
            }
        }
        __syncthreads();
        if (threadIdx.x < kWave) {
            const int top = kBins - 1 - 4 * lane;            // four bins a lane, from the greatest keys down
            unsigned long long mine[4], sum = 0ull;
#pragma unroll
            for (int i = 0; i < 4; ++i) sum += mine[i] = masses[top - i];
            const unsigned long long incl = sum_up_to(sum);
            unsigned long long need = s.need;
            if (first) need = need_of(static_cast<unsigned long long>(__builtin_amdgcn_readlane(static_cast<uint32_t>(incl >> 32), kWave - 1)) << 32 |
                                      static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<uint32_t>(incl), kWave - 1)));
            const unsigned long long reached = __ballot(above + incl >= need);
            if (lane == (reached ? __ffsll(static_cast<long long>(reached)) - 1 : 0)) {
                s.need = need;
                s.done = 1;
                s.lo = lo;
                s.hi = hi;
                if (reached) {
                    unsigned long long cum = above + incl - sum;
                    int bin = top;
#pragma unroll
                    for (int i = 0; i < 3; ++i)
                        if (bin == top - i && cum + mine[i] < need) {
                            cum += mine[i];
                            --bin;
                        }
                    s.lo = lo + (static_cast<uint32_t>(bin) << shift);
                    s.hi = min(hi, lo + (static_cast<uint32_t>(bin + 1) << shift));
                    s.above = cum;
                    s.done = shift == 0 || counts[bin] == 1u;
                }
            }
        } else if (threadIdx.x < kWave + kBins) {
            s.mass[turn][threadIdx.x - kWave] = 0ull;
            s.count[turn][threadIdx.x - kWave] = 0u;
        }
        __syncthreads();
        lo = s.lo;
        hi = s.hi;
        above = s.above;
        if (s.done) return;
    }
}

__device__ __forceinline__ unsigned long long needed_mass(float p, unsigned long long all) {
    return max(1ull, static_cast<unsigned long long>(static_cast<double>(p) * static_cast<double>(all)));
}
// The point of a mass that the uniform number names.
__device__ __forceinline__ unsigned long long drawn_point(float u, unsigned long long all) {
    const unsigned long long point = static_cast<unsigned long long>(static_cast<double>(fminf(fmaxf(u, 0.f), 0.99999994f)) * static_cast<double>(all));
    return all > 0ull && point >= all ? all - 1ull : point;
}

// The draw from a whole row's tokens at or above `threshold`, in masses of integers: every wavefront adds up a sixteenth of the row, all of them
// then runs of tokens of the sixteenth that holds the drawn point.  Returns the token (every thread).
__device__ __forceinline__ int draw_from_row(const float* __restrict__ row, int vocab, float mx, float inv_t, uint32_t threshold, float u, LeastSpace& s) {
    const int j = threadIdx.x, lane = j % kWave, wave = j / kWave;
    auto mass_of = [&](float x) {
        const float w = x <= mx ? weight_of(x, mx, inv_t) : 0.f;                    // (a NaN is no candidate)
        return __float_as_uint(w) >= threshold ? fixed_of(w) : 0ull;
    };
    const int sixteenth = (vocab + kWaves - 1) / kWaves, begin = min(vocab, wave * sixteenth);
    unsigned long long mine = 0ull;
    for_each_in_row<4>(row + begin, min(vocab, begin + sixteenth) - begin, lane, kWave, [&](int, float x) { mine += mass_of(x); });
#pragma unroll
    for (int o = kWave / 2; o > 0; o >>= 1) mine += __shfl_xor(mine, o, kWave);
    __syncthreads();
    if (lane == 0) s.sums[wave] = mine;
    if (j == 0) s.pick = 0;
    __syncthreads();
    unsigned long long total = 0ull;
    for (int i = 0; i < kWaves; ++i) total += s.sums[i];
    unsigned long long target = drawn_point(u, total);
    int owner = 0;
    while (owner < kWaves - 1 && target >= s.sums[owner]) target -= s.sums[owner++];
    const int from = min(vocab, owner * sixteenth), n = min(vocab, from + sixteenth) - from;
    const int run = (n + kSampleThreads - 1) / kSampleThreads, r_begin = min(n, j * run), r_end = min(n, r_begin + run);
    mine = 0ull;
    for (int i = r_begin; i < r_end; ++i) mine += mass_of(row[from + i]);
    unsigned long long incl = mine;
#pragma unroll
    for (int o = 1; o < kWave; o <<= 1) {
        const unsigned long long up = __shfl_up(incl, o, kWave);
        if (lane >= o) incl += up;
    }
    if (lane == kWave - 1) s.sums[kWaves + wave] = incl;
    __syncthreads();
    unsigned long long cum = incl - mine;
    for (int i = 0; i < wave; ++i) cum += s.sums[kWaves + i];
    if (cum <= target && target < cum + mine) {
        for (int i = r_begin; i < r_end; ++i) {
            cum += mass_of(row[from + i]);
            if (cum > target) {
                s.pick = from + i;
                break;
            }
        }
    }
    __syncthreads();
    return s.pick;
}

// kMore: the row has more than one part, and the next one is on its way while one is looked at.
template <int kQuads, bool kMore>
__global__ __launch_bounds__(kSampleThreads, kMore ? 4 : 8) void sample_least_kernel(
    const float* __restrict__ logits, const float* __restrict__ temperature, const int32_t* __restrict__ top_k, const float* __restrict__ top_p,
    const float* __restrict__ min_p, const float* __restrict__ uniform, int32_t* __restrict__ out, int vocab) {
    __shared__ __attribute__((aligned(16))) LeastSpace s;
    const int r = blockIdx.x, lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    const float* row = logits + static_cast<size_t>(r) * vocab;
    const int before = static_cast<int>(reinterpret_cast<uintptr_t>(row) >> 2 & 3u);
    float4 v[kQuads], next[kMore ? kQuads : 1];
    load_part(row, before, vocab, 0, v);
    const float temp = temperature[r], p = top_p[r], u = uniform[r], given = min_p[r];
    const int k = top_k[r];
    const float least = given > 0.f ? fminf(given, 1.0f) : 0.f;                     // (a NaN cuts nothing; the most likely tokens always stay)
    const bool greedy = !(temp > 0.f);
    const bool cut_by_count = k > 0 && k < vocab, cut_by_mass = p > 0.f && p < 1.f;
    const float t = fmaxf(temp, 1e-6f), inv_t = 1.0f / t;
    // What is listed: the tokens of a weight of at least `floor`, by a bound on the logit that stands a thousandth lower than it (the weight's argument, below
    // 2^7, is rounded twice), and of the k largest.  top-p behind top-k refers to the mass of all k.  A short row is listed whole, a greedy one's maxima, and those
    // of a row that nothing of it bounds.
    const float floor = cut_by_count && cut_by_mass ? 0.f : least;
    const bool whole = !greedy && vocab <= kSampleThreads, count_bounds = !greedy && !whole && cut_by_count && k <= kSampleThreads;
    const bool lists = !greedy && (whole || count_bounds || floor > 0.f);
    const float reach = !lists ? 0.f : whole || floor == 0.f ? -INFINITY : (logf(floor) - 1e-3f) * t;
    const bool sums_mass = lists && cut_by_mass && !cut_by_count;
    const float per_log2 = inv_t * 1.44269504f;
    if (threadIdx.x == 0) {
        s.listed = 0;
        s.best = kNoToken;
    }
    if (threadIdx.x < kBins) {
        s.mass[0][threadIdx.x] = 0ull;
        s.count[0][threadIdx.x] = 0u;
    }
    float mx = -INFINITY, k_bound = -INFINITY;
    double mass = 0.0;
    const int parts = kMore ? (vocab + before + 4 * kQuads * kSampleThreads - 1) / (4 * kQuads * kSampleThreads) : 1;
    for (int part = 0; part < parts; ++part) {
        if constexpr (kMore) {
            if (part + 1 < parts) load_part(row, before, vocab, part + 1, next);
        }
        float mine = -INFINITY;
#pragma unroll
        for (int i = 0; i < kQuads; ++i) mine = fmaxf(fmaxf(fmaxf(mine, v[i].x), fmaxf(v[i].y, v[i].z)), v[i].w);        // (past NaN)
        const float of_wave = wave_max(mine);
        if (lane == 0) s.max[part & 1][wave] = of_wave;
        __syncthreads();
        const float was = mx;
        mx = fmaxf(mx, fold_row(s.max[part & 1][lane % kWaves], MaxOf()));
        if (part == 0 && count_bounds) k_bound = bound_by_count(mine, k, s);
        if (sums_mass && mx > -INFINITY) {
            float sum = 0.f;
            auto share = [&](float x) { return __builtin_amdgcn_exp2f((fmaxf(x, -INFINITY) - mx) * per_log2); };
#pragma unroll
            for (int i = 0; i < kQuads; ++i) sum += (share(v[i].x) + share(v[i].y)) + (share(v[i].z) + share(v[i].w));
            mass = mass * static_cast<double>(__builtin_amdgcn_exp2f((was - mx) * per_log2)) + static_cast<double>(sum);
        }
        const float bound = fmaxf(k_bound, mx + reach);
        if (__any(mine >= bound)) {                          // a wavefront's tokens take places together
            unsigned long long in[4 * kQuads];
            int found = 0;
#pragma unroll
            for (int i = 0; i < 4 * kQuads; ++i) {
                in[i] = __ballot((&v[i / 4].x)[i % 4] >= bound);
                found += __popcll(in[i]);
            }
            int at = 0;
            if (lane == 0) at = atomicAdd(&s.listed, found);
            at = __builtin_amdgcn_readfirstlane(at);
            if (at + found <= kListed) {
#pragma unroll
                for (int i = 0; i < 4 * kQuads; ++i) {
                    if (in[i] == 0ull) continue;
                    if (in[i] >> lane & 1ull) {
                        const int to = at + __popcll(in[i] & ((1ull << lane) - 1ull));
                        s.w[to] = __float_as_uint((&v[i / 4].x)[i % 4]);
                        s.token[to] = 4 * ((part * kQuads + i / 4) * kSampleThreads + static_cast<int>(threadIdx.x)) - before + i % 4;
                    }
                    at += __popcll(in[i]);
                }
            }
        }
        if constexpr (kMore) {
#pragma unroll
            for (int i = 0; i < kQuads; ++i) v[i] = next[i];
        }
    }
    unsigned long long row_mass = 0ull;
    if (sums_mass) {
#pragma unroll
        for (int o = kWave / 2; o > 0; o >>= 1) mass += __shfl_xor(mass, o, kWave);
        if (lane == 0) s.row_mass[wave] = mass;
    }
    __syncthreads();
    if (sums_mass) {
        mass = 0.0;
        for (int i = 0; i < kWaves; ++i) mass += s.row_mass[i];
        row_mass = static_cast<unsigned long long>(mass * 1099511627776.0);        // as fixed_of counts
    }
    const int listed = s.listed;
    const bool have_list = listed <= kListed && mx > -INFINITY;
    if (greedy || !(fabsf(mx) < INFINITY)) {                 // no draw: temperature <= 0, an infinity, nothing but NaN.  The row's best token
        int best = kNoToken;
        if (have_list) {
            for (int j = threadIdx.x; j < listed; j += kSampleThreads)
                if (__uint_as_float(s.w[j]) == mx) atomicMin(&s.best, s.token[j]);
            __syncthreads();
            best = s.best;
        } else {                                             // (more equals than a list holds, or not a number to list)
            best = block_argmax(row, vocab, s.best_val, s.best_idx).index;
        }
        if (threadIdx.x == 0) out[r] = best == kNoToken ? 0 : best;
        return;
    }
    // the kept tokens' weights reach all of: what top-k leaves, what top-p leaves of it, min_p
    uint32_t threshold = 0u;
    if (have_list && lists) {
        for (int j = threadIdx.x; j < listed; j += kSampleThreads) s.w[j] = __float_as_uint(weight_of(__uint_as_float(s.w[j]), mx, inv_t));
        int turn = 0;
        constexpr uint32_t kTop = 0x3f800001u;
        // (the exponential may be off by a unit either way: 2^-18 below the bound is below all that is listed)
        const float bound = fmaxf(count_bounds ? weight_of(k_bound, mx, inv_t) : 0.f, floor) * (1.0f - 3.8147e-6f);
        const uint32_t least_listed = max(1u, __float_as_uint(bound));
        threshold = least_listed;
        uint32_t hi = kTop;
        if (cut_by_count) {
            bound_in_list(listed, [&](int j, uint32_t& key, unsigned long long& mass) { key = s.w[j]; mass = 1ull; return true; }, threshold, hi,
                          [&](unsigned long long) { return static_cast<unsigned long long>(k); }, turn, s);
            hi = kTop;
        }
        if (cut_by_mass) {
            bound_in_list(listed, [&](int j, uint32_t& key, unsigned long long& mass) { key = s.w[j]; mass = fixed_of(__uint_as_float(key)); return true; },
                          threshold, hi, [&](unsigned long long all) { return needed_mass(p, cut_by_count ? all : row_mass); }, turn, s);
        }
        threshold = max(threshold, __float_as_uint(least));
        // in the order of the tokens: the greatest of the numbers counted from the row's end
        uint32_t lo = 0u;
        hi = static_cast<uint32_t>(vocab);
        auto kept = [&](int j, uint32_t& key, unsigned long long& mass) {
            key = static_cast<uint32_t>(vocab - 1 - s.token[j]);
            mass = fixed_of(__uint_as_float(s.w[j]));
            return s.w[j] >= threshold;
        };
        bound_in_list(listed, kept, lo, hi, [&](unsigned long long all) { return drawn_point(u, all) + 1ull; }, turn, s);
        for (int j = threadIdx.x; j < listed; j += kSampleThreads) {
            uint32_t key;
            unsigned long long mass;
            if (kept(j, key, mass) && key >= lo && key < hi) out[r] = s.token[j];       // (one token, the most likely ones being kept)
        }
    } else {
        auto each = [&](auto f) {
            for_each_in_row<4>(row, vocab, threadIdx.x, kSampleThreads, [&](int j, float x) { f(j, x <= mx ? weight_of(x, mx, inv_t) : 0.f); });
        };
        __syncthreads();
        if (cut_by_count) threshold = select_by_count(each, static_cast<unsigned int>(k), s.hist, &s.lo, &s.needed);
        if (cut_by_mass) {
            unsigned long long mine = 0ull;
            each([&](int, float w) {
                if (__float_as_uint(w) >= threshold) mine += fixed_of(w);
            });
#pragma unroll
            for (int o = kWave / 2; o > 0; o >>= 1) mine += __shfl_xor(mine, o, kWave);
            if (lane == 0) s.sums[wave] = mine;
            __syncthreads();
            unsigned long long all = 0ull;
            for (int i = 0; i < kWaves; ++i) all += s.sums[i];
            __syncthreads();
            threshold = select_by_mass(each, threshold, 0x3f800001u, 0ull, needed_mass(p, all), s.sums, &s.lo, &s.hi, &s.above);
        }
        const int picked = draw_from_row(row, vocab, mx, inv_t, max(threshold, __float_as_uint(least)), u, s);
        if (threadIdx.x == 0) out[r] = picked;
    }
}

}  // namespace egpt

using namespace egpt;

extern "C" int egpt_sample_min_p(const float* logits, const float* temperature, const int32_t* top_k, const float* top_p, const float* min_p,
                                 const float* uniform, int32_t* out, int n_rows, int vocab, void* stream) {
    if (!logits || !temperature || !top_k || !top_p || !min_p || !uniform || !out || n_rows < 0 || vocab <= 0) return EGPT_BAD_ARGUMENT;
    if (vocab >= 1 << 23) return EGPT_UNSUPPORTED_SIZE;      // (masses in 64 bits, 40 behind the point)
    if (n_rows == 0) return EGPT_OK;
    hipStream_t st = static_cast<hipStream_t>(stream);
    // (three floats more: where a row begins between 16 bytes)
    if (vocab + 3 <= 8 * kSampleThreads)                     // a part of two quads a thread
        sample_least_kernel<2, false><<<n_rows, kSampleThreads, 0, st>>>(logits, temperature, top_k, top_p, min_p, uniform, out, vocab);
    else if (vocab + (vocab % 4 == 0 && (reinterpret_cast<uintptr_t>(logits) & 15) == 0 ? 0 : 3) <= 32 * kSampleThreads)
        sample_least_kernel<8, false><<<n_rows, kSampleThreads, 0, st>>>(logits, temperature, top_k, top_p, min_p, uniform, out, vocab);
    else
        sample_least_kernel<8, true><<<n_rows, kSampleThreads, 0, st>>>(logits, temperature, top_k, top_p, min_p, uniform, out, vocab);
    EGPT_CHECK_LAUNCH();
    return EGPT_OK;
}
