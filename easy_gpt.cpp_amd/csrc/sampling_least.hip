// Sampling with min-p: of what top-k and top-p keep, the tokens at least min_p times as likely as the most likely one.
//
// With weights w_j = exp((x_j - max) / T), which are at most 1, a token passes iff w_j >= min_p: a bound on the logit, max + T ln min_p,
// that needs no search and leaves a few dozen tokens of a model's distribution.  So a row is read once, into the registers of one workgroup or, a long one,
// of several: the greatest logit is known behind one barrier, the tokens that reach the bound below it go to a list.  Top-k needs the k-th
// largest weight: the k-th largest of the threads' own maxima is no larger, and stands in the same comparison.  Top-p without top-k refers to the
// mass of the whole row, added up from the registers too, in 32 bits a thread and 64 beyond; where that leaves in doubt which tokens reach top_p, the row is
// walked with masses in integers, as the kernels without min-p have them.  All cuts and the draw then run on the list, as searches for the bin that holds a count or a mass.
// A row in pieces leaves a list, a maximum and a mass for each, and a second kernel joins them: the pieces' bounds are lower than the row's, so their
// lists hold what the row's does.  Rows that leave too long a list (nearly flat ones; top-p alone with a min_p of 0) are walked again for each threshold.
//
// What bounds it: for many rows the one pass over the logits (1,024 rows of 32,768 with top-p and min-p: 30.1 us, 4.5 TB/s, where a copy reaches 5.1;
// 254 by the kernels that count and list in passes of their own, with a workgroup's list of hundreds compared pair by pair); for a few the chain of a load, a
// dozen barriers and a second launch (1 row of 151,936 7.9 us, where an almost empty row of 650 takes 6.6 by one launch; 64 rows with all three cuts 19.4).
// Rows without a usable bound: 64 of 151,936 with top-p alone 263 us, a min_p of 10^-6 45.
#include "api.h"
#include "common.h"
#include "sampling.h"

namespace egpt {

constexpr int kListed = 4096;                      // tokens that a row's list holds
constexpr int kWaves = kSampleThreads / kWave;

// Logits first_quad * 4 on of a row that begins `before` floats behind 16 bytes, kQuads * 4 a thread; NaN from logit `end` on and before the row.  Reads are of
// the 16 bytes that hold a logit of the row, by loads that the hardware keeps to them: all of a thread's are asked for before the first is looked at (with
// branches for the ends they waited for each other: 1,024 rows of 32,768, 33.1 -> 30.2 us).
template <int kQuads>
__device__ __forceinline__ void load_part(const float* __restrict__ row, int before, int end, int first_quad, float4 (&v)[kQuads]) {
    const auto held = __builtin_amdgcn_make_buffer_rsrc(const_cast<float*>(row - before), 0, (before + end + 3) / 4 * 16, 0x00020000);
#pragma unroll
    for (int i = 0; i < kQuads; ++i)
        v[i] = __builtin_bit_cast(float4, __builtin_amdgcn_raw_buffer_load_b128(held, (first_quad + i * kSampleThreads + static_cast<int>(threadIdx.x)) * 16, 0, 0));
    if (4 * first_quad >= before && 4 * (first_quad + kQuads * kSampleThreads) - before <= end) return;
#pragma unroll
    for (int i = 0; i < kQuads; ++i) {
        const int j = 4 * (first_quad + i * kSampleThreads + static_cast<int>(threadIdx.x)) - before;
        auto only = [&](float x, int t) { return t >= 0 && t < end ? x : NAN; };
        v[i] = float4{only(v[i].x, j), only(v[i].y, j + 1), only(v[i].z, j + 2), only(v[i].w, j + 3)};
    }
}

// What a row is cut by.  Its list holds the tokens of a weight of at least `floor`, by a bound on the logit, max + reach, and of the k largest; either bound
// stands a thousandth of the temperature lower (a weight's argument, below 2^7, is rounded twice, and equal weights are kept together).  top-p behind top-k refers to the mass of all k.  A short row is listed
// whole, a greedy one's maxima, and those of a row that nothing of it bounds.
struct RowCuts {
    float p, u, least, floor, inv_t, reach, slack;
    int k;
    bool greedy, by_count, by_mass, count_bounds, lists, sums_mass;
};
__device__ __forceinline__ RowCuts cuts_of(int r, const float* __restrict__ temperature, const int32_t* __restrict__ top_k,
                                           const float* __restrict__ top_p, const float* __restrict__ min_p, const float* __restrict__ uniform, int vocab) {
    RowCuts c;
    const float temp = temperature[r], given = min_p[r], t = fmaxf(temp, 1e-6f);
    c.p = top_p[r];
    c.u = uniform[r];
    c.k = top_k[r];
    c.least = given > 0.f ? fminf(given, 1.0f) : 0.f;        // (a NaN cuts nothing; the most likely tokens always stay)
    c.greedy = !(temp > 0.f);
    c.inv_t = 1.0f / t;
    c.by_count = c.k > 0 && c.k < vocab;
    c.by_mass = c.p > 0.f && c.p < 1.f;
    c.floor = c.by_count && c.by_mass ? 0.f : c.least;
    const bool whole = !c.greedy && vocab <= kSampleThreads;
    c.count_bounds = !c.greedy && !whole && c.by_count && c.k <= kSampleThreads;
    c.lists = !c.greedy && (whole || c.count_bounds || c.floor > 0.f);
    c.reach = !c.lists ? 0.f : whole || c.floor == 0.f ? -INFINITY : (logf(c.floor) - 1e-3f) * t;
    c.slack = 1e-3f * t;
    c.sums_mass = c.lists && c.by_mass && !c.by_count;
    return c;
}

constexpr int kBins = 256;

struct LeastSpace {
    uint32_t w[kListed];                             // the list, in no order: logits, then the patterns of their weights
    int token[kListed];
    float max[kWaves], min[kWaves];
    unsigned long long mass[2][kBins];
    unsigned int count[2][kBins];
    double row_mass[kWaves];
    unsigned long long sums[kWaves * 15], above, within, need;
    unsigned int hist[256], needed;
    float k_bound;
    float best_val[kWaves];
    int best_idx[kWaves], listed, best, pick, done;
    uint32_t lo, hi;
};

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
// entries need more than two.  One set of bins is cleared while the other is looked at: `turn`, the one that is clear.  BORDERS: the masses of all greater keys
// and of that key are left in s.above and s.within (where none reaches the need, the mass of all, and more than any need).
template <bool BORDERS, typename Entry, typename Need>
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
            unsigned long long all = 0ull;
            if (first) {
                all = static_cast<unsigned long long>(__builtin_amdgcn_readlane(static_cast<uint32_t>(incl >> 32), kWave - 1)) << 32 |
                      static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<uint32_t>(incl), kWave - 1));
                need = need_of(all);
            }
            const unsigned long long reached = __ballot(above + incl >= need);
            if (lane == (reached ? __ffsll(static_cast<long long>(reached)) - 1 : 0)) {
                s.need = need;
                s.done = 1;
                s.lo = lo;
                s.hi = hi;
                if constexpr (BORDERS) {                     // (for as long as nothing reaches it: in the first pass or never)
                    s.above = all;
                    s.within = 1ull << 63;
                }
                if (reached) {
                    unsigned long long cum = above + incl - sum;
                    [[maybe_unused]] unsigned long long within = mine[0];
                    int bin = top;
#pragma unroll
                    for (int i = 0; i < 3; ++i)
                        if (bin == top - i && cum + mine[i] < need) {
                            cum += mine[i];
                            within = mine[i + 1];
                            --bin;
                        }
                    if constexpr (BORDERS) s.within = within;
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

// The sum of a workgroup's numbers, in an order of its own (every thread).
__device__ __forceinline__ double sum_of_all(double v, LeastSpace& s) {
#pragma unroll
    for (int o = kWave / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, kWave);
    if (threadIdx.x % kWave == 0) s.row_mass[threadIdx.x / kWave] = v;
    __syncthreads();
    v = 0.0;
    for (int i = 0; i < kWaves; ++i) v += s.row_mass[i];
    return v;
}
__device__ __forceinline__ float max_of_all(float v, LeastSpace& s) {
    v = wave_max(v);
    if (threadIdx.x % kWave == 0) s.max[threadIdx.x / kWave] = v;
    __syncthreads();
    return fold_row(s.max[threadIdx.x % kWaves], MaxOf());
}
__device__ __forceinline__ void clear(LeastSpace& s) {
    if (threadIdx.x == 0) {
        s.listed = 0;
        s.best = kNoToken;
    }
    if (threadIdx.x < kBins) {
        s.mass[0][threadIdx.x] = 0ull;
        s.count[0][threadIdx.x] = 0u;
    }
}
// A bound that the k-th largest of the threads' numbers, and so of all that they are the maxima of, reaches: the foot of the bin that holds it, of 256 between
// the least and `most`, the greatest; -infinity if there are fewer than k.  (A thousandth of a bin lower, for what rounding moves.)  Uses the
// histogram that the cuts begin with, and leaves it clear.
__device__ __forceinline__ float bound_by_count(float mine, float most, int k, LeastSpace& s) {
    const int lane = threadIdx.x % kWave;
    float least = -wave_max(mine > -INFINITY ? -mine : -INFINITY);
    if (lane == 0) s.min[threadIdx.x / kWave] = least;
    __syncthreads();
    least = -fold_row(-s.min[threadIdx.x % kWaves], MaxOf());
    const float range = most - least;
    if (!(range < INFINITY)) return -INFINITY;               // (an infinity, or nothing at all)
    // (a range that has no reciprocal is one bin: all of them are beyond its foot)
    const float per_bin = range * (1.0f / (kBins - 1)), bins = range > 1e-30f ? (kBins - 1) / range : 0.f;
    if (mine > -INFINITY) atomicAdd(&s.count[0][min(kBins - 1, static_cast<int>((mine - least) * bins))], 1u);
    __syncthreads();
    if (threadIdx.x < kWave) {
        const int top = kBins - 1 - 4 * lane;
        unsigned int mine4[4], sum = 0u;
#pragma unroll
        for (int i = 0; i < 4; ++i) sum += mine4[i] = s.count[0][top - i];
        unsigned int cum = static_cast<unsigned int>(sum_up_to(sum));
        const unsigned long long reached = __ballot(cum >= static_cast<unsigned int>(k));
        if (lane == (reached ? __ffsll(static_cast<long long>(reached)) - 1 : 0)) {
            cum -= sum;
            int bin = top;
#pragma unroll
            for (int i = 0; i < 3; ++i)
                if (bin == top - i && cum + mine4[i] < static_cast<unsigned int>(k)) {
                    cum += mine4[i];
                    --bin;
                }
            s.k_bound = reached ? least + (static_cast<float>(bin) - 1e-3f) * per_bin : -INFINITY;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) s.count[0][top - i] = 0u;
    }
    __syncthreads();
    return s.k_bound;
}
__device__ __forceinline__ float times_two_to(float x) { return __builtin_amdgcn_exp2f(x); }
constexpr float kLog2e = 1.44269504f;

// A part of a row: its greatest logit, a bound on its k-th largest, what the thread's logits add to the mass (weights relative to that
// greatest logit), the thread's own greatest.  put(place, logit, token) of what the bounds leave, s.listed of them in all; none of a wavefront's beyond `room`.
struct PartOfRow {
    float max, k_bound, mine;
    double mass;
};
template <int kQuads, typename Put>
__device__ __forceinline__ PartOfRow list_part(const float4 (&v)[kQuads], int first_token, const RowCuts& c, int room, LeastSpace& s, Put put) {
    const int lane = threadIdx.x % kWave;
    PartOfRow part{0.f, -INFINITY, -INFINITY, 0.0};
#pragma unroll
    for (int i = 0; i < kQuads; ++i) part.mine = fmaxf(fmaxf(fmaxf(part.mine, v[i].x), fmaxf(v[i].y, v[i].z)), v[i].w);      // (past NaN)
    part.max = max_of_all(part.mine, s);
    if (c.count_bounds) part.k_bound = bound_by_count(part.mine, part.max, c.k, s);
    if (c.sums_mass && part.max > -INFINITY) {
        const float per_log2 = c.inv_t * kLog2e;
        float sum = 0.f;
        auto share = [&](float x) { return times_two_to((fmaxf(x, -INFINITY) - part.max) * per_log2); };
#pragma unroll
        for (int i = 0; i < kQuads; ++i) sum += (share(v[i].x) + share(v[i].y)) + (share(v[i].z) + share(v[i].w));
        part.mass = static_cast<double>(sum);
    }
    const float bound = fmaxf(part.k_bound - c.slack, part.max + c.reach);
    // (a part of nothing but -infinity and NaN has no bound, and no candidates either)
    if (__any(part.mine >= bound && part.max > -INFINITY)) {     // a wavefront's tokens take places together
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
        if (at + found <= room) {
#pragma unroll
            for (int i = 0; i < 4 * kQuads; ++i) {
                if (in[i] == 0ull) continue;
                if (in[i] >> lane & 1ull)
                    put(at + __popcll(in[i] & ((1ull << lane) - 1ull)), (&v[i / 4].x)[i % 4],
                        first_token + 4 * ((i / 4) * kSampleThreads + static_cast<int>(threadIdx.x)) + i % 4);
                at += __popcll(in[i]);
            }
        }
    }
    return part;
}

// The cuts and the draw behind the list of a row (s.w, s.token; s.listed > kListed: there was no room for it).  row_mass: the whole row's, where c.sums_mass.
__device__ __forceinline__ void pick_of_row(const float* __restrict__ row, int vocab, const RowCuts& c, float mx, float k_bound, double mass, int32_t* out,
                                            LeastSpace& s) {
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    const float inv_t = c.inv_t;
    const int listed = s.listed;
    const bool have_list = listed <= kListed && mx > -INFINITY;
    if (c.greedy || !(fabsf(mx) < INFINITY)) {               // no draw: temperature <= 0, an infinity, nothing but NaN.  The row's best token
        int best = kNoToken;
        if (have_list) {
            for (int j = threadIdx.x; j < listed; j += kSampleThreads)
                if (__uint_as_float(s.w[j]) == mx) atomicMin(&s.best, s.token[j]);
            __syncthreads();
            best = s.best;
        } else {                                             // (more equals than a list holds, or not a number to list)
            best = block_argmax(row, vocab, s.best_val, s.best_idx).index;
        }
        if (threadIdx.x == 0) *out = best == kNoToken ? 0 : best;
        return;
    }
    // the kept tokens' weights reach all of: what top-k leaves, what top-p leaves of it, min_p
    uint32_t threshold = 0u;
    if (have_list && c.lists) {
        for (int j = threadIdx.x; j < listed; j += kSampleThreads) s.w[j] = __float_as_uint(weight_of(__uint_as_float(s.w[j]), mx, inv_t));
        int turn = 0;
        const unsigned long long row_mass = static_cast<unsigned long long>(mass * 1099511627776.0);      // as fixed_of counts
        constexpr uint32_t kTop = 0x3f800001u;
        // (the exponential may be off by a unit either way: 2^-18 below the bound is below all that is listed)
        const float bound = fmaxf(c.count_bounds ? weight_of(k_bound, mx, inv_t) : 0.f, c.floor) * (1.0f - 3.8147e-6f);
        const uint32_t least_listed = max(1u, __float_as_uint(bound));
        threshold = least_listed;
        uint32_t hi = kTop;
        if (c.by_count) {
            bound_in_list<false>(listed, [&](int j, uint32_t& key, unsigned long long& mass) { key = s.w[j]; mass = 1ull; return true; }, threshold, hi,
                                 [&](unsigned long long) { return static_cast<unsigned long long>(c.k); }, turn, s);
            hi = kTop;
        }
        bool sure = true;
        if (c.by_mass) {
            bound_in_list<true>(listed, [&](int j, uint32_t& key, unsigned long long& mass) { key = s.w[j]; mass = fixed_of(__uint_as_float(key)); return true; },
                                threshold, hi, [&](unsigned long long all) { return needed_mass(c.p, c.by_count ? all : row_mass); }, turn, s);
            // Whether the row's mass in integers says the same.  The sum is off by less than 2^-17 of it and 2^-40 a token: with A = -log2 w a weight's argument is off by
            // 0.69 A 2^-22 here and 0.69 A 2^-23 there, and the mean of A over a mass of 1 and more in N tokens is at most log2 N <= 23 (an entropy); exponentials by
            // 2^-21 together; a thread's sum takes 10 roundings of 2^-24, and an integer cuts off 2^-40.
            const unsigned long long doubt = (s.need >> 17) + static_cast<unsigned>(vocab);
            sure = !c.sums_mass || (s.above + doubt < s.need && s.need + doubt <= s.above + s.within);
        }
        threshold = max(threshold, __float_as_uint(c.least));
        // in the order of the tokens: the greatest of the numbers counted from the row's end
        uint32_t lo = 0u;
        hi = static_cast<uint32_t>(vocab);
        auto kept = [&](int j, uint32_t& key, unsigned long long& mass) {
            key = static_cast<uint32_t>(vocab - 1 - s.token[j]);
            mass = fixed_of(__uint_as_float(s.w[j]));
            return s.w[j] >= threshold;
        };
        bound_in_list<false>(listed, kept, lo, hi, [&](unsigned long long all) { return drawn_point(c.u, all) + 1ull; }, turn, s);
        for (int j = threadIdx.x; j < listed; j += kSampleThreads) {
            uint32_t key;
            unsigned long long mass;
            if (kept(j, key, mass) && key >= lo && key < hi) *out = s.token[j];       // (one token, the most likely ones being kept)
        }
        // (asked behind the draw: with a branch around it 1,024 rows of 32,768 took 31.0 us, 29.9 so)
        if (sure) return;
        __syncthreads();
    }
    // a list without room or bounds, or one whose border is in doubt: the row is walked
    threshold = 0u;
    auto each = [&](auto f) {
        for_each_in_row<4>(row, vocab, threadIdx.x, kSampleThreads, [&](int j, float x) { f(j, x <= mx ? weight_of(x, mx, inv_t) : 0.f); });
    };
    __syncthreads();
    if (c.by_count) threshold = select_by_count(each, static_cast<unsigned int>(c.k), s.hist, &s.lo, &s.needed);
    if (c.by_mass) {
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
        threshold = select_by_mass(each, threshold, 0x3f800001u, 0ull, needed_mass(c.p, all), s.sums, &s.lo, &s.hi, &s.above);
    }
    const int picked = draw_from_row(row, vocab, mx, inv_t, max(threshold, __float_as_uint(c.least)), c.u, s);
    if (threadIdx.x == 0) *out = picked;
}

// A row that one workgroup's registers hold.
template <int kQuads>
__global__ __launch_bounds__(kSampleThreads, 8) void sample_row_kernel(
    const float* __restrict__ logits, const float* __restrict__ temperature, const int32_t* __restrict__ top_k, const float* __restrict__ top_p,
    const float* __restrict__ min_p, const float* __restrict__ uniform, int32_t* __restrict__ out, int vocab, int others) {
    __shared__ __attribute__((aligned(16))) LeastSpace s;
    const int r = blockIdx.x;
    if (others && !(min_p[r] > 0.f)) return;
    const float* row = logits + static_cast<size_t>(r) * vocab;
    const int before = static_cast<int>(reinterpret_cast<uintptr_t>(row) >> 2 & 3u);
    float4 v[kQuads];
    load_part(row, before, vocab, 0, v);
    const RowCuts c = cuts_of(r, temperature, top_k, top_p, min_p, uniform, vocab);
    clear(s);
    const PartOfRow part = list_part(v, -before, c, kListed, s, [&](int place, float x, int token) {
        s.w[place] = __float_as_uint(x);
        s.token[place] = token;
    });
    double mass = 0.0;
    if (c.sums_mass) mass = sum_of_all(part.mass, s);
    __syncthreads();
    pick_of_row(row, vocab, c, part.max, part.k_bound, mass, out + r, s);
}

// A longer row's pieces, by a workgroup each: what the second kernel needs of them.
constexpr int kListedOfPiece = 1024;
struct PieceOfRow {
    double mass;
    float max, k_bound;
    int listed, unused;
};
// shares of a piece whose maxima it leaves: some 1,024 of a row
__device__ __forceinline__ int shares_of_piece(int pieces) { return pieces <= 16 ? 64 : pieces <= 32 ? 32 : 16; }
constexpr int kMostShares = 64;

// (what is asked for first stands in the arguments that arrive with the wavefronts)
template <int kQuads>
__global__ __launch_bounds__(kSampleThreads, 8) void sample_pieces_kernel(
    const float* __restrict__ logits, const float* __restrict__ temperature, const int32_t* __restrict__ top_k, const float* __restrict__ top_p,
    const float* __restrict__ min_p, int vocab, int quads_of_piece, int others, const float* __restrict__ uniform, PieceOfRow* __restrict__ found,
    float* __restrict__ maxima, uint2* __restrict__ lists) {
    __shared__ __attribute__((aligned(16))) LeastSpace s;
    const int r = blockIdx.x, piece = blockIdx.y, pieces = gridDim.y;
    if (others && !(min_p[r] > 0.f)) return;
    const size_t at = static_cast<size_t>(r) * pieces + piece;
    const float* row = logits + static_cast<size_t>(r) * vocab;
    const int before = static_cast<int>(reinterpret_cast<uintptr_t>(row) >> 2 & 3u);
    const int first_quad = piece * quads_of_piece, end = min(vocab, 4 * (first_quad + quads_of_piece) - before);
    float4 v[kQuads];
    load_part(row, before, end, first_quad, v);
    const RowCuts c = cuts_of(r, temperature, top_k, top_p, min_p, uniform, vocab);
    clear(s);
    uint2* list = lists + at * kListedOfPiece;
    const PartOfRow part = list_part(v, 4 * first_quad - before, c, kListedOfPiece, s, [&](int place, float x, int token) {
        list[place] = uint2{__float_as_uint(x), static_cast<uint32_t>(token)};
    });
    if (c.count_bounds) {
        const int together = kSampleThreads / shares_of_piece(pieces);
        float mine = part.mine;
        for (int o = 1; o < together; o <<= 1) mine = fmaxf(mine, __shfl_xor(mine, o, kWave));
        if (threadIdx.x % together == 0) maxima[at * kMostShares + threadIdx.x / together] = mine;
    }
    double mass = 0.0;
    if (c.sums_mass) mass = sum_of_all(part.mass, s);
    __syncthreads();
    if (threadIdx.x == 0) found[at] = PieceOfRow{mass, part.max, part.k_bound, s.listed, 0};
}

__global__ __launch_bounds__(kSampleThreads, 8) void sample_joined_kernel(
    const float* __restrict__ logits, const float* __restrict__ temperature, const int32_t* __restrict__ top_k, const float* __restrict__ top_p,
    const float* __restrict__ min_p, const float* __restrict__ uniform, int32_t* __restrict__ out, int vocab, int pieces,
    const PieceOfRow* __restrict__ found, const float* __restrict__ maxima, const uint2* __restrict__ lists, int others) {
    __shared__ __attribute__((aligned(16))) LeastSpace s;
    const int r = blockIdx.x, t = threadIdx.x, lane = t % kWave, wave = t / kWave;
    if (others && !(min_p[r] > 0.f)) return;
    const size_t at = static_cast<size_t>(r) * pieces;
    // What may be asked for at once is: a piece to a thread, and of its wavefront's two first pieces an entry to a lane (where the piece listed so many).
    const int last = pieces - 1, shares = shares_of_piece(pieces);
    const PieceOfRow mine = found[at + min(t, last)];
    const int of_wave = wave + kWaves * lane;
    int n_of_wave = of_wave <= last ? found[at + of_wave].listed : 0;
    const float max_of_wave = of_wave <= last ? found[at + of_wave].max : -INFINITY;
    uint2 early[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) early[i] = lists[(at + min(wave + kWaves * i, last)) * kListedOfPiece + lane];
    const RowCuts c = cuts_of(r, temperature, top_k, top_p, min_p, uniform, vocab);
    clear(s);
    const float mx = max_of_all(mine.max, s);
    float k_bound = -INFINITY;
    if (c.count_bounds) {
        k_bound = bound_by_count(t < pieces * shares ? maxima[(at + t / shares) * kMostShares + t % shares] : -INFINITY, mx, c.k, s);
        k_bound = fmaxf(k_bound, max_of_all(mine.k_bound, s));
    }
    double mass = 0.0;
    if (c.sums_mass) mass = sum_of_all(t <= last ? mine.mass * static_cast<double>(times_two_to((mine.max - mx) * (c.inv_t * kLog2e))) : 0.0, s);
    const float bound = fmaxf(k_bound - c.slack, mx + c.reach);
    // (a piece far below the row's maximum, masked by a large negative number or flat, listed by a bound of its own: nothing of it reaches the row's.
    // 64 rows of 151,936 with top-k, top-p and min-p, five sixths at -10^9: 20.1 us, 291 where such a piece's list counted; with min-p alone 14.2, 43.7)
    if (max_of_wave < bound) n_of_wave = 0;
    for (int i = 0; wave + kWaves * i <= last; ++i) {
        const int n = __builtin_amdgcn_readlane(n_of_wave, i);
        if (n > kListedOfPiece) {                            // more than its list holds, some of which the row's may need: the row is walked
            if (lane == 0) atomicAdd(&s.listed, kListed + 1);
            continue;
        }
        const uint2* list = lists + (at + wave + kWaves * i) * kListedOfPiece;
        for (int j0 = 0; j0 < n; j0 += kWave) {
            const int j = j0 + lane;
            uint2 e{0u, 0u};
            if (j0 == 0 && i < 2) e = i == 0 ? early[0] : early[1];
            else if (j < n) e = list[j];
            const unsigned long long in = __ballot(j < n && __uint_as_float(e.x) >= bound);
            if (in == 0ull) continue;
            int to = 0;
            if (lane == 0) to = atomicAdd(&s.listed, __popcll(in));
            to = __builtin_amdgcn_readfirstlane(to) + __popcll(in & ((1ull << lane) - 1ull));
            if ((in >> lane & 1ull) && to < kListed) {
                s.w[to] = e.x;
                s.token[to] = static_cast<int>(e.y);
            }
        }
    }
    __syncthreads();
    pick_of_row(logits + static_cast<size_t>(r) * vocab, vocab, c, mx, k_bound, mass, out + r, s);
}

}  // namespace egpt

using namespace egpt;

static size_t whole_blocks(size_t n) { return (n + 255) / 256 * 256; }

extern "C" size_t egpt_sample_min_p_workspace(int n_rows, int pieces) {
    if (n_rows <= 0 || pieces <= 1) return 0;
    const size_t n = static_cast<size_t>(n_rows) * pieces;
    return whole_blocks(n * sizeof(PieceOfRow)) + whole_blocks(n * kMostShares * 4) + n * kListedOfPiece * 8;
}

extern "C" int egpt_sample_min_p(const float* logits, const float* temperature, const int32_t* top_k, const float* top_p, const float* min_p,
                                 const float* uniform, int32_t* out, void* workspace, int n_rows, int vocab, int pieces, int others, void* stream) {
    if (!logits || !temperature || !top_k || !top_p || !min_p || !uniform || !out || n_rows < 0 || vocab <= 0 || pieces < 1 || (pieces > 1 && !workspace))
        return EGPT_BAD_ARGUMENT;
    if (vocab >= 1 << 23 || pieces > kSampleThreads) return EGPT_UNSUPPORTED_SIZE;         // (masses in 64 bits, 40 behind the point)
    // three floats more where a row may begin between 16 bytes
    const int quads = (vocab + (vocab % 4 == 0 && (reinterpret_cast<uintptr_t>(logits) & 15) == 0 ? 0 : 3) + 3) / 4;
    const int quads_of_piece = (quads + pieces - 1) / pieces;
    if (quads_of_piece > 8 * kSampleThreads) return EGPT_UNSUPPORTED_SIZE;
    if (n_rows == 0) return EGPT_OK;
    hipStream_t st = static_cast<hipStream_t>(stream);
    const bool small = quads_of_piece <= 2 * kSampleThreads;
    if (pieces == 1) {
        if (small) sample_row_kernel<2><<<n_rows, kSampleThreads, 0, st>>>(logits, temperature, top_k, top_p, min_p, uniform, out, vocab, others);
        else sample_row_kernel<8><<<n_rows, kSampleThreads, 0, st>>>(logits, temperature, top_k, top_p, min_p, uniform, out, vocab, others);
        EGPT_CHECK_LAUNCH();
        return EGPT_OK;
    }
    const size_t n = static_cast<size_t>(n_rows) * pieces;
    char* at = static_cast<char*>(workspace);
    PieceOfRow* found = reinterpret_cast<PieceOfRow*>(at);
    float* maxima = reinterpret_cast<float*>(at += whole_blocks(n * sizeof(PieceOfRow)));
    uint2* lists = reinterpret_cast<uint2*>(at + whole_blocks(n * kMostShares * 4));
    const dim3 grid(n_rows, pieces);
    auto launch = [&](auto kernel) {
        kernel<<<grid, kSampleThreads, 0, st>>>(logits, temperature, top_k, top_p, min_p, vocab, quads_of_piece, others, uniform, found, maxima, lists);
    };
    switch ((quads_of_piece + kSampleThreads - 1) / kSampleThreads) {       // (quads a thread)
        case 1:
        case 2: launch(sample_pieces_kernel<2>); break;
        case 3: launch(sample_pieces_kernel<3>); break;
        case 4: launch(sample_pieces_kernel<4>); break;
        case 5: launch(sample_pieces_kernel<5>); break;
        case 6: launch(sample_pieces_kernel<6>); break;
        default: launch(sample_pieces_kernel<8>);
    }
    EGPT_CHECK_LAUNCH();
    sample_joined_kernel<<<n_rows, kSampleThreads, 0, st>>>(logits, temperature, top_k, top_p, min_p, uniform, out, vocab, pieces, found, maxima, lists, others);
    EGPT_CHECK_LAUNCH();
    return EGPT_OK;
}
