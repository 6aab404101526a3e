// Attention for trees of drafted tokens over the paged cache.
//
// Request b brings n = q_len[b] nodes, whose keys and values are the last n of its kv_len[b] tokens in the cache.  Row (node i,
// query head h) reads key j of kv head h / (nq / nkv) where
//     j < kv - n   and, with a window, j > position_i - window     (the tokens before the tree)
//     j = kv - n + m   and bit m of visible_i is set                 (node m; a request has at most 64)
// and is softmax_j(scale q . k_j) v_j over those, zeros where there are none.  A number that a row does not see does not reach it, be it an
// infinity or a NaN.
//
// What bounds it, on the device alone: few rows, the chain of memory trips, a few rounds of keys and the join of the parts (1 user of 8 nodes behind 301 tokens at 14 heads on 2 of
// 64 7.1 us, 8 users of 16 behind 2,048 at 12 heads on 2 of 128 15.7); rows of small heads, the vector instructions of the softmax (64 users of 1 to 32
// nodes behind 128 to 4,001 at 14 heads on 2 of 64 32.6, 2.3 TB/s of keys and values); many rows, the matrix cores and the softmax, which overlap for 37 % of
// the products' time (2 users of 64 nodes behind 32,001 at 28 heads on 4 of 128 78, 750 TFLOP/s, where a library product reaches 1,400).
#include <atomic>
#include <type_traits>

#include "api.h"
#include "common.h"
#include "lds_loads.h"
#include "tree_loads.h"

namespace egpt {

constexpr int kMaxTreeHead = 256;
constexpr float kSlack = 8.0f;                   // how far, in powers of two, a row's maximum may run ahead of the one in use
constexpr float kFar = 4096.0f;                  // how large a maximum, as a power of two, may be for its product with the scale to be rounded
constexpr int kMostParts = 64;                   // of a request's keys: a lane each where they are joined

// One row's view of the keys: the tokens before the tree from `lo` on, and the nodes of its bits.
struct TreeRow {
    int lo, before, kv;
    unsigned long long bits;
    __device__ __forceinline__ bool sees(int j) const {
        if (j < before) return j >= lo;
        const int m = j - before;
        return j < kv && m < 64 && (bits >> m & 1ull) != 0;
    }
};

// Any head and page size: a workgroup of eight wavefronts per row, keys dealt out 64 at a
// time; a lane scores one key, then owns features lane, lane + 64, ...
constexpr int kTreeWaves = 8;
template <typename T>
__global__ __launch_bounds__(64 * kTreeWaves) void tree_attention_generic_kernel(
    const T* __restrict__ qkv, const int32_t* __restrict__ q_start, const int32_t* __restrict__ q_len, const int32_t* __restrict__ kv_len,
    const long long* __restrict__ visible, const int32_t* __restrict__ positions, int n_seqs, int window, const T* __restrict__ k_cache,
    const T* __restrict__ v_cache, const int32_t* __restrict__ block_table, int table_width, int n_pages, int nq, int nkv, int hd, int page_size,
    float scale, T* __restrict__ out) {
    constexpr int kOwn = kMaxTreeHead / kWave;
    __shared__ float q_s[kMaxTreeHead];
    __shared__ float part_ml[kTreeWaves][2];
    __shared__ float part_o[kTreeWaves][kMaxTreeHead];
    const int t = blockIdx.x, h = blockIdx.y, lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    int b = 0;                                               // the request that has token t: the last one that begins at or before it
    for (int lo = 0, hi = n_seqs - 1; lo < hi;) {
        const int mid = (lo + hi + 1) / 2;
        if (q_start[mid] <= t) lo = mid; else hi = mid - 1;
        b = lo;
    }
    const int n = q_len[b], qs = q_start[b], i = t - max(qs, 0);
    if (qs < 0 || i < 0 || i >= n) return;                   // nobody's row stays as it was
    const int kv = static_cast<int>(min(static_cast<long long>(kv_len[b]), static_cast<long long>(table_width) * page_size));
    const int before = kv_len[b] - n;
    const TreeRow row{window > 0 ? max(0, positions[t] - window + 1) : 0, before, kv, static_cast<unsigned long long>(visible[t])};
    const int kvh = h / (nq / nkv);
    const T* q = qkv + static_cast<size_t>(t) * (nq + 2 * nkv) * hd + h * hd;
    // (the scale is for differences of products alone, which are exact where large ones are near; a negative one turns the query)
    const float steep = fabsf(scale);
    for (int d = threadIdx.x; d < hd; d += kWave * kTreeWaves) q_s[d] = scale < 0.f ? -to_float(q[d]) : to_float(q[d]);
    __syncthreads();
    const int32_t* table = block_table + static_cast<size_t>(b) * table_width;
    const size_t head_size = static_cast<size_t>(page_size) * hd;
    float acc[kOwn] = {};
    float m_run = -INFINITY, l_run = 0.f;
    const int first = max(0, min(row.lo, before));
    for (int c = first + wave * kWave; c < kv; c += kWave * kTreeWaves) {
        const int j = c + lane;
        float s = -INFINITY;
        int page = -1;
        bool sees = row.sees(j) && j < kv;
        if (sees) {
            page = table[j / page_size];
            sees = page >= 0 && page < n_pages;
        }
        if (sees) {
            const T* kr = k_cache + (static_cast<size_t>(page) * nkv + kvh) * head_size + static_cast<size_t>(j % page_size) * hd;
            float dot = 0.f;
            for (int d = 0; d < hd; ++d) dot = fmaf(q_s[d], to_float(kr[d]), dot);
            s = dot;
        }
        const float m_new = fmaxf(m_run, wave_max(s));
        const float m_use = m_new == -INFINITY ? 0.f : m_new;
        const float pj = sees ? expf((s - m_use) * steep) : 0.f;
        const float alpha = m_run == -INFINITY ? 0.f : expf((m_run - m_use) * steep);
        l_run = l_run * alpha + wave_sum(pj);
        m_run = m_new;
#pragma unroll
        for (int r = 0; r < kOwn; ++r) acc[r] *= alpha;
        for (unsigned long long left = __ballot(sees); left != 0; left &= left - 1) {      // (a key that is not seen is not read)
            const int jj = __builtin_ctzll(left);
            const float pw = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(pj), jj));
            const int pg = __builtin_amdgcn_readlane(page, jj);
            const T* vr = v_cache + (static_cast<size_t>(pg) * nkv + kvh) * head_size + (c + jj) % page_size;
#pragma unroll
            for (int r = 0; r < kOwn; ++r) {
                const int d = lane + r * kWave;
                if (d < hd) acc[r] = fmaf(pw, to_float(vr[static_cast<size_t>(d) * page_size]), acc[r]);
            }
        }
    }
    if (lane == 0) {
        part_ml[wave][0] = m_run;
        part_ml[wave][1] = l_run;
    }
#pragma unroll
    for (int r = 0; r < kOwn; ++r)
        if (lane + r * kWave < hd) part_o[wave][lane + r * kWave] = acc[r];
    __syncthreads();
    if (wave != 0) return;
    float m_all = -INFINITY;
    for (int w = 0; w < kTreeWaves; ++w) m_all = fmaxf(m_all, part_ml[w][0]);
    float l_all = 0.f, share[kTreeWaves];
#pragma unroll
    for (int w = 0; w < kTreeWaves; ++w) {
        // (a wavefront that saw nothing weighs nothing; one whose scores are infinite or no number makes the row one)
        share[w] = part_ml[w][1] == 0.f ? 0.f : expf((part_ml[w][0] - m_all) * steep);
        l_all = fmaf(part_ml[w][1], share[w], l_all);
    }
    T* o = out + static_cast<size_t>(t) * nq * hd + h * hd;
#pragma unroll
    for (int r = 0; r < kOwn; ++r) {
        const int d = lane + r * kWave;
        if (d >= hd) continue;
        float a = 0.f;
#pragma unroll
        for (int w = 0; w < kTreeWaves; ++w) a = part_ml[w][1] == 0.f ? a : fmaf(part_o[w][d], share[w], a);
        o[d] = from_float<T>(l_all == 0.f ? 0.f : a / l_all);
    }
}


// ---- on the matrix cores: bfloat16 and float32, keys and values of whole 16 bytes, pages of multiples of 16 tokens
//
// Rows of one request and kv head, (node, head) pairs node-major, in blocks of 32, a block to a wavefront; RB wavefronts share a tile of KT keys, and KS such groups
// take every KS-th tile.  The scores come transposed, S^T[key, row] = K Q^T on 32 x 32 products, so that a lane has 16 of a block's 32 scores of ONE row (the lane 32
// further has the others): the softmax is arithmetic within a lane but for one exchange, and the probabilities lie as the second product, O^T += V^T P^T,
// takes them, without a trip through LDS.  An operand is 16 bytes a lane in either type: one product of bfloat16, 8 x 2 features of a row, four of
// float32, 4 x 2; the order of the summed index is free as long as both sides have the same, so bfloat16 reads the keys of a block with bits 2 and 3 of
// their number exchanged, which gives a lane eight neighbouring keys for the second product, as a page has a feature's values.
//
// Tiles go from memory straight to LDS, NS - 1 of them ahead of their use, one barrier a tile.  A load takes 1,024 bytes that lie in one page: a
// resource with that page's base, bounded by it, and a constant offset per lane.  Keys lie in rows, 16-byte pieces exchanged by the row's number, values as a page of 16
// tokens has them, halves exchanged by the feature's: either way lanes that read together read different banks.  A head that is no power of two is filled up with zeros by the loads' bounds.
//
// A head beyond 128 is more registers of queries and sums than a wavefront has: two share a block of rows, each with half of the features, and add up their halves of
// the scores through LDS, one barrier more a tile (float32, 7 requests of one node behind 1,246 tokens at 12 heads on 2 of 256: 71.6 us by one wavefront with its
// registers in memory, 28 so, and half the rounding error).
//
// A request's keys are cut into parts, a workgroup each, so that few requests fill the card and a long context does not make the others wait;
// parts leave the unnormalised result with its maximum and sum, and tree_combine_kernel joins them.
typedef __attribute__((ext_vector_type(8))) __bf16 tree_bf16x8;
typedef __attribute__((ext_vector_type(2))) __bf16 tree_bf16x2;
typedef __attribute__((ext_vector_type(16))) float f32x16;
typedef __attribute__((ext_vector_type(4))) float tree_f32x4;

template <typename T>
__device__ __forceinline__ f32x16 product_of(u32x4 a, u32x4 b, f32x16 c) {
    if constexpr (sizeof(T) == 2) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(tree_bf16x8, a), __builtin_bit_cast(tree_bf16x8, b), c, 0, 0, 0);
    } else {
        const tree_f32x4 x = __builtin_bit_cast(tree_f32x4, a), y = __builtin_bit_cast(tree_f32x4, b);
#pragma unroll
        for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(x[e], y[e], c, 0, 0, 0);
        return c;
    }
}

// All ones if bit `at` of x is set.
__device__ __forceinline__ unsigned bit_filled(unsigned x, int at) { return static_cast<unsigned>(static_cast<int>(x << (31 - at)) >> 31); }

constexpr int kGroup = 16;                       // keys that a load's base is found for: never more than a page's

#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"        // (m0 is a reserved register; nothing else here uses it)
// 16 bytes a lane from byte `offset` + `more` of a resource to LDS, at address `to` (the same for the whole wavefront) + 16 x lane; zeros past its end.
__device__ __forceinline__ void load_1k(r_i32x4 resource, int offset, int more, unsigned to) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" ::"s"(__builtin_amdgcn_readfirstlane(to)), "v"(offset), "s"(resource),
                 "s"(more)
                 : "memory", "m0");
}
#pragma clang diagnostic pop
struct TreeSizes {
    int n_pages, page_size, nq, hd, window, n_tokens;
    unsigned magic_group, magic_page;
    float scale;
};

// What a difference of scores is an exponent of 2 by.  (A negative scale turns the queries' signs.)
__host__ __device__ __forceinline__ float base_2_scale(float scale) { return fabsf(scale) * 1.4426950408889634f; }

template <typename T, int HD, int RB, int KS, int KT, int NS, int FS>
constexpr int tree_lds() {
    constexpr int stages = NS * KS * 2 * KT * HD * static_cast<int>(sizeof(T)), join = KS * RB * 64 * (HD / 2 + 2) * 4;
    constexpr int given = FS > 1 ? RB * FS * (KT / 32) * 16 * 64 * 4 : 0;      // the halves of the scores, behind the tiles
    return (KS == 1 || stages > join ? stages : join) + given;
}

// The rounds of `keys` (a power of two) keys that a context takes, one at least; contexts are below 2^27.
__device__ __forceinline__ int rounds_of_keys(int kv, int keys) { return min(max(kv, 1) - 1, (1 << 27) - 1) / keys + 1; }
// ceil(x / d), x and d below 2^22; inv a reciprocal of d.
__device__ __forceinline__ int upper_quotient(int x, int d, float inv) {
    const int y = x + d - 1, q = static_cast<int>(static_cast<float>(y) * inv);
    return q + ((q + 1) * d <= y ? 1 : 0) - (q * d > y ? 1 : 0);
}

// Which request's work a workgroup has: a block of rows over a part of its keys, of `per` rounds (KT * KS keys each).  The host says how many works would be best if
// every context were as long as the longest can be (`want`); here `per` follows from what the contexts are, so that there are about as many, and no request has more
// than `most` parts.  (64 requests of 1 to 32 nodes behind 128 to 4,000 tokens: 43.1 us with parts of a length chosen
// by the longest alone, 36.6 so; both with the join as it was.)
//
// The requests' works lie one after the other, request b has blocks_of(q_len[b]) * ceil(rounds_of(kv_len[b]) / per) of them.  Workgroups go to the eight
// dies in turn, so those of a die take works that follow each other: blocks of rows that read the same keys are on one die.  As many workgroups as works, not
// as the most of any request for each: workgroups without work, in a pattern, leave the same compute units idle (154 of 256 busy there).
// 64 requests at a time, by a sum over the lanes.  False: nobody's.
struct TreeWork {
    int request, index, n, kv, per, parts;
    bool first;
};
template <class Blocks, class Rounds>
__device__ __forceinline__ bool find_work(const int32_t* __restrict__ q_len, const int32_t* __restrict__ kv_len, int n_seqs, Blocks blocks_of, Rounds rounds_of,
                                          int want, int most, unsigned magic_most, TreeWork& found) {
    const int lane = threadIdx.x % kWave;
    auto upto_of = [&](int v) {
        v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, true);                // row_shr:1, 2, 4, 8: the sum within a row
        v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, true);
        v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, true);
        v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, true);
        v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);               // row_bcast:15 and 31: the rows before it
        v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);
        return v;
    };
    auto sum_of = [&](int v) { return __builtin_amdgcn_readlane(upto_of(v), kWave - 1); };
    const int n0 = lane < n_seqs ? q_len[lane] : 0, kv0 = lane < n_seqs ? kv_len[lane] : 0;
    const int blocks0 = blocks_of(n0), rounds0 = rounds_of(kv0);
    int per = 1 << 21;                           // (one part of each: as many rounds as it takes)
    if (most > 1 && n_seqs == 1) {               // (the host knew it all)
        per = divided(__builtin_amdgcn_readfirstlane(rounds0) + most - 1, most, magic_most);
    } else if (most > 1) {
        int blocks = sum_of(blocks0);
        float all = wave_sum(static_cast<float>(blocks0) * static_cast<float>(rounds0)), longest = blocks0 > 0 ? static_cast<float>(rounds0) : 0.f;
        for (int s0 = kWave; s0 < n_seqs; s0 += kWave) {
            const int i = s0 + lane, b = i < n_seqs ? blocks_of(q_len[i]) : 0, r = i < n_seqs ? rounds_of(kv_len[i]) : 0;
            all += wave_sum(static_cast<float>(b) * static_cast<float>(r));
            blocks += sum_of(b);
            longest = fmaxf(longest, b > 0 ? static_cast<float>(r) : 0.f);
        }
        const int least = divided(__builtin_amdgcn_readfirstlane(static_cast<int>(wave_max(longest))) + most - 1, most, magic_most);
        auto rounds_for = [&](int works) {                   // ceil(all / works)
            const float w = static_cast<float>(works);
            const int q = static_cast<int>(fminf(all * __builtin_amdgcn_rcpf(w), 2097152.f));
            return q + (static_cast<float>(q) * w < all ? 1 : 0);
        };
        per = max(max(least, rounds_for(want)), 1);
        // (parts that do not come out even are some half a part more for each block of rows)
        const float inv = __builtin_amdgcn_rcpf(static_cast<float>(per));
        int works = sum_of(blocks0 * upper_quotient(rounds0, per, inv));
        for (int s0 = kWave; s0 < n_seqs; s0 += kWave) {
            const int i = s0 + lane;
            works += sum_of(i < n_seqs ? blocks_of(q_len[i]) * upper_quotient(rounds_of(kv_len[i]), per, inv) : 0);
        }
        if (works > want) per = max(per, rounds_for(max(want - blocks / 2, 1)));
        per = __builtin_amdgcn_readfirstlane(per);
    }
    const float inv = __builtin_amdgcn_rcpf(static_cast<float>(per));
    int n = n0, kv = kv0, parts = most > 1 ? upper_quotient(rounds0, per, inv) : 1, work = blocks0 * parts, upto = upto_of(work);
    int total = __builtin_amdgcn_readlane(upto, kWave - 1);
    auto parts_of = [&](int kv_) { return most > 1 ? upper_quotient(rounds_of(kv_), per, inv) : 1; };
    for (int s0 = kWave; s0 < n_seqs; s0 += kWave) {
        const int i = s0 + lane;
        total += sum_of(i < n_seqs ? blocks_of(q_len[i]) * parts_of(kv_len[i]) : 0);
    }
    const int each = (total + 7) / 8;
    int index = static_cast<int>(blockIdx.x % 8) * each + static_cast<int>(blockIdx.x / 8);
    if (static_cast<int>(blockIdx.x / 8) >= each || index >= total) return false;
    found.per = per;
    found.first = index == 0;
    for (int s0 = 0;;) {
        const unsigned long long behind = __ballot(upto > index);
        if (behind != 0) {
            const int at = __builtin_ctzll(behind);
            found.request = s0 + at;
            found.index = index - (__builtin_amdgcn_readlane(upto, at) - __builtin_amdgcn_readlane(work, at));
            found.n = __builtin_amdgcn_readlane(n, at);
            found.kv = __builtin_amdgcn_readlane(kv, at);
            found.parts = __builtin_amdgcn_readlane(parts, at);
            return true;
        }
        index -= __builtin_amdgcn_readlane(upto, kWave - 1);
        s0 += kWave;
        const int i = s0 + lane;
        n = i < n_seqs ? q_len[i] : 0;
        kv = i < n_seqs ? kv_len[i] : 0;
        parts = parts_of(kv);
        work = blocks_of(n) * parts;
        upto = upto_of(work);
    }
}

// (the first 14 words of the arguments arrive with the wavefronts: all that the first trip to memory needs)
template <typename T, int HD, int RB, int KS, int KT, int NS, int FS>
__global__ __launch_bounds__(64 * RB * KS * FS, HD * static_cast<int>(sizeof(T)) <= 256 || RB * FS > 4 ? 2 : 1) void tree_attention_kernel(
    const int32_t* __restrict__ q_len, const int32_t* __restrict__ kv_len, const int32_t* __restrict__ block_table, int n_seqs, int nkv, int most_parts,
    int want, int group, int max_q_len, int table_width, unsigned magic_most, const int32_t* __restrict__ q_start,
    const T* __restrict__ qkv, const long long* __restrict__ visible, const int32_t* __restrict__ positions, const T* __restrict__ k_cache,
    const T* __restrict__ v_cache, T* __restrict__ out, float* __restrict__ part_o, float* __restrict__ part_ml, int* __restrict__ per_out, TreeSizes z) {
    constexpr int SZ = sizeof(T);
    constexpr int ROWB = HD * SZ, PIECES = ROWB / 16, KC = ROWB / 32, DB = HD / 32, KB = KT / 32;
    constexpr int HALF = KT * ROWB, TILE = 2 * HALF;             // bytes of a tile's keys, and of it all
    constexpr int KC_OWN = KC / FS, DB_OWN = DB / FS;            // pieces of 32 bytes of a key, blocks of 32 features of a value: a wavefront's
    constexpr int LOADS = HALF / 1024 / (RB * FS);               // of a wavefront and tile, keys and values each
    constexpr int PER_GROUP = ROWB / 64;                         // loads of a group of 16 keys
    constexpr int OWN = LOADS > PER_GROUP ? LOADS / PER_GROUP : 1, EACH = LOADS > PER_GROUP ? PER_GROUP : LOADS;
    constexpr int STEPS = SZ == 2 ? 2 : 4;                       // second products of a block of 32 keys: 32 bytes of a feature each
    static_assert(FS == 1 || KS == 1, "wavefronts that share features have the same keys");
    static_assert(LOADS >= 1 && HALF % (1024 * RB * FS) == 0 && OWN * EACH == LOADS, "every wavefront loads as much");
    static_assert(kWave * kGroup % (KT * KS) == 0, "the 64 groups that a wavefront has the pages of are whole rounds");
    extern __shared__ __attribute__((aligned(1024))) char smem[];
    const int tid = threadIdx.x, lane = tid % kWave, lr = lane % 32, lh = lane / 32;
    const int wave = __builtin_amdgcn_readfirstlane(tid / kWave), rb = wave % RB, fs = wave / RB % FS, ksi = wave / (RB * FS);

    // which part of which request and kv head, and which block of its rows
    auto blocks_of = [&](int n_) { return (min(max(n_, 0), max_q_len) * group + 32 * RB - 1) / (32 * RB); };
    TreeWork work;
    if (!find_work(q_len, kv_len, n_seqs, [&](int n_) { return blocks_of(n_) * nkv; }, [](int kv_) { return rounds_of_keys(kv_, KT * KS); }, want, most_parts,
                   magic_most, work))
        return;
    const int b = work.request, n = work.n, kv_all = work.kv, chunk = work.per * (KT * KS);
    const int blocks = blocks_of(n), n_parts = work.parts;
    const int unit = work.index / blocks, block = work.index - unit * blocks, kvh = unit / n_parts, part = unit - kvh * n_parts;
    if (most_parts > 1 && work.first && tid == 0) *per_out = work.per;
    const int qs = q_start[b];
    const int from = part * chunk;
    // The pages of 64 groups of keys, a lane each, asked for before it is known how many keys there are; the next 64 while these are walked.
    const int32_t* const table = block_table + static_cast<size_t>(b) * table_width;
    struct Places {
        int page, off;                                           // (page -1: none)
    };
    auto places_from = [&](int first_key) {
        const int key = min(first_key + lane * kGroup, table_width * z.page_size - 1), at = divided(key, z.page_size, z.magic_page);
        const int page = table[at];
        return Places{page >= z.n_pages ? -1 : page, key - at * z.page_size};
    };
    Places here = places_from(from);
    const int rows = n * group, row0 = block * 32 * RB;
    const int before = kv_all - n, kv = min(kv_all, table_width * z.page_size);
    const int to = min(kv - from, chunk) + from;
    const int groups = to > from ? (to - from + kGroup - 1) / kGroup : 0;

    const int key_bytes = z.hd * SZ;
    const size_t head_bytes = static_cast<size_t>(z.page_size) * key_bytes, page_bytes = head_bytes * nkv;
    const char* const k_head = reinterpret_cast<const char*>(k_cache) + kvh * head_bytes;
    const char* const v_head = reinterpret_cast<const char*>(v_cache) + kvh * head_bytes;
    // A wavefront's loads of a tile: EACH of a group's PER_GROUP, of OWN groups.  Load u has the group's keys from u * (1024 / ROWB) on, and the values' features from
    // u * (64 / SZ) on; what differs between a wavefront's loads is a scalar offset and, in the exchange of a key's pieces, bits of its number above the lane's.
    constexpr int KEYS = 1024 / ROWB;
    const int first_load = (fs * RB + rb) * LOADS, group_first = first_load / PER_GROUP, load_first = first_load % PER_GROUP;
    // (16 lanes read 256 bytes, all banks, at a time: their rows' pieces lie in 16 different places, two rows of 128 bytes side by side)
    auto swap_at = [](int lane_row) { return PIECES >= 16 ? lane_row & 15 : lane_row >> 1 & 7; };
    auto swap_of = [&](int key) { return swap_at(SZ == 2 ? (key & 3) | (key >> 1 & 4) | (key << 1 & 8) : key); };      // bfloat16: bits 2 and 3 exchanged
    const int k_row_of_lane = lane / PIECES, k_place = lane % PIECES ^ swap_of(k_row_of_lane);
    const int v_at = value_lane(lane, SZ, z.page_size, z.hd, kNowhere);
    const int n_tiles = (groups * kGroup + KT - 1) / KT, rounds = (n_tiles + KS - 1) / KS;
    const unsigned lds0 = static_cast<unsigned>(reinterpret_cast<uintptr_t>((lds_void*)smem));
    // (`places`: those of the 64 groups that the round's keys are among)
    auto load_tile = [&](int round, const Places& places) {
        const unsigned base = lds0 + (round % NS * KS + ksi) * TILE + first_load * 1024;
        const int g0 = (round * KS + ksi) * (KT / kGroup) + group_first;
#pragma unroll
        for (int o = 0; o < OWN; ++o) {
            const int page = g0 + o < groups ? __builtin_amdgcn_readlane(places.page, (g0 + o) % kWave) : -1;
            const int off = __builtin_amdgcn_readlane(places.off, (g0 + o) % kWave);
            const bool missing = page < 0;
            const size_t at = static_cast<size_t>(max(page, 0)) * page_bytes;
            const char* const keys = k_head + at + static_cast<size_t>(off) * key_bytes;
            const char* const values = v_head + at + static_cast<size_t>(off) * SZ;
#pragma unroll
            for (int j = 0; j < EACH; ++j) {
                const GroupLoad from_here = key_load(load_first + j, KEYS, key_bytes, missing);
                load_1k(buffer_of(keys, from_here.bytes), key_lane(k_row_of_lane, key_bytes, k_place ^ swap_of((load_first + j) * KEYS), kNowhere), from_here.more,
                        base + (o * PER_GROUP + j) * 1024);
            }
#pragma unroll
            for (int j = 0; j < EACH; ++j) {
                const GroupLoad from_here = value_load(load_first + j, SZ, z.page_size, z.hd, static_cast<unsigned>(head_bytes) - off * SZ, missing);
                load_1k(buffer_of(values, from_here.bytes), v_at, from_here.more, base + HALF + (o * PER_GROUP + j) * 1024);
            }
        }
    };
    constexpr int AHEAD = kWave * kGroup / (KT * KS);            // rounds that the places of 64 groups serve
    static_assert(AHEAD >= NS, "the tiles ahead lie within the next places");

    // this lane's row
    const int r = row0 + rb * 32 + lr;
    const int node_at = divided(r, group, z.magic_group);
    const bool valid = r < rows && qs >= 0 && node_at < z.n_tokens - qs;
    const int node = valid ? node_at : 0, head = kvh * group + (valid ? r - node * group : 0);
    const int token = qs + node;
    // the first round: with a window the one that has the first key that any row of the workgroup sees
    int lo = valid ? 0 : 0x7fffffff, first_round = 0, all_see = 0;       // all_see: from which key on all rows see everything before the tree
    if (z.window > 0) {
        __shared__ int s_least, s_most;
        if (tid == 0) {
            s_least = 0x7fffffff;
            s_most = 0;
        }
        __syncthreads();
        if (valid) {
            lo = min(max(0, positions[token] - z.window + 1), max(before, 0));
            atomicMin(&s_least, lo);
            atomicMax(&s_most, lo);
        }
        __syncthreads();
        first_round = __builtin_amdgcn_readfirstlane(max(0, min(s_least, max(before, 0)) - from) / (KT * KS));
        all_see = __builtin_amdgcn_readfirstlane(s_most);
    }
    int window_of = 0;                                           // `here` has the places of groups [64 window_of, 64 window_of + 64)
    if (first_round >= AHEAD) {
        window_of = first_round / AHEAD;
        here = places_from(from + window_of * kWave * kGroup);
    }
    Places next = places_from(from + (window_of + 1) * kWave * kGroup);
    auto load_round = [&](int round) { load_tile(round, round / AHEAD == window_of ? here : next); };
#pragma unroll
    for (int i = 0; i < NS - 1; ++i)
        if (first_round + i < rounds) load_round(first_round + i);

    const unsigned long long bits = valid ? static_cast<unsigned long long>(visible[token]) : 0ull;
    const char* const q_row = reinterpret_cast<const char*>(qkv + static_cast<size_t>(token) * (z.nq + 2 * nkv) * z.hd + head * z.hd);
    auto query_at = [&](int i) {
        const int at = i * 32 + lh * 16;
        u32x4 one = valid && at < key_bytes ? *reinterpret_cast<const u32x4*>(q_row + at) : u32x4{0u, 0u, 0u, 0u};
        if (z.scale < 0.f) one ^= SZ == 2 ? 0x80008000u : 0x80000000u;             // (the greatest score is the greatest product then as well)
        return one;
    };
    u32x4 q[KC_OWN];
#pragma unroll
    for (int i = 0; i < KC_OWN; ++i) q[i] = query_at(fs * KC_OWN + i);

    f32x16 acc[DB_OWN];
#pragma unroll
    for (int d = 0; d < DB_OWN; ++d)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[d][e] = 0.f;
    float m_run = -INFINITY, l_run = 0.f;
    bool far = false;                                            // some row's maximum lies beyond kFar
    const float scale2 = base_2_scale(z.scale);
    const int my_key = SZ == 2 ? (lr & 3) | (lr >> 1 & 4) | (lr << 1 & 8) | (lr & 16) : lr;
    const int k_row = my_key * ROWB, k_piece = (lh ^ swap_at(lr)) * 16;
    const int v_row = lr * kGroup * SZ + (SZ == 2 ? (lh ^ (lr >> 3 & 1)) * 16 : ((lh ^ (lr >> 2 & 3)) * 16));

    auto piece_at = [&](const char* at) { return *reinterpret_cast<const u32x4*>(at); };
    auto values_at = [&](const char* tile, int kb, int step, int d) {
        const int g = kb * 2 + (SZ == 2 ? step : step / 2);
        const int row = SZ == 2 ? v_row : v_row ^ ((step % 2) * 32);
        return piece_at(tile + HALF + (g * HD + (fs * DB_OWN + d) * 32) * kGroup * SZ + row);
    };
    // A tile with values that are no finite numbers, some of them of nodes that not every row sees: a row's weight for such a key is zero, and zero times
    // an infinity is none.  So one key after the other, on the vector pipe, left out where it is not seen.  (Rare, and slow: registers that it held would be the other tiles'.)
    auto strange_tile = [&](const char* tile, int key0, const Places& places) {
#pragma unroll 1
        for (int key = 0; key < KT; ++key) {
            const int j = key0 + key;
            if (j >= to) break;
            if (__builtin_amdgcn_readlane(places.page, (j - from) / kGroup % kWave) < 0) continue;
            const bool sees = valid && (j < before ? j >= lo : j - before < 64 && (bits >> (j - before) & 1ull) != 0);
            if (!__any(sees)) continue;
            float dot = 0.f;
            auto add = [&](int i, u32x4 query) {
                const u32x4 k = *reinterpret_cast<const u32x4*>(tile + key * ROWB + (((2 * i + lh) ^ swap_of(key)) * 16));
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if constexpr (SZ == 2) {
                        dot = fmaf(__uint_as_float(k[e] << 16), __uint_as_float(query[e] << 16), dot);
                        dot = fmaf(__uint_as_float(k[e] & 0xffff0000u), __uint_as_float(query[e] & 0xffff0000u), dot);
                    } else {
                        dot = fmaf(__uint_as_float(k[e]), __uint_as_float(query[e]), dot);
                    }
                }
            };
            if constexpr (FS > 1) {                                             // (the others' features as well, from memory)
#pragma unroll 1
                for (int i = 0; i < KC; ++i) add(i, query_at(i));
            } else {
#pragma unroll
                for (int i = 0; i < KC; ++i) add(i, q[i]);
            }
            dot = fold_32_apart(dot, AddOf());
            const float m_new = sees ? fmaxf(m_run, dot) : m_run, m_use = m_new == -INFINITY ? 0.f : m_new;
            const float alpha = m_run == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m_run - m_use) * scale2), w = __builtin_amdgcn_exp2f((dot - m_use) * scale2);
            m_run = m_new;
            far = far || __any(fabsf(m_run) * scale2 > kFar && m_run != -INFINITY);
            l_run = l_run * alpha + (sees && lh == 0 ? w : 0.f);             // (the halves' sums are added up in the end)
            const char* const values = tile + HALF + key / kGroup * HD * kGroup * SZ;
#pragma unroll
            for (int d = 0; d < DB_OWN; ++d) {
                asm volatile("" ::: "memory");                                // (not all of them at once)
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const int feature = (fs * DB_OWN + d) * 32 + e / 4 * 8 + lh * 4 + e % 4, in = key % kGroup;
                    float v;
                    if constexpr (SZ == 2) v = __uint_as_float(static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(values + feature * 32 + ((in / 8) ^ (feature >> 3 & 1)) * 16 + in % 8 * 2)) << 16);
                    else v = *reinterpret_cast<const float*>(values + feature * 64 + ((in / 4) ^ (feature >> 2 & 3)) * 16 + in % 4 * 4);
                    const float scaled = acc[d][e] * alpha;
                    acc[d][e] = sees ? fmaf(w, v, scaled) : scaled;
                }
            }
        }
    };
    // A tile.  MASKED: its scores are compared with what the row sees.
    auto tile_of = [&](auto masked, const char* tile, int key0, const Places& places) {
        constexpr bool MASKED = decltype(masked)::value;
        constexpr int R = SZ == 2 ? 8 : 4;                                      // neighbouring keys of a lane
        f32x16 s[KB];
        unsigned sees[KB];
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
#pragma unroll
            for (int e = 0; e < 16; ++e) s[kb][e] = 0.f;
#pragma unroll
            for (int i = 0; i < KC_OWN; ++i)
                s[kb] = product_of<T>(piece_at(tile + kb * 32 * ROWB + k_row + fs * KC_OWN * 32 + (k_piece ^ (i * 32))), q[i], s[kb]);
        }
        if constexpr (MASKED) {
            // Whether any value is no finite number: their products with zeros are zeros unless it is.  (bfloat16 by the matrix cores, beside the scores' products,
            // which wait for other results; float32's are eight times as long as the few vector instructions.)
            float sum = 0.f;
            if constexpr (SZ == 2) {
                f32x16 probe;
#pragma unroll
                for (int e = 0; e < 16; ++e) probe[e] = 0.f;
#pragma unroll
                for (int kb = 0; kb < KB; ++kb)
#pragma unroll
                    for (int step = 0; step < STEPS; ++step)
#pragma unroll
                        for (int d = 0; d < DB_OWN; ++d) probe = product_of<T>(values_at(tile, kb, step, d), u32x4{0u, 0u, 0u, 0u}, probe);
#pragma unroll
                for (int e = 0; e < 16; ++e) sum += probe[e];
            } else {
#pragma unroll
                for (int kb = 0; kb < KB; ++kb)
#pragma unroll
                    for (int step = 0; step < STEPS; ++step)
#pragma unroll
                        for (int d = 0; d < DB_OWN; ++d) {
                            const u32x4 v = values_at(tile, kb, step, d);
#pragma unroll
                            for (int e = 0; e < 4; ++e) sum = fmaf(__uint_as_float(v[e]), 0.f, sum);
                        }
            }
            bool strange = __any(sum != 0.f) != 0;
            if constexpr (FS > 1) strange = __syncthreads_or(strange) != 0;     // (the wavefronts of a row go the same way)
            if (__builtin_expect(strange, 0)) return strange_tile(tile, key0, places);
        }
        if constexpr (FS > 1) {                          // the scores of the other features, from the wavefronts that have them
            tree_f32x4* const given = reinterpret_cast<tree_f32x4*>(smem + NS * KS * TILE) + lane;
#pragma unroll
            for (int kb = 0; kb < KB; ++kb)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    given[((wave * KB + kb) * 4 + e) * kWave] = tree_f32x4{s[kb][4 * e], s[kb][4 * e + 1], s[kb][4 * e + 2], s[kb][4 * e + 3]};
            __syncthreads();
#pragma unroll
            for (int f = 1; f < FS; ++f) {
                const int other = (fs + f) % FS * RB + rb;
#pragma unroll
                for (int kb = 0; kb < KB; ++kb)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const tree_f32x4 one = given[((other * KB + kb) * 4 + e) * kWave];
#pragma unroll
                        for (int i = 0; i < 4; ++i) s[kb][4 * e + i] += one[i];
                    }
            }
        }
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
            if constexpr (MASKED) {
                const int k0 = key0 + kb * 32, cut = before - k0;               // keys of the block before the tree
                unsigned long long w = cut >= 0 ? (cut < 32 ? bits << cut : 0ull) : (cut > -64 ? bits >> -cut : 0ull);
                unsigned early = cut >= 32 ? 0xffffffffu : cut > 0 ? (1u << cut) - 1u : 0u;
                const int skip = lo - k0;
                if (skip > 0) early = skip >= 32 ? 0u : early & (0xffffffffu << skip);
                unsigned all = static_cast<unsigned>(w) | early;
                const int end = to - k0;
                if (end < 32) all = end > 0 ? all & ((1u << end) - 1u) : 0u;
#pragma unroll
                for (int g = 0; g < 2; ++g)
                    if (__builtin_amdgcn_readlane(places.page, ((k0 - from) / kGroup + g) % kWave) < 0) all &= g == 0 ? 0xffff0000u : 0x0000ffffu;
                if (!valid) all = 0u;
                sees[kb] = all >> (lh * R);
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const unsigned it = bit_filled(sees[kb], e / R * 2 * R + e % R);
                    s[kb][e] = __uint_as_float((__float_as_uint(s[kb][e]) & it) | (0xff800000u & ~it));
                }
            }
        }
        float mx = s[0][0];          // (two at a time are one instruction)
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int e = 0; e < 16; e += 2) mx = fmaxf(fmaxf(mx, s[kb][e]), s[kb][e + 1]);
        mx = fold_32_apart(mx, MaxOf());
        // The maximum that exponentials are taken against follows a row's once that has grown by more than 2^kSlack: they may reach 2^kSlack meanwhile, which
        // float32 sums do not mind, nor bfloat16, as near at any magnitude; and the sums are rescaled a few times a context and not every few tiles.
        if (__any((mx - m_run) * scale2 > kSlack || (m_run == -INFINITY && mx > m_run))) {
            const float m_new = fmaxf(m_run, mx);
            const float alpha = m_run == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m_run - m_new) * scale2);
            l_run *= alpha;
            m_run = m_new;
            far = __any(fabsf(m_run) * scale2 > kFar && m_run != -INFINITY) != 0;
#pragma unroll
            for (int d = 0; d < DB_OWN; ++d)
#pragma unroll
                for (int e = 0; e < 16; ++e) acc[d][e] *= alpha;
        }
        const float m_use = m_run == -INFINITY ? 0.f : m_run;
        [[maybe_unused]] float m_scaled = m_use * scale2;
        if constexpr (SZ == 2) {
            if (__builtin_expect(far, 0)) {
                m_scaled = 0.f;
#pragma unroll
                for (int kb = 0; kb < KB; ++kb)
#pragma unroll
                    for (int e = 0; e < 16; ++e) s[kb][e] -= m_use;
            }
        }
        u32x4 weights[KB][STEPS];
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
            float sum = 0.f;
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                // (bfloat16: the argument by one operation; what the rounding of the maximum's product leaves in it, 2^-13 at kFar, is nothing beside the
                // probabilities' rounding.  Beyond, where it would be, and at 2^31 exceed every exponent, the maximum is taken off first, as float32 has it.)
                float p = SZ == 2 ? __builtin_amdgcn_exp2f(fmaf(s[kb][e], scale2, -m_scaled)) : __builtin_amdgcn_exp2f((s[kb][e] - m_use) * scale2);
                if constexpr (MASKED) p = __uint_as_float(__float_as_uint(p) & bit_filled(sees[kb], e / R * 2 * R + e % R));
                s[kb][e] = p;
                if constexpr (SZ == 4) {
                    sum += p;
                    weights[kb][e / 4][e % 4] = __float_as_uint(p);
                } else {
                    // (beyond heads of 64 the sum is of the rounded weights, as the values' sums are, two to an instruction: two long users 84.5 -> 81.1 us; the shapes
                    // for heads of 64 are 1 % slower so, 30.6 -> 30.9)
                    if constexpr (HD <= 64) sum += p;
                    if (e % 2 == 1) {
                        const uint32_t pair = bf16_pair(s[kb][e - 1], p);
                        weights[kb][e / 8][e / 2 % 4] = pair;
                        if constexpr (HD > 64)
                            sum = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(tree_bf16x2, pair), __builtin_bit_cast(tree_bf16x2, 0x3f803f80u), sum, false);
                    }
                }
            }
            l_run += sum;
        }
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int step = 0; step < STEPS; ++step) {
                const u32x4 p = weights[kb][step];
#pragma unroll
                for (int d = 0; d < DB_OWN; ++d) acc[d] = product_of<T>(values_at(tile, kb, step, d), p, acc[d]);
            }
    };

    // Rounds whose keys every row sees, all before the tree, behind all windows and in pages, go without masks; they lie together.  (One loop that asked every
    // time would carry the accumulators from one kind's registers to the other's.)
    auto begin_round = [&](int round) {
        // this wavefront's loads of the tile are there when no more than those of the later ones are on their way; then everybody's
        if (round + NS - 1 <= rounds) arrived<(NS - 2) * 2 * LOADS>();
        else arrived<0>();
        __syncthreads();
        if (round + NS - 1 < rounds) load_round(round + NS - 1);
    };
    auto tile_at = [&](int round) { return smem + (round % NS * KS + ksi) * TILE; };
    auto gone_here = [&]() {
        const int key = from + (window_of * kWave + lane) * kGroup;
        return __any(here.page < 0 && key < before && key + kGroup > all_see) != 0;
    };
    bool gone = gone_here();                                     // some key of `here` that all rows would see is in no page
    auto end_round = [&](int round) {
        if ((round + 1) % AHEAD != 0) return;
        here = next;
        ++window_of;
        if ((window_of + 1) * AHEAD < rounds) next = places_from(from + (window_of + 1) * kWave * kGroup);
        gone = gone_here();
    };
    // (a wavefront behind the last row loads its share of the tiles and leaves the pipes to the others; where wavefronts share features all of them meet in a tile)
    const bool has_rows = FS > 1 || row0 + rb * 32 < rows;
    constexpr int ROUND = KT * KS;
    const int open_from = (all_see - from + ROUND - 1) / ROUND, open_end = (min(before, to) - from) / ROUND;
    for (int round = first_round;;) {
        for (; round < rounds && (gone || round < open_from || round >= open_end); ++round) {
            begin_round(round);
            const int tile = round * KS + ksi;
            if (tile < n_tiles && has_rows) tile_of(std::true_type{}, tile_at(round), from + tile * KT, here);
            end_round(round);
        }
        if (round >= rounds) break;
        for (; round < open_end && !gone; ++round) {
            begin_round(round);
            if (has_rows) tile_of(std::false_type{}, tile_at(round), from + (round * KS + ksi) * KT, here);
            end_round(round);
        }
    }
    float l = fold_32_apart(l_run, AddOf());

    // Four neighbouring features of a row are a quad: quad 4 d + e / 4 of a lane the ones from d * 32 + 2 e + 4 lh on.  The groups' results are joined, each group
    // its share of the quads (one wavefront that joins them all is as long alone as two tiles: an instruction of a wavefront that has its SIMD to itself is 5 cycles).
    const size_t row = static_cast<size_t>(token) * z.nq + head, mine = static_cast<size_t>(part) * z.n_tokens * z.nq + row;
    const bool whole = n_parts == 1;
    constexpr int QUADS = DB_OWN * 4, SHARE = QUADS / KS;
    static_assert(QUADS % KS == 0, "as many quads for every group");
    auto leave = [&](const float (&v)[4], int quad, float factor) {
        const int at = (fs * DB_OWN + quad / 4) * 32 + quad % 4 * 8 + lh * 4;
        const float o[4] = {v[0] * factor, v[1] * factor, v[2] * factor, v[3] * factor};
        if (at >= z.hd) return;
        if (whole) write_quad(out + row * z.hd + at, o);
        else write_quad(part_o + mine * z.hd + at, o);
    };
    float m_all = m_run;
    if constexpr (KS > 1) {
        tree_f32x4* const results = reinterpret_cast<tree_f32x4*>(smem) + static_cast<size_t>(rb) * QUADS * kWave + lane;         // [group][rb][quad][lane]
        float2* const sums = reinterpret_cast<float2*>(smem + KS * RB * QUADS * kWave * 16) + rb * kWave + lane;                  // [group][rb][lane]
        __syncthreads();
#pragma unroll
        for (int d = 0; d < DB_OWN; ++d)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                results[(ksi * RB * QUADS + d * 4 + e) * kWave] = tree_f32x4{acc[d][4 * e], acc[d][4 * e + 1], acc[d][4 * e + 2], acc[d][4 * e + 3]};
        sums[ksi * RB * kWave] = float2{m_run, l};
        __syncthreads();
        float factor[KS], l_of[KS];
#pragma unroll
        for (int k = 0; k < KS; ++k) {
            const float2 one = sums[k * RB * kWave];
            factor[k] = one.x;
            l_of[k] = one.y;
        }
        m_all = factor[0];
#pragma unroll
        for (int k = 1; k < KS; ++k) m_all = fmaxf(m_all, factor[k]);
        l = 0.f;
#pragma unroll
        for (int k = 0; k < KS; ++k) {
            factor[k] = factor[k] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((factor[k] - m_all) * scale2);
            l = fmaf(l_of[k], factor[k], l);
        }
        const float inv = !whole ? 1.0f : l == 0.f ? 0.f : 1.0f / l;
        if (!valid) return;
#pragma unroll
        for (int i = 0; i < SHARE; ++i) {
            const int quad = ksi * SHARE + i;
            float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int k = 0; k < KS; ++k) {
                const tree_f32x4 one = results[(k * RB * QUADS + quad) * kWave];
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = fmaf(one[e], factor[k], v[e]);
            }
            leave(v, quad, inv);
        }
    } else {
        if (!valid) return;
        const float inv = !whole ? 1.0f : l == 0.f ? 0.f : 1.0f / l;
#pragma unroll
        for (int d = 0; d < DB_OWN; ++d)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float v[4] = {acc[d][4 * e], acc[d][4 * e + 1], acc[d][4 * e + 2], acc[d][4 * e + 3]};
                leave(v, d * 4 + e, inv);
            }
    }
    if (!whole && lh == 0 && ksi == 0 && fs == 0) {
        part_ml[mine * 2] = m_all;                       // (as it is: its product with the scale would be rounded, and may be no number)
        part_ml[mine * 2 + 1] = l;
    }
}

// The parts of a request's keys joined, with s = scale log2 e: out = sum_p 2^(s (m_p - M)) o_p / sum_p 2^(s (m_p - M)) l_p.  A row has L lanes, four features each, and a wavefront 64 / L rows; the
// lanes take the parts' maxima and sums between them, so that the weights of all are known after one trip, and then the parts' sums, kAhead on their way at a time.  A
// part that saw nothing weighs nothing, whatever it holds.  (64 uneven requests at heads of 64: a row to a
// wavefront 8.8 us, four 5.6.)
template <typename T, int L>
__global__ __launch_bounds__(256) void tree_combine_kernel(const int32_t* __restrict__ q_len, const int32_t* __restrict__ kv_len, const int32_t* __restrict__ q_start,
                                                           const float* __restrict__ part_ml, const float* __restrict__ part_o, const int* __restrict__ per_of, int round_keys,
                                                           int nq, unsigned magic_heads, int nodes, int n_tokens, int hd, float scale2, T* __restrict__ out) {
    constexpr int kAhead = 8, ROWS = kWave / L, OWN = kMostParts / L;
    __shared__ float s_weight[4 * ROWS][kMostParts];
    const int lane = threadIdx.x % kWave, sub = lane % L, in = threadIdx.x / L, b = blockIdx.y;
    const int w = blockIdx.x * 4 * ROWS + in, node = divided(w, nq, magic_heads), head = w - node * nq;
    const int n = q_len[b], kv = kv_len[b], qs = q_start[b], token = qs + node;
    const int per = *per_of, parts = min(upper_quotient(rounds_of_keys(kv, round_keys), per, __builtin_amdgcn_rcpf(static_cast<float>(per))), kMostParts);
    if (parts < 2) return;
    const bool there = node < n && node < nodes && qs >= 0 && node < n_tokens - qs;
    if (!__any(there)) return;
    const size_t row = there ? static_cast<size_t>(token) * nq + head : 0, step = static_cast<size_t>(n_tokens) * nq;
    const int quads = hd / 4, at = min(sub, quads - 1) * 4;
    const float* const from = part_o + row * hd + at;
    float v[kAhead][4];
    auto ask = [&](int p0) {
#pragma unroll
        for (int i = 0; i < kAhead; ++i)
            if (p0 + i < parts) read_quad(from + (p0 + i) * step * hd, v[i]);
    };
    ask(0);
    float m[OWN], l[OWN], most = -INFINITY, total = 0.f;
#pragma unroll
    for (int j = 0; j < OWN; ++j) {
        const int p = sub + j * L;
        const size_t mine = (min(p, parts - 1) * step + row) * 2;
        if (j == 0 || j * L < parts) {
            m[j] = part_ml[mine];
            l[j] = p < parts ? part_ml[mine + 1] : 0.f;
            most = fmaxf(most, l[j] != 0.f ? m[j] : -INFINITY);
        }
    }
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor(most, o, kWave));
#pragma unroll
    for (int j = 0; j < OWN; ++j) {
        if (j > 0 && j * L >= parts) continue;
        const float weight = l[j] != 0.f ? __builtin_amdgcn_exp2f((m[j] - most) * scale2) : 0.f;
        total = fmaf(weight, l[j], total);
        s_weight[in][sub + j * L] = l[j] != 0.f ? weight : -1.f;      // (of a part that saw nothing, whose sums may be anything)
    }
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) total += __shfl_xor(total, o, kWave);
    __builtin_amdgcn_wave_barrier();                                   // (a row's weights are read by the wavefront that wrote them)
    float sum[4] = {};
    for (int p0 = 0;;) {
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            if (p0 + i >= parts) break;
            const float share = s_weight[in][p0 + i];
#pragma unroll
            for (int e = 0; e < 4; ++e) sum[e] = share == -1.f ? sum[e] : fmaf(v[i][e], share, sum[e]);
        }
        p0 += kAhead;
        if (p0 >= parts) break;
        ask(p0);
    }
    if (!there || sub >= quads) return;
    const float inv = total == 0.f ? 0.f : 1.0f / total;
    const float o[4] = {sum[0] * inv, sum[1] * inv, sum[2] * inv, sum[3] * inv};
    write_quad(out + row * hd + at, o);
}

template <typename T, int HD, int RB, int KS, int KT, int NS, int FS = 1>
static int launch_tree(const void* qkv, void* out, float* part_o, float* part_ml, const void* k_cache, const void* v_cache, const int32_t* block_table,
                       int table_width, const int32_t* q_start, const int32_t* q_len, const int32_t* kv_len, const long long* visible,
                       const int32_t* positions, const TreeSizes& z, int n_seqs, int nkv, int group, int max_q_len, int parts, int want, hipStream_t s) {
    constexpr int lds = tree_lds<T, HD, RB, KS, KT, NS, FS>();
    static_assert(lds <= 159 * 1024, "a CU's LDS");
    if (parts > kMostParts) return EGPT_BAD_ARGUMENT;
    // No more blocks than this: of rows of all tokens and one begun per request, and the most of a request times the requests.  And no more works: `want`, or half a
    // part a block beyond it where they do not come out even.
    const long long rows = static_cast<long long>(z.n_tokens) * group, most = (max_q_len * group + 32 * RB - 1) / (32 * RB);
    const long long blocks = (rows / (32 * RB) + n_seqs < most * n_seqs ? rows / (32 * RB) + n_seqs : most * n_seqs) * nkv;
    const long long wanted = want > blocks ? want : blocks, works = parts > 1 ? wanted + blocks : blocks;
    const long long grid = (works + 7) / 8 * 8;
    if (grid >= 1 << 26) return EGPT_UNSUPPORTED_SIZE;
    auto kernel = tree_attention_kernel<T, HD, RB, KS, KT, NS, FS>;
    if (lds > 60 * 1024) {                                   // more than a launch may have unasked: asked for once per instance and device
        static std::atomic<unsigned long long> raised{0};
        int device = -1;
        if (hipGetDevice(&device) != hipSuccess) return EGPT_LAUNCH_FAILED;
        const unsigned long long bit = device < 64 ? 1ull << device : 0ull;
        if ((raised.load(std::memory_order_relaxed) & bit) == 0ull) {
            if (hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, lds) != hipSuccess) return EGPT_LAUNCH_FAILED;
            raised.fetch_or(bit, std::memory_order_relaxed);
        }
    }
    int* const per = parts > 1 ? reinterpret_cast<int*>(part_ml + static_cast<size_t>(parts) * z.n_tokens * z.nq * 2) : nullptr;
    kernel<<<static_cast<unsigned>(grid), 64 * RB * KS * FS, lds, s>>>(q_len, kv_len, block_table, n_seqs, nkv, parts, static_cast<int>(wanted), group, max_q_len,
                                                                   table_width, magic_of(parts), q_start, static_cast<const T*>(qkv), visible, positions,
                                                                   static_cast<const T*>(k_cache), static_cast<const T*>(v_cache), static_cast<T*>(out),
                                                                   part_o, part_ml, per, z);
    EGPT_CHECK_LAUNCH();
    if (parts > 1) {
        constexpr int L = HD <= 64 ? 16 : HD <= 128 ? 32 : 64, rows_of_group = 4 * (kWave / L);
        tree_combine_kernel<T, L><<<dim3((max_q_len * z.nq + rows_of_group - 1) / rows_of_group, n_seqs), 256, 0, s>>>(
            q_len, kv_len, q_start, part_ml, part_o, per, KT * KS, z.nq, magic_of(z.nq), max_q_len, z.n_tokens, z.hd, base_2_scale(z.scale),
            static_cast<T*>(out));
        EGPT_CHECK_LAUNCH();
    }
    return EGPT_OK;
}

}  // namespace egpt

using namespace egpt;

extern "C" int egpt_tree_attention_generic(const void* qkv, void* out, const void* k_cache, const void* v_cache, const int32_t* block_table,
                                           int table_width, int n_pages, const int32_t* q_start, const int32_t* q_len, const int32_t* kv_len,
                                           const long long* visible, const int32_t* positions, int n_seqs, int n_tokens, int nq, int nkv, int hd,
                                           int page_size, float scale, int window, int dtype, void* stream) {
    if (!qkv || !out || !k_cache || !v_cache || !block_table || !q_start || !q_len || !kv_len || !visible || (window > 0 && !positions))
        return EGPT_BAD_ARGUMENT;
    if (n_seqs <= 0 || n_tokens < 0 || nq <= 0 || nkv <= 0 || nq % nkv != 0 || hd <= 0 || page_size <= 0 || table_width <= 0 || window < 0 ||
        n_pages < 0 || dtype < 0 || dtype > 1)
        return EGPT_BAD_ARGUMENT;
    // (a key's number and the step to the next ones of a wavefront are added in 32 bits)
    if (hd > kMaxTreeHead || nq > 65535 || static_cast<long long>(table_width) * page_size > 1LL << 30) return EGPT_UNSUPPORTED_SIZE;
    if (n_tokens == 0) return EGPT_OK;
    auto launch = [&](auto zero) {
        using T = decltype(zero);
        tree_attention_generic_kernel<T><<<dim3(n_tokens, nq), kWave * kTreeWaves, 0, static_cast<hipStream_t>(stream)>>>(
            static_cast<const T*>(qkv), q_start, q_len, kv_len, visible, positions, n_seqs, window, static_cast<const T*>(k_cache),
            static_cast<const T*>(v_cache), block_table, table_width, n_pages, nq, nkv, hd, page_size, scale, static_cast<T*>(out));
    };
    if (dtype == 0) launch(float{});
    else launch(bf16_t{});
    EGPT_CHECK_LAUNCH();
    return EGPT_OK;
}

// shape: 10 * (blocks of 32 rows that a workgroup takes) + wavefronts that share a block's keys.
extern "C" int egpt_tree_attention(const void* qkv, void* out, float* part_o, float* part_ml, const void* k_cache, const void* v_cache,
                                   const int32_t* block_table, int table_width, int n_pages, const int32_t* q_start, const int32_t* q_len,
                                   const int32_t* kv_len, const long long* visible, const int32_t* positions, int n_seqs, int n_tokens, int nq, int nkv,
                                   int hd, int page_size, float scale, int window, int max_q_len, int shape, int parts, int want, int dtype, void* stream) {
    if (!qkv || !out || !k_cache || !v_cache || !block_table || !q_start || !q_len || !kv_len || !visible || (window > 0 && !positions))
        return EGPT_BAD_ARGUMENT;
    if (n_seqs <= 0 || n_tokens < 0 || nq <= 0 || nkv <= 0 || nq % nkv != 0 || hd <= 0 || page_size <= 0 || table_width <= 0 || window < 0 ||
        n_pages < 0 || max_q_len < 0 || dtype < 0 || dtype > 1 || parts <= 0 || want <= 0 || (parts > 1 && (!part_o || !part_ml)))
        return EGPT_BAD_ARGUMENT;
    const int size = dtype == 0 ? 4 : 2;
    if (hd > kMaxTreeHead || hd * size % 16 != 0 || page_size % kGroup != 0 || max_q_len > 64 || nq > 65535 || n_seqs > 65535 ||
        static_cast<long long>(hd) * page_size * size > 0x7fffffffLL || static_cast<long long>(table_width) * page_size > 0x7fffffLL * kGroup)
        return EGPT_UNSUPPORTED_SIZE;
    if ((reinterpret_cast<uintptr_t>(qkv) | reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(k_cache) | reinterpret_cast<uintptr_t>(v_cache)) & 15)
        return EGPT_UNSUPPORTED_SIZE;
    if (n_tokens == 0 || max_q_len == 0) return EGPT_OK;
    const int group = nq / nkv;
    const TreeSizes z{n_pages, page_size, nq, hd, window, n_tokens, magic_of(group), magic_of(page_size), scale};
#define EGPT_TREE(...) \
    return launch_tree<__VA_ARGS__>(qkv, out, part_o, part_ml, k_cache, v_cache, block_table, table_width, q_start, q_len, kv_len, visible, positions, z, n_seqs, nkv, \
                                    group, max_q_len, parts, want, static_cast<hipStream_t>(stream))
    // (type, head size, blocks of rows, groups of wavefronts, keys of a tile, tiles in LDS, wavefronts that share a block's features)
    if (dtype == 1 && hd <= 64) {
        if (shape == 14) EGPT_TREE(bf16_t, 64, 1, 4, 32, 2);
        if (shape == 22) EGPT_TREE(bf16_t, 64, 2, 2, 64, 2);
        if (shape == 41) EGPT_TREE(bf16_t, 64, 4, 1, 64, 2);
    } else if (dtype == 1 && hd <= 128) {
        if (shape == 14) EGPT_TREE(bf16_t, 128, 1, 4, 32, 2);
        if (shape == 22) EGPT_TREE(bf16_t, 128, 2, 2, 32, 2);
        if (shape == 81) EGPT_TREE(bf16_t, 128, 8, 1, 64, 3);
    } else if (dtype == 1) {
        if (shape == 11) EGPT_TREE(bf16_t, 256, 1, 1, 32, 2, 2);
        if (shape == 21) EGPT_TREE(bf16_t, 256, 2, 1, 32, 3, 2);
        if (shape == 41) EGPT_TREE(bf16_t, 256, 4, 1, 32, 3, 2);
    } else if (hd <= 64) {
        if (shape == 14) EGPT_TREE(float, 64, 1, 4, 32, 2);
        if (shape == 22) EGPT_TREE(float, 64, 2, 2, 32, 2);
    } else if (hd <= 128) {
        if (shape == 22) EGPT_TREE(float, 128, 2, 2, 32, 2);
        if (shape == 41) EGPT_TREE(float, 128, 4, 1, 32, 2);
    } else if (shape == 21) {
        EGPT_TREE(float, 256, 2, 1, 32, 2, 2);
    }
#undef EGPT_TREE
    return EGPT_BAD_ARGUMENT;
}
