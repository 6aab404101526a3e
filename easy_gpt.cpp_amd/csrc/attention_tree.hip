// Attention for trees of drafted tokens over the paged cache.
//
// Request b brings n = q_len[b] nodes, whose keys and values are the last n of its kv_len[b] tokens in the cache.  Row (node i,
// query head h) reads key j of kv head h / (nq / nkv) where
//     j < kv - n   and, with a window, j > position_i - window     (the tokens before the tree)
//     j = kv - n + m   and bit m of visible_i is set                 (node m; a request has at most 64)
// and is softmax_j(scale q . k_j) v_j over those, zeros where there are none.  A number that a row does not see does not reach it, be it an
// infinity or a NaN.
#include "api.h"
#include "common.h"

namespace egpt {

constexpr int kMaxTreeHead = 256;

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
    const int n = q_len[b], i = t - q_start[b];
    if (i < 0 || i >= n) return;                             // nobody's row stays as it was
    const int kv = static_cast<int>(min(static_cast<long long>(kv_len[b]), static_cast<long long>(table_width) * page_size));
    const int before = kv_len[b] - n;
    const TreeRow row{window > 0 ? max(0, positions[t] - window + 1) : 0, before, kv, static_cast<unsigned long long>(visible[t])};
    const int kvh = h / (nq / nkv);
    const T* q = qkv + static_cast<size_t>(t) * (nq + 2 * nkv) * hd + h * hd;
    for (int d = threadIdx.x; d < hd; d += kWave * kTreeWaves) q_s[d] = to_float(q[d]);
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
            s = dot * scale;
        }
        const float m_new = fmaxf(m_run, wave_max(s));
        const float m_use = m_new == -INFINITY ? 0.f : m_new;
        const float pj = sees ? expf(s - m_use) : 0.f;
        const float alpha = expf(m_run - m_use);
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
        share[w] = part_ml[w][1] == 0.f ? 0.f : expf(part_ml[w][0] - m_all);
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
    if (hd > kMaxTreeHead || nq > 65535) return EGPT_UNSUPPORTED_SIZE;
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
