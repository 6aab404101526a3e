// What follows the check of drafted tokens: the walk that takes those the model agrees with, and the move of their keys and values.
#include "api.h"
#include "common.h"
#include "lds_loads.h"

namespace egpt {

constexpr int kTreeNodes = 64;          // nodes of a request's tree at most: a lane each

// The walk.  From the root (node 0) to the child whose token is what was sampled after its parent, the lowest of several, until there is none:
//     path[b][0] = 0,  path[b][k + 1] = min { i > c : parent_i = c and token_i = sampled_c },  c = path[b][k]
// One wavefront per request; a step compares all nodes at once and takes the lowest of the ballot, so that a tree of depth d costs d dependent
// steps of some ten instructions and one trip to memory for everything.  path and tokens [n_seqs][64], -1 behind the
// last; token k is what was sampled after node path[k], so the last one is the model's own next token.
__global__ __launch_bounds__(64) void accept_drafts_kernel(const int32_t* __restrict__ tokens, const int32_t* __restrict__ parents,
                                                           const int32_t* __restrict__ sampled, const int32_t* __restrict__ q_start,
                                                           const int32_t* __restrict__ q_len, int n_tokens, int32_t* __restrict__ path,
                                                           int32_t* __restrict__ count, int32_t* __restrict__ accepted) {
    const int b = blockIdx.x, lane = threadIdx.x;
    const int at = q_start[b], n = at >= 0 && at < n_tokens ? min(q_len[b], kTreeNodes) : 0;         // (one that begins nowhere has no nodes)
    const bool here = lane < n && lane < n_tokens - at;
    const int token = here ? tokens[at + lane] : -1, parent = here ? parents[at + lane] : -1, next = here ? sampled[at + lane] : -1;
    int length = 0, mine = -1;
    if (n > 0) {
        int node = 0;
        for (;;) {
            if (lane == length) mine = node;
            ++length;
            const int wanted = __builtin_amdgcn_readlane(next, node);
            const unsigned long long agree = __ballot(here && lane > node && parent == node && token == wanted);
            if (agree == 0) break;                           // (a child lies behind its parent: 63 steps at most)
            node = __builtin_ctzll(agree);
        }
    }
    const int said = __shfl(next, max(mine, 0), kWave);
    path[b * kTreeNodes + lane] = mine;
    accepted[b * kTreeNodes + lane] = mine >= 0 ? said : -1;
    if (lane == 0) count[b] = length;
}

// Entry path[b][k] of the tree goes to place k behind the start[b] tokens before it, key and value of every slab and kv head.  A path
// ascends (a child lies behind its parent), so path[k] >= k: entries are moved in their order, what is read together before any of it is written, and no
// entry is written over that a later one still has to be read from.  One workgroup per (request, slab); a thread owns the same 16 bytes of all keys, or one
// feature of all values, so nobody waits for anybody.
//
// Values lie feature by feature, an entry is hd elements page_size apart: written one by one they are a few bytes here and there of every line of a page, which
// costs memory more than whole lines do.  Where 16 bytes of a feature's row lie in one page (pages of whole 16 bytes a row) a thread writes
// those, the places between as they were.  64 users with 395 of 1,024 entries to move, 28 slabs of 2 heads of 128: 36.7 -> 21.2 us (by 32 bytes
// 22.8); what is left is the pages' lines, 128 bytes for each 16 that change.  No two requests of a call may write into one page.
constexpr int kMoveAhead = 16;          // entries read before the first is written: a trip to memory for most paths
constexpr int kRowAhead = 3;            // 16 bytes of a feature's row likewise
constexpr int kMostRows = kTreeNodes / 4 + 1;

template <typename U>
__device__ __forceinline__ void move_entries(U* __restrict__ base, const long long* s_from, const long long* s_to, int n, size_t at) {
    for (int k0 = 0; k0 < n; k0 += kMoveAhead) {
        U v[kMoveAhead];
#pragma unroll
        for (int k = 0; k < kMoveAhead; ++k)
            if (k0 + k < n) v[k] = base[s_from[k0 + k] + at];
#pragma unroll
        for (int k = 0; k < kMoveAhead; ++k)
            if (k0 + k < n) base[s_to[k0 + k] + at] = v[k];
    }
}

// The same for one feature of the values, 16 bytes of its row at a time: s_row where they lie, s_place the elements that come into each of their places (-1: it
// stays as it is).
template <typename U>
__device__ __forceinline__ void move_rows(U* __restrict__ base, const long long* s_row, const long long (*s_place)[16 / sizeof(U)], int n, size_t at) {
    constexpr int kIn = 16 / sizeof(U);
    for (int k0 = 0; k0 < n; k0 += kRowAhead) {
        U v[kRowAhead][kIn];
        u32x4 was[kRowAhead];
#pragma unroll
        for (int k = 0; k < kRowAhead; ++k) {
            if (k0 + k >= n) continue;
            was[k] = *reinterpret_cast<const u32x4*>(base + s_row[k0 + k] + at);
#pragma unroll
            for (int e = 0; e < kIn; ++e) {
                const long long from = s_place[k0 + k][e];
                if (from >= 0) v[k][e] = base[from + at];
            }
        }
#pragma unroll
        for (int k = 0; k < kRowAhead; ++k) {
            if (k0 + k >= n) continue;
            uint32_t w[4] = {was[k].x, was[k].y, was[k].z, was[k].w};
#pragma unroll
            for (int e = 0; e < kIn; ++e) {
                if (s_place[k0 + k][e] < 0) continue;
                if constexpr (sizeof(U) == 4) w[e] = v[k][e];
                else w[e / 2] = e % 2 ? (w[e / 2] & 0xffffu) | static_cast<uint32_t>(v[k][e]) << 16 : (w[e / 2] & 0xffff0000u) | v[k][e];
            }
            *reinterpret_cast<u32x4*>(base + s_row[k0 + k] + at) = u32x4{w[0], w[1], w[2], w[3]};
        }
    }
}

// KU: the unit that keys are moved by; VU: a value; kRows: values by 16 bytes of a row.  k_units: units of a key (of one head).
template <typename KU, typename VU, bool kRows>
__global__ __launch_bounds__(256) void keep_drafts_kernel(const int32_t* __restrict__ path, const int32_t* __restrict__ count,
                                                          const int32_t* __restrict__ start, const int32_t* __restrict__ block_table,
                                                          int path_width, int table_width, int n_pages, int page_size, int nkv, int k_units, int dv,
                                                          KU* __restrict__ k_cache, VU* __restrict__ v_cache) {
    constexpr int kIn = 16 / sizeof(VU);
    __shared__ long long s_from_k[kTreeNodes], s_to_k[kTreeNodes], s_from_v[kTreeNodes], s_to_v[kTreeNodes];
    __shared__ long long s_row[kMostRows], s_place[kMostRows][kIn];
    __shared__ int s_n, s_rows;
    const int b = blockIdx.x;
    if (threadIdx.x < kWave) {
        const int lane = threadIdx.x;
        const int n = min(min(count[b], path_width), kTreeNodes), before = start[b];
        const int node = lane < n ? path[static_cast<size_t>(b) * path_width + lane] : -1;
        // (what lies where it belongs stays; what has no page, or would be written over, is not touched)
        bool moves = node > lane && node < kTreeNodes && before >= 0 && before < 0x7fffffff - kTreeNodes;
        int from = -1, to = -1;
        const int of = before + node, into = before + lane;
        if (moves && of / page_size < table_width) {
            const int32_t* table = block_table + static_cast<size_t>(b) * table_width;
            from = table[of / page_size];
            to = table[into / page_size];
        }
        moves = moves && from >= 0 && from < n_pages && to >= 0 && to < n_pages;
        const unsigned long long all = __ballot(moves), up_to_me = (2ull << lane) - 1ull;
        const long long kf = static_cast<long long>(from) * nkv * page_size, kt = static_cast<long long>(to) * nkv * page_size;
        if (moves) {
            const int k = __popcll(all & up_to_me) - 1;
            s_from_k[k] = (kf + of % page_size) * k_units;
            s_to_k[k] = (kt + into % page_size) * k_units;
            s_from_v[k] = kf * dv + of % page_size;
            s_to_v[k] = kt * dv + into % page_size;
        }
        if (lane == 0) s_n = __popcll(all);
        if constexpr (kRows) {
            for (int i = lane; i < kMostRows * kIn; i += kWave) (&s_place[0][0])[i] = -1;
            // the first of the entries that go to the same 16 bytes of a row, places before + lane (16 bytes begin at multiples of kIn: pages do)
            const int place = into % kIn, first = lane - place;                             // (the lane of their first place)
            const unsigned long long earlier = all & ((1ull << lane) - 1ull) & (first > 0 ? ~0ull << first : ~0ull);
            const unsigned long long heads = __ballot(moves && earlier == 0ull);
            if (moves) {
                const int row = __popcll(heads & up_to_me) - 1;
                s_row[row] = kt * dv + into % page_size - place;
                s_place[row][place] = kf * dv + of % page_size;
            }
            if (lane == 0) s_rows = __popcll(heads);
        }
    }
    __syncthreads();
    const int n = s_n;
    if (n == 0) return;
    const size_t slab = static_cast<size_t>(blockIdx.y) * n_pages * nkv * page_size;
    const int keys = nkv * k_units, values = nkv * dv;
    for (int i = threadIdx.x; i < keys + values; i += 256) {
        if (i < values) {
            VU* base = v_cache + slab * dv;
            const size_t at = static_cast<size_t>(i) * page_size;
            if constexpr (kRows) move_rows(base, s_row, s_place, s_rows, at);
            else move_entries(base, s_from_v, s_to_v, n, at);
        } else {
            const int h = (i - values) / k_units;
            move_entries(k_cache + slab * k_units, s_from_k, s_to_k, n, static_cast<size_t>(h) * page_size * k_units + (i - values) % k_units);
        }
    }
}

}  // namespace egpt

using namespace egpt;

extern "C" int egpt_accept_drafts(const int32_t* tokens, const int32_t* parents, const int32_t* sampled, const int32_t* q_start,
                                  const int32_t* q_len, int n_seqs, int n_tokens, int32_t* path, int32_t* count, int32_t* accepted, void* stream) {
    if (!q_start || !q_len || !path || !count || !accepted || n_seqs < 0 || n_tokens < 0) return EGPT_BAD_ARGUMENT;
    if (n_tokens > 0 && (!tokens || !parents || !sampled)) return EGPT_BAD_ARGUMENT;
    if (n_seqs == 0) return EGPT_OK;
    accept_drafts_kernel<<<n_seqs, kWave, 0, static_cast<hipStream_t>(stream)>>>(tokens, parents, sampled, q_start, q_len, n_tokens, path, count, accepted);
    EGPT_CHECK_LAUNCH();
    return EGPT_OK;
}

extern "C" int egpt_keep_drafts(void* k_cache, void* v_cache, const int32_t* block_table, int table_width, const int32_t* start, const int32_t* path,
                                int path_width, const int32_t* count, int n_seqs, int n_slabs, int n_pages, int page_size, int nkv, int dk, int dv,
                                int dtype, void* stream) {
    if (!k_cache || !v_cache || !block_table || !start || !path || !count) return EGPT_BAD_ARGUMENT;
    if (n_seqs < 0 || n_slabs < 0 || n_pages < 0 || page_size <= 0 || nkv <= 0 || dk <= 0 || dv <= 0 || table_width <= 0 || path_width <= 0 || dtype < 0 ||
        dtype > 1)
        return EGPT_BAD_ARGUMENT;
    if (n_slabs > 65535) return EGPT_UNSUPPORTED_SIZE;
    if (n_seqs == 0 || n_slabs == 0 || n_pages == 0) return EGPT_OK;
    const dim3 grid(n_seqs, n_slabs);
    hipStream_t s = static_cast<hipStream_t>(stream);
    const int size = dtype == 0 ? 4 : 2, key_bytes = dk * size;
    const bool rows = page_size * size % 16 == 0 && reinterpret_cast<uintptr_t>(v_cache) % 16 == 0;
    auto launch = [&](auto key, auto value, int k_units) {
        using KU = decltype(key);
        using VU = decltype(value);
        auto kernel = rows ? keep_drafts_kernel<KU, VU, true> : keep_drafts_kernel<KU, VU, false>;
        kernel<<<grid, 256, 0, s>>>(path, count, start, block_table, path_width, table_width, n_pages, page_size, nkv, k_units, dv,
                                    static_cast<KU*>(k_cache), static_cast<VU*>(v_cache));
    };
    const bool wide = key_bytes % 16 == 0 && reinterpret_cast<uintptr_t>(k_cache) % 16 == 0;       // keys by 16 bytes
    if (dtype == 0) {
        if (wide) launch(u32x4{}, uint32_t{}, key_bytes / 16);
        else launch(uint32_t{}, uint32_t{}, dk);
    } else {
        if (wide) launch(u32x4{}, uint16_t{}, key_bytes / 16);
        else launch(uint16_t{}, uint16_t{}, dk);
    }
    EGPT_CHECK_LAUNCH();
    return EGPT_OK;
}
