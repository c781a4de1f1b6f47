// qk_kv.h -- the paged cache and the runs of rows as the kernels see them (include/qk_kernels.h: qkk_kv_cache,
// qkk_kv_runs), with the host's checks of both.
#pragma once
#include "qk_device.h"
#include "qk_host.h"

namespace qk {

// One layer of the cache.  Row r of sequence s is row (r & row_mask) of page table[s * seq_pages + (r >> shift)];
// without a table the page is s and shift 31 leaves the row as it is.
struct KvView {
    void *k, *v;
    const int32_t* table;
    uint32_t n_page, n_kv, page_rows, shift, row_mask, n_seq, seq_pages, cap;
};
struct RunsView {
    const int32_t *start, *seq, *pos;
    uint32_t n_rows, n_run, max_run;
};

constexpr uint32_t KV_NO_PAGE = 0xFFFFFFFFu;

// Page that holds row r (r < cap) of a sequence, KV_NO_PAGE where there is none.
__device__ __forceinline__ uint32_t kv_page(const KvView& c, uint32_t seq, uint32_t r)
{
    const uint32_t p = c.table ? (uint32_t)c.table[(size_t)seq * c.seq_pages + (r >> c.shift)] : seq;
    return p < c.n_page ? p : KV_NO_PAGE;
}
// Where the page id of row r is to be read, for loops that request ids ahead of their use: to be compared with n_page THEN, since a
// comparison here would wait for the load, and with it for every load in front of it.  seq_at holds the sequence's own id,
// which is the page of a slot cache.
__device__ __forceinline__ const int32_t* kv_page_at(const KvView& c, const int32_t* seq_at, uint32_t seq, uint32_t r)
{
    return c.table ? c.table + ((size_t)seq * c.seq_pages + (r >> c.shift)) : seq_at;
}
// Element offset of a row of KV head h in k or v (64 bits: a long cache passes 2^32 elements).
__device__ __forceinline__ size_t kv_row(const KvView& c, uint32_t page, uint32_t h, uint32_t r, uint32_t dh)
{
    return (((size_t)page * c.n_kv + h) * c.page_rows + (r & c.row_mask)) * dh;
}

// Last i < n with first(i) <= x for an ascending first(), or n if there is none: 64 candidates per step, one per
// lane, so up to 64 entries cost one round trip and 4096 two.  All 64 lanes of the wave call it; x wave-uniform.
template <class F>
__device__ __forceinline__ uint32_t wave_last_le(uint32_t n, int64_t x, F first)
{
    uint32_t lo = 0, len = n;
    const uint32_t lane = threadIdx.x & 63u;
    while (true) {
        const uint32_t step = (len + 63) / 64, at = lane * step;
        const bool le = at < len && first(lo + min(at, len - 1)) <= x;
        const uint32_t cnt = (uint32_t)__builtin_popcountll(__builtin_amdgcn_ballot_w64(le));
        if (cnt == 0) return n; // only in the first step: later ones begin at an entry that is <= x
        lo += (cnt - 1) * step;
        if (step == 1) return lo;
        len = min(step, len - (cnt - 1) * step);
    }
}

// A run as its rows see it: rows r0 .. r0 + n - 1, cache row pos + t for its row t.
struct Run {
    uint32_t r0, n, seq, pos;
    bool ok; // sequence and position in range
};
__device__ __forceinline__ Run run_at(const KvView& c, const RunsView& R, uint32_t i)
{
    Run u;
    const int32_t a = R.start[i], b = R.start[i + 1], s = R.seq[i], p = R.pos[i];
    const uint32_t lo = min((uint32_t)max(a, 0), R.n_rows), hi = min((uint32_t)max(b, 0), R.n_rows);
    u.r0 = lo;
    u.n = hi > lo ? min(hi - lo, R.max_run) : 0u;
    u.seq = (uint32_t)s;
    u.pos = (uint32_t)p;
    u.ok = s >= 0 && (uint32_t)s < c.n_seq && p >= 0 && (uint32_t)p <= c.cap;
    return u;
}

// ---- host ---------------------------------------------------------------------------------------------

// Checks the cache and hands back the view of one layer.
int kv_view(const char* who, const qkk_kv_cache* C, uint32_t layer, KvView* view);
// Checks the runs.
int runs_view(const char* who, const qkk_kv_runs* R, RunsView* view);

} // namespace qk
