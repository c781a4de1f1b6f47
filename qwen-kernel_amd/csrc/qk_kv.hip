// qk_kv.hip -- the books of the paged cache, kept on the device (qkk_kv_resize, qkk_kv_fork), the copies they ask
// for, and the compaction of accepted drafted rows (qkk_kv_compact).  No counterpart in the reference.
//
// The books are a few thousand integers: one workgroup keeps them, so that no allocation depends on the order in
// which workgroups run -- the k-th page that is needed, counted over the sequences in ascending order, is the k-th
// free page in ascending order.  What is to be copied goes into a list of (page, page, rows) in the workspace, and a
// second launch over the whole device copies it for all layers, bound by memory: six copies of 1777 and 4001 rows, 20 fp32
// heads of 256, K and V (1.4 GB moved), 284 us or 5.0 TB/s.  The books themselves are a chain of passes over the tables between
// barriers: resize 2 to 6 us on pools of up to 200 pages (another pass per 1024 pages that are passed over in the search for free
// ones), fork 3.3 us for sixteen sequences; compaction of sixteen paths 5.7 us, three round trips.
#include "qk_kv.h"

#include <algorithm>

namespace qk {

constexpr uint32_t KV_TPB = 1024; // threads of the books' workgroup

// Workspace of resize / fork (words): the number of copies, then per sequence its need, its first page of the list and
// a copy (3 words), then the pages taken.
struct KvWs {
    uint32_t *n_copy, *need, *first, *copy, *taken;
};
__host__ __device__ inline KvWs kv_ws(void* p, uint32_t n_seq)
{
    uint32_t* w = (uint32_t*)p;
    return KvWs{w, w + 64, w + 64 + n_seq, w + 64 + 2 * (size_t)n_seq, w + 64 + 5 * (size_t)n_seq};
}

// References change by atomics (several sequences may hold a page), which act behind the CU's L1: read the same way.
__device__ __forceinline__ int32_t ref_load(const int32_t* p)
{
    return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ uint32_t pages_for(uint32_t rows, uint32_t shift) { return (rows >> shift) + ((rows & ((1u << shift) - 1u)) ? 1u : 0u); }

// Sum over the workgroup's 16 waves and this thread's exclusive prefix.
__device__ __forceinline__ uint32_t block_scan(uint32_t v, uint32_t* s_wave, uint32_t& total)
{
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    const uint32_t incl = wave_incl_scan_u32(v);
    if (lane == 63) s_wave[wave] = incl;
    __syncthreads();
    uint32_t before = 0, all = 0;
    for (uint32_t w = 0; w < KV_TPB / 64; w++) {
        if (w < wave) before += s_wave[w];
        all += s_wave[w];
    }
    __syncthreads(); // s_wave is used again
    total = all;
    return before + incl - v;
}

// One workgroup: see qkk_kv_resize.
__global__ __launch_bounds__(1024) void kv_resize_kernel(KvView c, int32_t* table, int32_t* ref, int32_t* len,
                                                         const int32_t* __restrict__ len_new, int32_t* status, KvWs ws)
{
    __shared__ uint32_t s_wave[KV_TPB / 64], s_n, s_bad;
    __shared__ unsigned long long s_need;
    const uint32_t t = threadIdx.x, lane = t & 63u, wave = t >> 6;
    if (t == 0) { s_n = 0; s_bad = 0; s_need = 0; }
    __syncthreads();
    for (uint32_t s = t; s < c.n_seq; s += KV_TPB)
        if (len_new[s] >= 0 && (uint32_t)len_new[s] > c.cap) s_bad = 1;
    __syncthreads();
    if (s_bad) { // the whole workgroup
        if (t == 0) { *status = -1; *ws.n_copy = 0; }
        return;
    }
    if (!c.table) {
        for (uint32_t s = t; s < c.n_seq; s += KV_TPB)
            if (len_new[s] >= 0) len[s] = len_new[s];
        if (t == 0) { *status = 0; *ws.n_copy = 0; }
        return;
    }
    auto held = [&](uint32_t s) { return min((uint32_t)max(len[s], 0), c.cap); };
    // pages behind the new end: one wave per sequence
    for (uint32_t s = wave; s < c.n_seq; s += KV_TPB / 64) {
        const uint32_t old = held(s);
        const uint32_t now = len_new[s] < 0 ? old : (uint32_t)len_new[s];
        if (now >= old) continue;
        const uint32_t have = pages_for(old, c.shift);
        for (uint32_t b = pages_for(now, c.shift) + lane; b < have; b += 64) {
            int32_t* e = table + (size_t)s * c.seq_pages + b;
            if ((uint32_t)*e < c.n_page) atomicAdd(ref + *e, -1);
            *e = -1;
        }
        __builtin_amdgcn_wave_barrier(); // every lane has read the old length
        if (lane == 0) len[s] = (int32_t)now;
    }
    publish_wait(); // the references are back where ref_load reads them
    __syncthreads();
    // what the growing sequences need, and whether they begin with a copy of a shared page
    uint32_t needed = 0; // exact where it matters: while all of it is no more than there are pages
    for (uint32_t s0 = 0; s0 < c.n_seq; s0 += KV_TPB) {
        const uint32_t s = s0 + t;
        uint32_t need = 0;
        if (s < c.n_seq) {
            const uint32_t old = held(s), now = len_new[s] < 0 ? old : (uint32_t)len_new[s];
            uint32_t split = 0;
            if (now > old) {
                if (old & c.row_mask) {
                    const uint32_t p = (uint32_t)table[(size_t)s * c.seq_pages + (old >> c.shift)];
                    split = p < c.n_page && ref_load(ref + p) > 1;
                }
                need = pages_for(now, c.shift) - pages_for(old, c.shift) + split;
            }
            ws.need[s] = 2 * need + split;
            if (need) atomicAdd(&s_need, (unsigned long long)need);
        }
        uint32_t total;
        const uint32_t before = block_scan(need, s_wave, total);
        if (s < c.n_seq) ws.first[s] = needed + before;
        needed += total;
    }
    __syncthreads();
    const uint64_t all = s_need;
    if (all > c.n_page) needed = 0xFFFFFFFFu; // cannot be met: only the free pages are counted below
    // the free pages, lowest first, as many as are needed
    uint32_t found = 0;
    for (uint32_t p0 = 0; p0 < c.n_page && found < needed; p0 += KV_TPB) {
        const uint32_t p = p0 + t;
        const uint32_t is_free = p < c.n_page && ref_load(ref + p) == 0;
        uint32_t total;
        const uint32_t at = found + block_scan(is_free, s_wave, total);
        if (is_free && at < needed) ws.taken[at] = p;
        found += total;
    }
    __syncthreads();
    if (found < needed) {
        if (t == 0) { *status = (int32_t)min(all - found, (uint64_t)0x7FFFFFFF); *ws.n_copy = 0; }
        return;
    }
    for (uint32_t s = wave; s < c.n_seq; s += KV_TPB / 64) {
        const uint32_t need = ws.need[s] >> 1, split = ws.need[s] & 1u, first = ws.first[s], old = held(s);
        const int32_t now = len_new[s];
        __builtin_amdgcn_wave_barrier(); // every lane has read the old length
        if (now < 0 || (uint32_t)now <= old) continue;
        const uint32_t have = pages_for(old, c.shift);
        int32_t* row = table + (size_t)s * c.seq_pages;
        for (uint32_t i = split + lane; i < need; i += 64) {
            const uint32_t p = ws.taken[first + i];
            row[have + i - split] = (int32_t)p;
            ref[p] = 1;
        }
        if (lane == 0) {
            if (split) {
                const uint32_t p = ws.taken[first], from = (uint32_t)row[have - 1];
                row[have - 1] = (int32_t)p;
                ref[p] = 1;
                atomicAdd(ref + from, -1);
                uint32_t* cp = ws.copy + 3 * (size_t)atomicAdd(&s_n, 1u);
                cp[0] = from;
                cp[1] = p;
                cp[2] = old & c.row_mask;
            }
            len[s] = now;
        }
    }
    __syncthreads();
    if (t == 0) { *status = 0; *ws.n_copy = s_n; }
}

// One workgroup: see qkk_kv_fork.
__global__ __launch_bounds__(1024) void kv_fork_kernel(KvView c, int32_t* table, int32_t* ref, int32_t* len,
                                                       const int32_t* __restrict__ src, const int32_t* __restrict__ dst, uint32_t n,
                                                       int32_t* status, KvWs ws)
{
    __shared__ uint32_t s_bad;
    const uint32_t t = threadIdx.x, lane = t & 63u, wave = t >> 6;
    if (t == 0) s_bad = 0;
    for (uint32_t s = t; s < c.n_seq; s += KV_TPB) publish(ws.need + s, 0u); // how often a sequence is a dst
    publish_wait();
    __syncthreads();
    for (uint32_t i = t; i < n; i += KV_TPB) {
        const uint32_t a = (uint32_t)src[i], b = (uint32_t)dst[i];
        if (a >= c.n_seq || b >= c.n_seq || len[b] != 0 || len[a] < 0 || (uint32_t)len[a] > c.cap || atomicAdd(ws.need + b, 1u) != 0)
            s_bad = 1;
    }
    __syncthreads();
    if (s_bad) { // the whole workgroup
        if (t == 0) { *status = -1; *ws.n_copy = 0; }
        return;
    }
    // the lengths are written behind the next barrier: a src that holds nothing may be another pair's dst
    for (uint32_t i = wave; i < n; i += KV_TPB / 64) {
        const uint32_t a = (uint32_t)src[i], b = (uint32_t)dst[i];
        if (lane == 0) ws.first[i] = (uint32_t)len[a];
        if (c.table) {
            const uint32_t have = pages_for((uint32_t)len[a], c.shift);
            for (uint32_t k = lane; k < have; k += 64) {
                const int32_t p = table[(size_t)a * c.seq_pages + k];
                table[(size_t)b * c.seq_pages + k] = p;
                if ((uint32_t)p < c.n_page) atomicAdd(ref + p, 1);
            }
        } else if (lane == 0) {
            uint32_t* cp = ws.copy + 3 * (size_t)i;
            cp[0] = a;
            cp[1] = b;
            cp[2] = (uint32_t)len[a];
        }
    }
    __syncthreads();
    for (uint32_t i = t; i < n; i += KV_TPB) len[dst[i]] = (int32_t)ws.first[i];
    if (t == 0) { *status = 0; *ws.n_copy = c.table ? 0u : n; }
}

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// The listed copies (page, page, rows), all layers and heads, K and V: the rows of a head lie side by side in a page, so
// a copy is a run of 16-byte pieces, cut into chunks of 1024 pieces.  A grid that fills the device goes over the chunks
// of all copies; chunks behind a copy's rows are passed over.
constexpr uint32_t KV_CHUNK = 1024;
__global__ __launch_bounds__(256) void kv_copy_kernel(uint8_t* k, uint8_t* v, KvWs ws, uint32_t n_layer, uint32_t n_page, uint32_t n_kv,
                                                      uint32_t page_rows, uint32_t row_pieces)
{
    const uint32_t n = *ws.n_copy;
    const uint32_t chunks = (uint32_t)(((uint64_t)page_rows * row_pieces + KV_CHUNK - 1) / KV_CHUNK);
    const uint64_t per = (uint64_t)n_layer * n_kv * 2 * chunks;
    for (uint64_t it = blockIdx.x; it < per * n; it += gridDim.x) {
        const uint32_t i = (uint32_t)(it / per);
        uint64_t r = it % per;
        const uint32_t at = (uint32_t)(r % chunks) * KV_CHUNK;
        r /= chunks;
        const uint32_t* cp = ws.copy + 3 * (size_t)i;
        const uint32_t end = cp[2] * row_pieces;
        if (at >= end) continue;
        u32x4* pool = (u32x4*)((r & 1) ? v : k);
        r >>= 1;
        const uint32_t h = (uint32_t)(r % n_kv), layer = (uint32_t)(r / n_kv);
        const size_t page = (size_t)page_rows * row_pieces;
        const u32x4* from = pool + (((size_t)layer * n_page + cp[0]) * n_kv + h) * page;
        u32x4* to = pool + (((size_t)layer * n_page + cp[1]) * n_kv + h) * page;
        u32x4 x[KV_CHUNK / 256];
#pragma unroll
        for (uint32_t j = 0; j < KV_CHUNK / 256; j++) x[j] = from[min(at + j * 256 + threadIdx.x, end - 1)];
#pragma unroll
        for (uint32_t j = 0; j < KV_CHUNK / 256; j++)
            if (at + j * 256 + threadIdx.x < end) to[at + j * 256 + threadIdx.x] = x[j];
    }
}

// One wave per (path, layer, KV head, K or V): rows base + path[j] to base + j.  path[j] >= j, strictly ascending, so a
// row that is written is never one that a later j reads: batches of rows are read whole before they are written.
constexpr uint32_t KV_BATCH = 8; // pieces per lane and batch
__global__ __launch_bounds__(256) void kv_compact_kernel(uint8_t* k, uint8_t* v, KvView c, const int32_t* __restrict__ seq,
                                                         const int32_t* __restrict__ base, const int32_t* __restrict__ path,
                                                         const int32_t* __restrict__ n_path, uint32_t n, uint32_t max_path, uint32_t n_layer,
                                                         uint32_t row_pieces)
{
    const uint32_t lane = threadIdx.x & 63u;
    const uint64_t job = (uint64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const uint32_t per = n_layer * c.n_kv * 2;
    if (job >= (uint64_t)n * per) return; // the whole wave
    const uint32_t i = (uint32_t)(job / per), r = (uint32_t)(job % per), h = (r >> 1) % c.n_kv, layer = (r >> 1) / c.n_kv;
    const uint32_t s = (uint32_t)seq[i], b = (uint32_t)base[i];
    const int32_t cnt = n_path[i];
    if (s >= c.n_seq || b > c.cap || cnt <= 0 || (uint32_t)cnt > max_path) return; // the whole wave
    const int32_t* P = path + (size_t)i * max_path;
    bool ok = true;
    for (uint32_t j = lane; j < (uint32_t)cnt; j += 64) {
        const int32_t p = P[j];
        ok = ok && p > (j ? P[j - 1] : -1) && (uint32_t)p < c.cap - b && kv_page(c, s, b + (uint32_t)p) != KV_NO_PAGE &&
             kv_page(c, s, b + j) != KV_NO_PAGE;
    }
    if (__builtin_amdgcn_ballot_w64(!ok)) return; // the whole wave
    u32x4* pool = (u32x4*)((r & 1) ? v : k) + (size_t)layer * c.n_page * c.n_kv * c.page_rows * row_pieces;
    const uint32_t rows = 64 / row_pieces, sub = lane / row_pieces, piece = lane % row_pieces; // rows per wave instruction
    for (uint32_t j0 = 0; j0 < (uint32_t)cnt; j0 += KV_BATCH * rows) {
        u32x4 x[KV_BATCH];
#pragma unroll
        for (uint32_t q = 0; q < KV_BATCH; q++) {
            const uint32_t j = min(j0 + q * rows + sub, (uint32_t)cnt - 1), from = b + (uint32_t)P[j];
            x[q] = pool[kv_row(c, kv_page(c, s, from), h, from, row_pieces) + piece];
        }
        publish_wait(); // every row of the batch has arrived before one is overwritten
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (uint32_t q = 0; q < KV_BATCH; q++) {
            const uint32_t j = j0 + q * rows + sub;
            if (j < (uint32_t)cnt) pool[kv_row(c, kv_page(c, s, b + j), h, b + j, row_pieces) + piece] = x[q];
        }
        publish_wait();
        __builtin_amdgcn_wave_barrier();
    }
}

// ---- host ---------------------------------------------------------------------------------------------

int kv_view(const char* who, const qkk_kv_cache* C, uint32_t layer, KvView* view)
{
    if (!C || !C->k || !C->v) return fail(QKK_EINVAL, "%s: null pointer", who);
    if (C->type != QKK_F32 && C->type != QKK_F16) return fail(QKK_ETYPE, "%s: cache type %d not supported (F32, F16)", who, C->type);
    if (C->dh != 128 && C->dh != 256) return fail(QKK_ESHAPE, "%s: head size %u not supported (128, 256)", who, C->dh);
    if (!aligned16(C->k) || !aligned16(C->v)) return fail(QKK_EINVAL, "%s: k and v must be 16-byte aligned", who);
    if (C->n_layer < 1 || C->n_page < 1 || C->n_kv < 1 || C->n_seq < 1 || C->seq_pages < 1 || C->page_rows < 1)
        return fail(QKK_EINVAL, "%s: a size of the cache is zero", who);
    if (C->n_kv > 4096 || C->n_layer > 65535 || C->n_seq > (1u << 20) || C->n_page > (1u << 28))
        return fail(QKK_ESHAPE, "%s: cache too large (n_kv 4096, n_layer 65535, n_seq 2^20, n_page 2^28 at most)", who);
    if (layer >= C->n_layer) return fail(QKK_ESHAPE, "%s: layer %u of %u", who, layer, C->n_layer);
    uint32_t shift = 31;
    if (C->table) {
        shift = 4;
        while (shift < 16 && (1u << shift) < C->page_rows) shift++;
        if ((1u << shift) != C->page_rows)
            return fail(QKK_ESHAPE, "%s: page_rows %u must be a power of two, 16..65536", who, C->page_rows);
        if (reinterpret_cast<uintptr_t>(C->table) & 3u) return fail(QKK_EINVAL, "%s: table must be 4-byte aligned", who);
    } else if (C->seq_pages != 1 || C->n_seq > C->n_page || C->page_rows > (1u << 24))
        return fail(QKK_ESHAPE, "%s: a slot cache has one page per sequence, of at most 2^24 rows", who);
    const uint64_t cap = (uint64_t)C->seq_pages * C->page_rows;
    if (cap > (1u << 30)) return fail(QKK_ESHAPE, "%s: more than 2^30 rows per sequence", who);
    const size_t layer_bytes = (size_t)C->n_page * C->n_kv * C->page_rows * C->dh * (C->type == QKK_F32 ? 4 : 2);
    view->k = (uint8_t*)C->k + layer * layer_bytes;
    view->v = (uint8_t*)C->v + layer * layer_bytes;
    view->table = C->table;
    view->n_page = C->n_page;
    view->n_kv = C->n_kv;
    view->page_rows = C->page_rows;
    view->shift = shift;
    view->row_mask = C->table ? C->page_rows - 1u : 0x7FFFFFFFu;
    view->n_seq = C->n_seq;
    view->seq_pages = C->seq_pages;
    view->cap = (uint32_t)cap;
    return QKK_OK;
}

int runs_view(const char* who, const qkk_kv_runs* R, RunsView* view)
{
    if (!R || (R->n_run && (!R->start || !R->seq || !R->pos))) return fail(QKK_EINVAL, "%s: null pointer", who);
    if (R->n_rows > (1u << 20) || R->n_run > (1u << 20)) return fail(QKK_ESHAPE, "%s: more than 2^20 rows or runs", who);
    *view = RunsView{R->start, R->seq, R->pos, R->n_rows, R->n_run, std::min(R->max_run, R->n_rows)};
    return QKK_OK;
}

// What resize and fork share: the books must be there and the workspace large enough.
static int books_check(const char* who, const qkk_kv_cache* C, KvView* view, const void* status, const void* workspace, size_t workspace_bytes)
{
    if (int rc = kv_view(who, C, 0, view)) return rc;
    if (!C->len || (C->table && !C->ref) || !status || !workspace) return fail(QKK_EINVAL, "%s: null pointer", who);
    if (reinterpret_cast<uintptr_t>(workspace) & 255u) return fail(QKK_EINVAL, "%s: workspace must be 256-byte aligned", who);
    const size_t want = qkk_kv_workspace_bytes(C);
    if (workspace_bytes < want) return fail(QKK_EWORKSPACE, "%s: workspace %zu < %zu bytes", who, workspace_bytes, want);
    return QKK_OK;
}

static void launch_copy(const qkk_kv_cache* C, const KvWs& ws, uint32_t n_max, hipStream_t st)
{
    const uint32_t row_pieces = C->dh * (C->type == QKK_F32 ? 4 : 2) / 16;
    const uint64_t chunks = ((uint64_t)C->page_rows * row_pieces + KV_CHUNK - 1) / KV_CHUNK;
    const uint64_t items = (uint64_t)n_max * C->n_layer * C->n_kv * 2 * chunks;
    const uint32_t grid = (uint32_t)std::min<uint64_t>(items, 2 * (uint64_t)persistent_blocks());
    hipLaunchKernelGGL(kv_copy_kernel, dim3(grid), dim3(256), 0, st, (uint8_t*)C->k, (uint8_t*)C->v, ws, C->n_layer, C->n_page, C->n_kv,
                       C->page_rows, row_pieces);
}

} // namespace qk

using namespace qk;

extern "C" {

size_t qkk_kv_workspace_bytes(const qkk_kv_cache* C)
{
    if (!C) return 0;
    return (64 + 5 * (size_t)C->n_seq + C->n_page) * sizeof(uint32_t);
}

int qkk_kv_resize(const qkk_kv_cache* C, const int32_t* len_new, int32_t* status, void* workspace, size_t workspace_bytes, void* stream)
{
    KvView view;
    if (int rc = books_check("qkk_kv_resize", C, &view, status, workspace, workspace_bytes)) return rc;
    if (!len_new) return fail(QKK_EINVAL, "qkk_kv_resize: null pointer");
    if (int rc = require_device()) return rc;
    const KvWs ws = kv_ws(workspace, C->n_seq);
    hipLaunchKernelGGL(kv_resize_kernel, dim3(1), dim3(KV_TPB), 0, as_stream(stream), view, C->table, C->ref, C->len, len_new, status, ws);
    if (C->table) launch_copy(C, ws, C->n_seq, as_stream(stream));
    return check_launch("qkk_kv_resize");
}

int qkk_kv_fork(const qkk_kv_cache* C, const int32_t* src, const int32_t* dst, uint32_t n, int32_t* status, void* workspace,
                size_t workspace_bytes, void* stream)
{
    KvView view;
    if (int rc = books_check("qkk_kv_fork", C, &view, status, workspace, workspace_bytes)) return rc;
    if (n && (!src || !dst)) return fail(QKK_EINVAL, "qkk_kv_fork: null pointer");
    if (n > C->n_seq) return fail(QKK_ESHAPE, "qkk_kv_fork: %u forks, %u sequences", n, C->n_seq);
    if (int rc = require_device()) return rc;
    const KvWs ws = kv_ws(workspace, C->n_seq);
    hipLaunchKernelGGL(kv_fork_kernel, dim3(1), dim3(KV_TPB), 0, as_stream(stream), view, C->table, C->ref, C->len, src, dst, n, status, ws);
    if (!C->table && n) launch_copy(C, ws, n, as_stream(stream));
    return check_launch("qkk_kv_fork");
}

int qkk_kv_compact(const qkk_kv_cache* C, const int32_t* seq, const int32_t* base, const int32_t* path, const int32_t* n_path, uint32_t n,
                   uint32_t max_path, void* stream)
{
    KvView view;
    if (int rc = kv_view("qkk_kv_compact", C, 0, &view)) return rc;
    if (n && max_path && (!seq || !base || !path || !n_path)) return fail(QKK_EINVAL, "qkk_kv_compact: null pointer");
    if (n > C->n_seq || max_path > QKK_TREE_MAX)
        return fail(QKK_ESHAPE, "qkk_kv_compact: %u paths (of %u sequences) of up to %u rows (at most %u)", n, C->n_seq, max_path, QKK_TREE_MAX);
    const uint64_t jobs = (uint64_t)n * C->n_layer * C->n_kv * 2;
    if (jobs > (1ull << 25)) return fail(QKK_ESHAPE, "qkk_kv_compact: paths x layers x heads too large");
    if (int rc = require_device()) return rc;
    if (!n || !max_path) return QKK_OK;
    const uint32_t row_pieces = C->dh * (C->type == QKK_F32 ? 4 : 2) / 16;
    hipLaunchKernelGGL(kv_compact_kernel, dim3((uint32_t)((jobs + 3) / 4)), dim3(256), 0, as_stream(stream), (uint8_t*)C->k, (uint8_t*)C->v, view,
                       seq, base, path, n_path, n, max_path, C->n_layer, row_pieces);
    return check_launch("qkk_kv_compact");
}

} // extern "C"
