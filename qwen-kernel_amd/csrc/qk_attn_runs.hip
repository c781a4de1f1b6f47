// qk_attn_runs.hip -- attention of runs of rows over the paged cache (qkk_attn_packed, qkk_attn_tree).
//   att = softmax(q . K / sqrt(dh)) V * sigmoid(gate) over the cache rows a row sees: 0 .. pos + t of its sequence, or
//   for a tree the rows below pos, the node's ancestors and itself.
// The one-sequence forms on a slot's own cache are in qk_attn.hip.
#include "qk_attn_runs.h"

#include <algorithm>

namespace qk {

// One workgroup per row and 4 HB heads: folds their ranges in range order and applies the gate, each wave HB heads side by side.  Ranges
// behind the row's own position hold nothing for it.  A chain of round trips (run -> sums -> ranges),
// 5 to 13 us where its bytes would take 1 to 4: HB = 4 where that still fills the device (763 rows of 16 heads: 12.4 us, 15.7
// with one head per wave), one head per wave where there are few rows (16 of 32 heads: 3.9 us against 9).
template <int DH, int HB>
__global__ __launch_bounds__(256) void attn_join_kernel(RunsCall a)
{
    constexpr uint32_t PER = DH / 64; // floats per lane
    typedef float vec __attribute__((ext_vector_type(PER)));
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, row = blockIdx.x;
    const uint32_t common = *a.chunk_used;
    const uint32_t ri = wave_last_le(a.R.n_run, row, [&](uint32_t i) { return (int64_t)a.R.start[i]; });
    if (ri >= a.R.n_run) return; // the whole workgroup
    const Run u = run_at(a.c, a.R, ri);
    if (!u.ok || row - u.r0 >= u.n) return; // the whole workgroup
    const uint32_t chunk = run_chunk(min(u.pos + u.n, a.c.cap), common, a.grain);
    const uint32_t n = __builtin_amdgcn_readfirstlane((min(u.pos + (row - u.r0) + 1, a.c.cap) + chunk - 1) / chunk);
    {
        const uint32_t h0 = blockIdx.y * 4 * HB + wave; // and every fourth behind it
        float f[HB], l[HB];
        size_t at[HB];
        vec gate[HB], o[HB];
#pragma unroll
        for (uint32_t b = 0; b < HB; b++) {
            const size_t rh = (size_t)row * a.hQ + min(h0 + 4 * b, a.hQ - 1); // behind the last head that one again, not stored
            at[b] = rh * a.n_split;
            f[b] = AR_FLOOR;
            l[b] = 0.f;
            if (lane < n) {
                f[b] = a.ml[2 * (at[b] + lane)];
                l[b] = a.ml[2 * (at[b] + lane) + 1];
            }
            if (a.qfull) gate[b] = *(const vec*)(a.qfull + rh * 2 * DH + DH + PER * lane);
#pragma unroll
            for (uint32_t e = 0; e < PER; e++) o[b][e] = 0.f;
        }
        // a range's share of the whole sum; NaN where a range saw one, which the sums below carry on
#pragma unroll
        for (uint32_t b = 0; b < HB; b++) {
            const float top = wave_max(f[b]);
            f[b] = lane < n ? __builtin_amdgcn_exp2f(f[b] - top) * l[b] : 0.f;
            const float sum = wave_sum(f[b]);
            f[b] *= sum == 0.f ? 0.f : 1.f / sum;
        }
        for (uint32_t s0 = 0; s0 < n; s0 += 4) {
            vec x[HB][4];
#pragma unroll
            for (uint32_t b = 0; b < HB; b++)
#pragma unroll
                for (uint32_t i = 0; i < 4; i++) x[b][i] = *(const vec*)(a.acc + (at[b] + min(s0 + i, n - 1)) * DH + PER * lane);
#pragma unroll
            for (uint32_t b = 0; b < HB; b++)
#pragma unroll
                for (uint32_t i = 0; i < 4; i++) {
                    const float w = __shfl(f[b], (int)min(s0 + i, 63u));
                    if (s0 + i < n) o[b] += x[b][i] * w; // uniform
                }
        }
#pragma unroll
        for (uint32_t b = 0; b < HB; b++) {
            if (h0 + 4 * b >= a.hQ) continue; // uniform
            vec v = o[b];
            if (a.qfull) {
#pragma unroll
                for (uint32_t e = 0; e < PER; e++) v[e] *= 1.f / (1.f + expf(-gate[b][e]));
            }
            *(vec*)(a.att + ((size_t)row * a.hQ + h0 + 4 * b) * DH + PER * lane) = v;
        }
    }
}

// How a call is cut, from what the host knows (never from the lengths, which live on the device, so that a captured launch
// follows them): which kernel, and how short the ranges of keys that run in parallel may get.  The workspace is sized by it.
struct Plan {
    bool few;
    uint32_t n_split, chunk, grain, slots;
};
static Plan plan_of(const qkk_kv_cache* C, const qkk_kv_runs* R, uint32_t hQ)
{
    const uint32_t G = hQ / C->n_kv, max_run = std::min(R->max_run, R->n_rows);
    const uint64_t cap = (uint64_t)C->seq_pages * C->page_rows;
    Plan p;
    p.few = (uint64_t)max_run * G <= few_rows(C->dh);
    // places on the device: two workgroups per CU (256) where registers and LDS allow two
    const bool two = C->dh == 128 && (!p.few || (uint64_t)max_run * G <= 16);
    p.slots = std::max(1u, (two ? 512u : 256u) / C->n_kv);
    uint64_t ranges = 64; // at most: the join's lanes
    if (!p.few) {
        // one range where the blocks of rows fill the chip, else no more than two per place: the partial results are memory, too
        const uint64_t groups = std::max<uint64_t>(((uint64_t)R->n_rows * G + AR_TILE_ROWS - 1) / AR_TILE_ROWS, R->n_run) * C->n_kv;
        ranges = groups >= 256 ? 1 : std::min<uint64_t>(64, (1024 + groups - 1) / groups);
    }
    // few rows: a range is at least one step per wave (128 keys; 256 on halves with dh 128); many rows: one or two tiles
    p.grain = !p.few ? 64 : C->type == QKK_F16 && C->dh == 128 ? 256 : 128;
    p.chunk = (uint32_t)std::max<uint64_t>(1, ((cap + ranges - 1) / ranges + p.grain - 1) / p.grain) * p.grain;
    p.n_split = (uint32_t)((cap + p.chunk - 1) / p.chunk);
    return p;
}

static int attn_runs(const char* who, const qkk_kv_cache* C, uint32_t layer, const qkk_kv_runs* R, const int32_t* parent, bool tree,
                     const float* qhat, const float* qfull, float* att, void* workspace, size_t workspace_bytes, uint32_t hQ, void* stream)
{
    KvView c;
    RunsView runs;
    if (int rc = kv_view(who, C, layer, &c)) return rc;
    if (int rc = runs_view(who, R, &runs)) return rc;
    if (!workspace || (runs.n_rows && (!qhat || !att || (tree && !parent)))) return fail(QKK_EINVAL, "%s: null pointer", who);
    if (hQ < c.n_kv || hQ % c.n_kv || hQ > 4096)
        return fail(QKK_ESHAPE, "%s: %u query heads on %u KV heads not supported (a multiple, at most 4096)", who, hQ, c.n_kv);
    if (tree && runs.max_run > QKK_TREE_MAX) return fail(QKK_ESHAPE, "%s: trees of up to %u nodes (at most %u)", who, runs.max_run, QKK_TREE_MAX);
    if (!aligned16(qhat) || !aligned16(att) || !aligned16(qfull) || (reinterpret_cast<uintptr_t>(workspace) & 255u))
        return fail(QKK_EINVAL, "%s: qhat, qfull and att must be 16-byte, workspace 256-byte aligned", who);
    const size_t want = qkk_attn_runs_workspace_bytes(C, R, hQ);
    if (workspace_bytes < want) return fail(QKK_EWORKSPACE, "%s: workspace %zu < %zu bytes", who, workspace_bytes, want);
    if (int rc = require_device()) return rc;
    if (!runs.n_rows || !runs.n_run) return QKK_OK;
    const Plan plan = plan_of(C, R, hQ);
    if (((uint64_t)(tile_blocks(runs.n_rows, runs.n_run, hQ / c.n_kv)) + 2 * plan.slots) * c.n_kv > (1u << 22) || (uint64_t)runs.n_rows * hQ > (1u << 30))
        return fail(QKK_ESHAPE, "%s: rows x heads or runs x heads too large", who);
    {
        RunsCall a;
        a.c = c;
        a.R = runs;
        a.parent = parent;
        a.q = qhat;
        a.qfull = qfull;
        a.att = att;
        a.acc = (float*)workspace;
        a.ml = a.acc + (size_t)runs.n_rows * hQ * plan.n_split * C->dh;
        a.hQ = hQ;
        a.G = hQ / c.n_kv;
        a.n_split = plan.n_split;
        a.chunk = plan.chunk;
        a.grain = plan.grain;
        a.slots = plan.slots;
        a.chunk_used = (uint32_t*)(a.ml + 2 * (size_t)runs.n_rows * hQ * plan.n_split);
        if (plan.few) launch_attn_few(a, C->type, C->dh, tree, as_stream(stream));
        else launch_attn_tile(a, C->type, C->dh, tree, as_stream(stream));
        if (plan.n_split > 1) {
            const bool side = (uint64_t)runs.n_rows * hQ >= 16 * 512;
            const dim3 jobs(runs.n_rows, (hQ + (side ? 15 : 3)) / (side ? 16 : 4));
            if (C->dh == 256) {
                if (side) hipLaunchKernelGGL((attn_join_kernel<256, 4>), jobs, dim3(256), 0, as_stream(stream), a);
                else hipLaunchKernelGGL((attn_join_kernel<256, 1>), jobs, dim3(256), 0, as_stream(stream), a);
            } else {
                if (side) hipLaunchKernelGGL((attn_join_kernel<128, 4>), jobs, dim3(256), 0, as_stream(stream), a);
                else hipLaunchKernelGGL((attn_join_kernel<128, 1>), jobs, dim3(256), 0, as_stream(stream), a);
            }
        }
    }
    return check_launch(who);
}

} // namespace qk

using namespace qk;

extern "C" {

size_t qkk_attn_runs_workspace_bytes(const qkk_kv_cache* C, const qkk_kv_runs* R, uint32_t hQ)
{
    if (!C || !R || !C->n_kv || hQ < C->n_kv || !C->seq_pages || !C->page_rows) return 0;
    // what the calls refuse: the sums below are not made for it
    if ((uint64_t)C->seq_pages * C->page_rows > (1u << 30) || R->n_rows > (1u << 20) || R->n_run > (1u << 20) || hQ > 4096 || C->dh > 256) return 0;
    const Plan p = plan_of(C, R, hQ);
    return (p.n_split > 1 ? (size_t)R->n_rows * hQ * p.n_split * (C->dh + 2) * sizeof(float) : 0) + 256;
}

int qkk_attn_packed(const qkk_kv_cache* C, uint32_t layer, const qkk_kv_runs* R, const float* qhat, const float* qfull, float* att,
                    void* workspace, size_t workspace_bytes, uint32_t hQ, void* stream)
{
    return attn_runs("qkk_attn_packed", C, layer, R, nullptr, false, qhat, qfull, att, workspace, workspace_bytes, hQ, stream);
}

int qkk_attn_tree(const qkk_kv_cache* C, uint32_t layer, const qkk_kv_runs* R, const int32_t* parent, const float* qhat, const float* qfull,
                  float* att, void* workspace, size_t workspace_bytes, uint32_t hQ, void* stream)
{
    return attn_runs("qkk_attn_tree", C, layer, R, parent, true, qhat, qfull, att, workspace, workspace_bytes, hQ, stream);
}

} // extern "C"
