// qk_attn_axes.hip -- what stands in front of the attention over runs (qkk_attn_prep_axes): per head RMS norm of the
// queries and keys, rotation with several position axes, keys and values written to their rows of the paged cache.
// The one-axis form on a slot's own cache is qkk_attn_prep (qk_attn.hip); no reference counterpart for the axes.
//   x^ = x * w / sqrt(mean(x^2) + eps);  pair (j, j + n_rot/2) turned by (cos, sin) = rope[axis_pos[pair_axis[j]][row]][j]
// Bound by memory: a row's heads are read once and written once, and the angles are a few hundred bytes per row.
#include "qk_kv.h"

namespace qk {

// One wave per (row, head): a lane holds dh / 64 neighbouring values, the partner of a rotated value comes through a
// wave-private LDS row.  grid ceil(rows * heads / 4), heads = hQ queries, then n_kv keys, then n_kv values.
template <int DH, typename T>
__global__ __launch_bounds__(256) void attn_prep_axes_kernel(KvView c, RunsView R, const float* __restrict__ q, const float* __restrict__ kin,
                                                             const float* __restrict__ vin, const float* __restrict__ qn,
                                                             const float* __restrict__ kn, const float* __restrict__ rope, uint32_t rope_rows,
                                                             const uint8_t* __restrict__ pair_axis, uint32_t n_axis,
                                                             const int32_t* __restrict__ axis_pos, float* __restrict__ qhat, uint32_t hQ,
                                                             uint32_t n_rot, uint32_t q_pitch, float eps)
{
    constexpr uint32_t PER = DH / 64;
    __shared__ float s_row[4][DH];
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, heads = hQ + 2 * c.n_kv;
    const uint64_t job = (uint64_t)blockIdx.x * 4 + wave;
    const uint32_t row = (uint32_t)(job / heads), w = (uint32_t)(job % heads);
    if (row >= R.n_rows) return; // the whole wave; no workgroup barrier below
    const uint32_t ri = wave_last_le(R.n_run, row, [&](uint32_t i) { return (int64_t)R.start[i]; });
    if (ri >= R.n_run) return;
    const Run u = run_at(c, R, ri);
    if (!u.ok || row - u.r0 >= u.n) return;
    const bool is_q = w < hQ, is_v = w >= hQ + c.n_kv;
    const uint32_t h = is_q ? w : is_v ? w - hQ - c.n_kv : w - hQ;
    const uint32_t at = u.pos + (row - u.r0);
    uint32_t page = KV_NO_PAGE;
    if (!is_q) {
        if (at < c.cap) page = kv_page(c, u.seq, at);
        if (page == KV_NO_PAGE) return;
    }
    const float* x = is_q ? q + ((size_t)row * hQ + h) * q_pitch : (is_v ? vin : kin) + ((size_t)row * c.n_kv + h) * DH;
    float y[PER];
#pragma unroll
    for (uint32_t e = 0; e < PER; e++) y[e] = x[PER * lane + e];
    if (!is_v) {
        const float* g = is_q ? qn : kn;
        float ss = 0.f;
#pragma unroll
        for (uint32_t e = 0; e < PER; e++) ss += y[e] * y[e];
        const float scale = 1.f / sqrtf(wave_sum(ss) / (float)DH + eps);
#pragma unroll
        for (uint32_t e = 0; e < PER; e++) {
            y[e] = y[e] * scale * g[PER * lane + e];
            s_row[wave][PER * lane + e] = y[e];
        }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        const uint32_t half = n_rot / 2;
#pragma unroll
        for (uint32_t e = 0; e < PER; e++) {
            const uint32_t d = PER * lane + e;
            if (d >= n_rot) continue;
            const uint32_t j = d < half ? d : d - half;
            const int32_t p = axis_pos[(size_t)min((uint32_t)pair_axis[j], n_axis - 1u) * R.n_rows + row];
            const size_t ang = 2 * ((size_t)min((uint32_t)max(p, 0), rope_rows - 1u) * half + j);
            const float cs = rope[ang], sn = rope[ang + 1], x0 = s_row[wave][j], x1 = s_row[wave][j + half];
            y[e] = d < half ? x0 * cs - x1 * sn : x0 * sn + x1 * cs;
        }
    }
    if (is_q) {
        float* out = qhat + ((size_t)row * hQ + h) * DH + PER * lane;
#pragma unroll
        for (uint32_t e = 0; e < PER; e++) out[e] = y[e];
    } else {
        T* out = (T*)(is_v ? c.v : c.k) + kv_row(c, page, h, at, DH) + PER * lane;
#pragma unroll
        for (uint32_t e = 0; e < PER; e++) out[e] = (T)y[e];
    }
}

} // namespace qk

using namespace qk;

extern "C" {

int qkk_rope_axes(uint8_t* axis_host, uint32_t n_rot, const uint32_t* sections_host, uint32_t n_axis, int in_turn)
{
    if (!axis_host || !sections_host) return fail(QKK_EINVAL, "qkk_rope_axes: null pointer");
    if (n_axis < 1 || n_axis > QKK_MAX_AXES) return fail(QKK_ESHAPE, "qkk_rope_axes: %u axes outside 1..%u", n_axis, QKK_MAX_AXES);
    uint32_t left[QKK_MAX_AXES];
    uint64_t sum = 0;
    for (uint32_t a = 0; a < n_axis; a++) sum += left[a] = sections_host[a];
    if (n_rot < 2 || n_rot % 2 || sum != n_rot / 2)
        return fail(QKK_ESHAPE, "qkk_rope_axes: the sections hold %llu pairs, n_rot %u has %u", (unsigned long long)sum, n_rot, n_rot / 2);
    for (uint32_t j = 0, a = 0; j < n_rot / 2; j++) {
        while (!left[a]) a = (a + 1) % n_axis;
        axis_host[j] = (uint8_t)a;
        left[a]--;
        if (in_turn) a = (a + 1) % n_axis;
    }
    return QKK_OK;
}

int qkk_attn_prep_axes(const qkk_kv_cache* C, uint32_t layer, const qkk_kv_runs* R, const float* q, const float* kin, const float* vin,
                       const float* q_norm_w, const float* k_norm_w, const float* rope, uint32_t rope_rows, const uint8_t* pair_axis,
                       uint32_t n_axis, const int32_t* axis_pos, float* qhat, uint32_t hQ, uint32_t n_rot, int gated, float eps, void* stream)
{
    const char* who = "qkk_attn_prep_axes";
    KvView c;
    RunsView runs;
    if (int rc = kv_view(who, C, layer, &c)) return rc;
    if (int rc = runs_view(who, R, &runs)) return rc;
    if (!q || !kin || !vin || !q_norm_w || !k_norm_w || !rope || !pair_axis || !axis_pos || !qhat) return fail(QKK_EINVAL, "%s: null pointer", who);
    if (!aligned16(q) || !aligned16(kin) || !aligned16(vin) || !aligned16(qhat) || !aligned16(q_norm_w) || !aligned16(k_norm_w) || !aligned16(rope))
        return fail(QKK_EINVAL, "%s: q, kin, vin, qhat, the norm weights and rope must be 16-byte aligned", who);
    if (hQ < 1 || hQ > 4096) return fail(QKK_ESHAPE, "%s: %u query heads outside 1..4096", who, hQ);
    if (n_rot < 2 || n_rot % 2 || n_rot > C->dh) return fail(QKK_ESHAPE, "%s: n_rot %u must be even, 2..%u", who, n_rot, C->dh);
    if (n_axis < 1 || n_axis > QKK_MAX_AXES) return fail(QKK_ESHAPE, "%s: %u axes outside 1..%u", who, n_axis, QKK_MAX_AXES);
    if (rope_rows < 1) return fail(QKK_ESHAPE, "%s: rope_rows must be positive", who);
    if (!(eps >= 0.f)) return fail(QKK_EINVAL, "%s: eps must be non-negative", who);
    if (int rc = require_device()) return rc;
    if (!runs.n_rows || !runs.n_run) return QKK_OK;
    const uint64_t jobs = (uint64_t)runs.n_rows * (hQ + 2 * c.n_kv);
    if (jobs > (1ull << 32)) return fail(QKK_ESHAPE, "%s: rows x heads too large", who);
    const dim3 grid((uint32_t)((jobs + 3) / 4)), block(256);
    const uint32_t pitch = (gated ? 2u : 1u) * C->dh;
#define QK_PREP(DH, T)                                                                                                                     \
    hipLaunchKernelGGL((attn_prep_axes_kernel<DH, T>), grid, block, 0, as_stream(stream), c, runs, q, kin, vin, q_norm_w, k_norm_w, rope,  \
                       rope_rows, pair_axis, n_axis, axis_pos, qhat, hQ, n_rot, pitch, eps)
    if (C->dh == 256) {
        if (C->type == QKK_F32) QK_PREP(256, float);
        else QK_PREP(256, _Float16);
    } else {
        if (C->type == QKK_F32) QK_PREP(128, float);
        else QK_PREP(128, _Float16);
    }
#undef QK_PREP
    return check_launch(who);
}

} // extern "C"
