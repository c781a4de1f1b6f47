// qk_attn_axes.hip -- what stands in front of the attention over runs (qkk_attn_prep_axes): per head RMS norm of the
// queries and keys, rotation with several position axes, keys and values written to their rows of the paged cache.
// The one-axis form on a slot's own cache is qkk_attn_prep (qk_attn.hip); no reference counterpart for the axes.
//   x^ = x * w / sqrt(mean(x^2) + eps);  pair (j, j + n_rot/2) turned by (cos, sin) = rope[axis_pos[pair_axis[j]][row]][j]
// Bound by memory: a row's heads are read once and written once, and the angles are a few hundred bytes per row.
#include "qk_kv.h"

namespace qk {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef f32x4 __attribute__((may_alias)) lds_f32x4;
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));

// One workgroup per row and group of heads (hQ queries, then n_kv keys, then n_kv values, counted through).  A lane holds four
// neighbouring values of a head, so a wave takes 64 / (dh / 4) heads at a time, N times; all its loads are requested before
// anything else.  Which four dims a lane holds does not depend on the head, so it fetches its angles once for all of them: per dim d
//   out = y * c + partner * s,  partner = y[d + half] and s = -sin for d < half, y[d - half] and sin behind, c = 1, s = 0 past n_rot.
// The partner comes through a wave-private LDS row.  (One wave per head, each with its own search for the run and its own angles, spent
// 117 us on 4312 rows of 48 heads of 128, a chain of round trips per wave; the bytes alone take 41.)
template <int DH, typename T, int N>
__global__ __launch_bounds__(256) void attn_prep_axes_kernel(KvView c, RunsView R, const float* __restrict__ q, const float* __restrict__ kin,
                                                             const float* __restrict__ vin, const float* __restrict__ qn,
                                                             const float* __restrict__ kn, const float* __restrict__ rope, uint32_t rope_rows,
                                                             const uint8_t* __restrict__ pair_axis, uint32_t n_axis,
                                                             const int32_t* __restrict__ axis_pos, float* __restrict__ qhat, uint32_t hQ,
                                                             uint32_t n_rot, uint32_t q_pitch, float eps)
{
    constexpr uint32_t LPH = DH / 4, HW = 64 / LPH; // lanes per head, heads per wave and step
    __shared__ __attribute__((aligned(16))) float s_row[4][HW * DH];
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, sub = lane / LPH, d0 = lane % LPH * 4;
    const uint32_t row = blockIdx.x, heads = hQ + 2 * c.n_kv, w0 = (blockIdx.y * 4 + wave) * N * HW + sub;
    f32x4 x[N];
#pragma unroll
    for (uint32_t i = 0; i < N; i++) {
        const uint32_t w = min(w0 + i * HW, heads - 1); // behind the last head that one again, not stored
        const float* from = w < hQ ? q + ((size_t)row * hQ + w) * q_pitch
                          : w < hQ + c.n_kv ? kin + ((size_t)row * c.n_kv + (w - hQ)) * DH : vin + ((size_t)row * c.n_kv + (w - hQ - c.n_kv)) * DH;
        x[i] = *(const f32x4*)(from + d0);
    }
    const f32x4 gq = *(const f32x4*)(qn + d0), gk = *(const f32x4*)(kn + d0);
    const uint32_t half = n_rot / 2;
    float cs[4], sn[4];
    uint32_t partner[4];
#pragma unroll
    for (uint32_t e = 0; e < 4; e++) {
        const uint32_t d = d0 + e, j = d < half ? d : d - half;
        cs[e] = 1.f;
        sn[e] = 0.f;
        partner[e] = d;
        if (d < n_rot) {
            const int32_t p = axis_pos[(size_t)min((uint32_t)pair_axis[j], n_axis - 1u) * R.n_rows + row];
            const size_t ang = 2 * ((size_t)min((uint32_t)max(p, 0), rope_rows - 1u) * half + j);
            cs[e] = rope[ang];
            sn[e] = d < half ? -rope[ang + 1] : rope[ang + 1];
            partner[e] = d < half ? d + half : j;
        }
    }
    const uint32_t ri = wave_last_le(R.n_run, row, [&](uint32_t i) { return (int64_t)R.start[i]; });
    if (ri >= R.n_run) return; // the whole workgroup, and no barrier below
    const Run u = run_at(c, R, ri);
    if (!u.ok || row - u.r0 >= u.n) return;
    const uint32_t at = u.pos + (row - u.r0);
    uint32_t page = KV_NO_PAGE;
    if (at < c.cap) page = kv_page(c, u.seq, at);
#pragma unroll
    for (uint32_t i = 0; i < N; i++) {
        const uint32_t w = w0 + i * HW;
        const bool is_q = w < hQ, is_v = w >= hQ + c.n_kv;
        const f32x4 v = x[i];
        const float scale = 1.f / sqrtf(lanes_sum<(int)LPH>(v[0] * v[0] + v[1] * v[1] + v[2] * v[2] + v[3] * v[3]) / (float)DH + eps);
        f32x4 y;
#pragma unroll
        for (uint32_t e = 0; e < 4; e++) y[e] = v[e] * scale * (is_q ? gq[e] : gk[e]);
        *(lds_f32x4*)&s_row[wave][sub * DH + d0] = y;
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        f32x4 out;
#pragma unroll
        for (uint32_t e = 0; e < 4; e++) {
            const float turned = y[e] * cs[e] + s_row[wave][sub * DH + partner[e]] * sn[e];
            out[e] = is_v ? v[e] : turned;
        }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier(); // the next head overwrites the row
        if (w >= heads) continue;
        if (is_q) *(f32x4*)(qhat + ((size_t)row * hQ + w) * DH + d0) = out;
        else if (page != KV_NO_PAGE) {
            const uint32_t h = is_v ? w - hQ - c.n_kv : w - hQ;
            T* to = (T*)(is_v ? c.v : c.k) + kv_row(c, page, h, at, DH) + d0;
            if constexpr (sizeof(T) == 4) *(f32x4*)to = out;
            else *(f16x4*)to = f16x4{(_Float16)out[0], (_Float16)out[1], (_Float16)out[2], (_Float16)out[3]};
        }
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
    if (!q_norm_w || !k_norm_w || !rope || !pair_axis || (runs.n_rows && (!q || !kin || !vin || !axis_pos || !qhat))) return fail(QKK_EINVAL, "%s: null pointer", who);
    if (!aligned16(q) || !aligned16(kin) || !aligned16(vin) || !aligned16(qhat) || !aligned16(q_norm_w) || !aligned16(k_norm_w) || !aligned16(rope))
        return fail(QKK_EINVAL, "%s: q, kin, vin, qhat, the norm weights and rope must be 16-byte aligned", who);
    if (hQ < 1 || hQ > 4096) return fail(QKK_ESHAPE, "%s: %u query heads outside 1..4096", who, hQ);
    if (n_rot < 2 || n_rot % 2 || n_rot > C->dh) return fail(QKK_ESHAPE, "%s: n_rot %u must be even, 2..%u", who, n_rot, C->dh);
    if (n_axis < 1 || n_axis > QKK_MAX_AXES) return fail(QKK_ESHAPE, "%s: %u axes outside 1..%u", who, n_axis, QKK_MAX_AXES);
    if (rope_rows < 1) return fail(QKK_ESHAPE, "%s: rope_rows must be positive", who);
    if (!(eps >= 0.f)) return fail(QKK_EINVAL, "%s: eps must be non-negative", who);
    if (int rc = require_device()) return rc;
    if (!runs.n_rows || !runs.n_run) return QKK_OK;
    // heads per workgroup: 4 waves times heads per wave and step, times steps -- six where the rows alone fill the device several times
    // (4312 rows of 48 heads: 8 workgroups per CU), one where few rows have to be spread
    const uint32_t heads = hQ + 2 * c.n_kv, per = 4 * (256 / C->dh), steps = runs.n_rows >= 1024 ? 6 : 1;
    const dim3 grid(runs.n_rows, (heads + per * steps - 1) / (per * steps)), block(256);
    const uint32_t pitch = (gated ? 2u : 1u) * C->dh;
#define QK_PREP(DH, T, N)                                                                                                                  \
    hipLaunchKernelGGL((attn_prep_axes_kernel<DH, T, N>), grid, block, 0, as_stream(stream), c, runs, q, kin, vin, q_norm_w, k_norm_w, rope, \
                       rope_rows, pair_axis, n_axis, axis_pos, qhat, hQ, n_rot, pitch, eps)
#define QK_PREP_N(DH, T) do { if (steps == 6) QK_PREP(DH, T, 6); else QK_PREP(DH, T, 1); } while (0)
    if (C->dh == 256) {
        if (C->type == QKK_F32) QK_PREP_N(256, float);
        else QK_PREP_N(256, _Float16);
    } else {
        if (C->type == QKK_F32) QK_PREP_N(128, float);
        else QK_PREP_N(128, _Float16);
    }
#undef QK_PREP_N
#undef QK_PREP
    return check_launch(who);
}

} // extern "C"
