// qk_attn_few.hip -- attention of runs with FEW query rows (one or two blocks of 16 per run and KV head: decode steps, small trees) over
// the paged cache.  Bound by reading the cache, which every run does once per KV head.
//
// A workgroup takes one run, one KV head and one range of keys; its four waves take the range's steps in turn, 32 keys or (half
// cache, dh 128) 64.  A wave loads the A operands of both products straight from the cache into registers, nothing goes
// through LDS:
//   K  lane (m, g) holds 8 dims per step of 32 dims of key m (rows of the S^T block);
//   V  lane (m, g) holds, of the 8 keys that its P covers, 4 (fp32) or 8 (half) NEIGHBOURING dims: which dims a block of 16
//      rows of O^T stands for is free, so block e of a group takes dim E*m + e of lane m, and loads stay 16 bytes wide, 256
//      bytes side by side, without a transposition.
// A step is 32 KB per wave in flight: its K and V are requested together, the next step's K when this one's scores are done and
// its V when this one's values are.  Only fp32 with dh 256, where a step is 64 KB, requests V in two halves behind the two
// halves of K (registers).  What a launch of a few steps per wave spends is the chain of round trips: run -> page table -> keys;
// queries and parents are requested before the keys and prepared while those arrive.
// An fp32 cache is split into three bf16 pieces in registers (exact, fp32's whole range, NaN and infinities stay in their
// key), six of the nine products are kept (the others are below 2^-23 of their terms); a half cache is an operand as it is,
// and queries and weights go in as hi + lo halves: two products.  Matrix work is a few percent of the time either way.
//   One row for each of sixteen sequences of 1 .. 4096 half rows, 32 heads on 8 of 128 (63 MB): 21 us and 4 us for the join, 2.6 TB/s
// where a large copy moves 4.8; six of the 21 pass before the first keys arrive (lengths, page ids, keys: three round trips).
#include "qk_attn_runs.h"

namespace qk {

typedef u32x4 __attribute__((may_alias)) lds_u32x4;
typedef f32x4 __attribute__((may_alias)) lds_f32x4;
typedef uint32_t __attribute__((may_alias)) lds_pair;

template <int DH, bool F32, int RT, bool TREE>
__global__ __launch_bounds__(256, (DH == 128 && RT == 1 ? 2 : 1)) void attn_few_kernel(RunsCall a)
{
    constexpr uint32_t KS = DH / 32;            // steps of 32 dims
    constexpr uint32_t E = F32 ? 4 : 8;         // neighbouring dims a lane loads
    constexpr uint32_t NC = DH / (16 * E);      // groups of 16 E dims
    constexpr uint32_t NT = DH / 16;            // blocks of 16 dims
    constexpr uint32_t NP = F32 ? 3 : 2;        // pieces of a split operand
    constexpr uint32_t OP = DH + 4;             // pitch of an accumulator row in LDS (floats)
    QK_DYN_LDS(uint8_t, s_dyn);                 // the Q operand [piece][rt][ks][lane], later two waves' accumulators
    __shared__ float s_m[2][RT * 16], s_l[2][RT * 16];
    __shared__ int32_t s_up[TREE ? QKK_TREE_MAX : 1];
    __shared__ uint32_t s_kin[TREE ? RT * 16 : 1][QKK_TREE_MAX / 32];
    const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), m = lane & 15u, g = lane >> 4;
    const uint32_t kv = blockIdx.x % a.c.n_kv;
    const Item it = item_of(a, blockIdx.x / a.c.n_kv, RT * 16, false);
    if (!it.ok) return; // the whole workgroup
    const Run u = it.u;
    const uint32_t run = it.run, split = it.split;
    const uint32_t nr = u.n * a.G, end = min(u.pos + u.n, a.c.cap), k_begin = split * it.chunk;
    const uint32_t k_end = min(end, k_begin + it.chunk);
    const bool drafts = TREE && k_end > u.pos; // uniform: this range holds rows of the tree itself
    int32_t up_of = -1;
    if (drafts) up_of = tree_parent(a.parent, u);

    // Q: wave w prepares rows 4 RT w .. 4 RT w + 4 RT - 1, a lane PER neighbouring dims
    constexpr uint32_t PER = DH / 64;
    float qx[4 * RT][PER];
#pragma unroll
    for (uint32_t i = 0; i < 4 * RT; i++) {
        const uint32_t f = 4 * RT * wave + i;
#pragma unroll
        for (uint32_t j = 0; j < PER; j++)
            qx[i][j] = f < nr ? a.q[((size_t)(u.r0 + f / a.G) * a.hQ + kv * a.G + f % a.G) * DH + PER * lane + j] : 0.f;
    }

    // one step's operands: K [sub-step of 32 keys][block of 16 keys][step of 32 dims], V [sub-step][group][key of the lane's 8]
    constexpr uint32_t SUB = !F32 && DH == 128 ? 2 : 1, SK = 32 * SUB; // sub-steps, keys per step
    constexpr uint32_t KW = F32 ? 2 : 1;                               // 16-byte pieces per lane, block and step of dims
    constexpr bool HALVES = F32 && DH == 256;                          // V in two halves, behind those of K
    constexpr uint32_t CA = HALVES ? NC / 2 : NC;                      // groups of V's first part
    const uint32_t n_step = (k_end - k_begin + SK - 1) / SK;
    u32x4 kreg[SUB][2][KS][KW], vreg[SUB][NC][8];
    const u32x4 zero = {0, 0, 0, 0};
    const uint8_t* kbase = (const uint8_t*)a.c.k;
    const uint8_t* vbase = (const uint8_t*)a.c.v;
    constexpr uint32_t ES = F32 ? 4 : 2;
    // the page ids of a step's blocks of 16 keys (a page holds a multiple of 16 rows; a slot cache is one page), requested a step ahead of
    // the rows and not looked at before; behind the last step the last block's again
    auto pages = [&](uint32_t step, uint32_t* pg) {
#pragma unroll
        for (uint32_t b = 0; b < 2 * SUB; b++) pg[b] = (uint32_t)*kv_page_at(a.c, a.R.seq + run, u.seq, min(k_begin + SK * step + 16 * b, k_end - 1));
    };
    auto valid = [&](uint32_t step, uint32_t b, const uint32_t* pg) { return pg[b] < a.c.n_page && k_begin + SK * step + 16 * b < k_end; };
    // block b of K.  Rows behind the range repeat its last one (masked below); without a page, and behind the last step: zeros, no load
    auto fetch_k = [&](uint32_t step, uint32_t b, const uint32_t* pg) {
        const uint32_t key = min(k_begin + SK * step + 16 * b + m, k_end - 1);
        if (valid(step, b, pg)) { // uniform
            const uint8_t* row = kbase + kv_row(a.c, pg[b], kv, key, DH) * ES;
#pragma unroll
            for (uint32_t ks = 0; ks < KS; ks++)
#pragma unroll
                for (uint32_t w = 0; w < KW; w++) kreg[b / 2][b % 2][ks][w] = *(const u32x4*)(row + (F32 ? ks * 128 + w * 64 : ks * 64) + g * 16);
        } else {
#pragma unroll
            for (uint32_t ks = 0; ks < KS; ks++)
#pragma unroll
                for (uint32_t w = 0; w < KW; w++) kreg[b / 2][b % 2][ks][w] = zero;
        }
    };
    // groups c0 .. c1 - 1 of sub-step sb of V
    auto fetch_v = [&](uint32_t step, uint32_t sb, uint32_t c0, uint32_t c1, const uint32_t* pg) {
#pragma unroll
        for (uint32_t i = 0; i < 8; i++) {
            const uint32_t b = 2 * sb + i / 4, key = min(k_begin + SK * step + 16 * b + 4 * g + i % 4, k_end - 1);
            if (valid(step, b, pg)) { // uniform
                const uint8_t* row = vbase + kv_row(a.c, pg[b], kv, key, DH) * ES;
#pragma unroll
                for (uint32_t c = c0; c < c1; c++) vreg[sb][c][i] = *(const u32x4*)(row + (c * 16 + m) * 16);
            } else {
#pragma unroll
                for (uint32_t c = c0; c < c1; c++) vreg[sb][c][i] = zero;
            }
        }
    };
    uint32_t pg[2 * SUB], pg_next[2 * SUB];
    pages(wave, pg);
    __builtin_amdgcn_sched_barrier(0); // the queries are on their way before the keys
#pragma unroll
    for (uint32_t b = 0; b < 2 * SUB; b++) fetch_k(wave, b, pg);
    if (!HALVES) {
#pragma unroll
        for (uint32_t sb = 0; sb < SUB; sb++) fetch_v(wave, sb, 0, NC, pg);
    }
    __builtin_amdgcn_sched_barrier(0);

    {
        uint16_t* s_q = (uint16_t*)s_dyn;
        const uint32_t d = PER * lane, ks = d / 32, in = d % 32;
        // the lane group and the place among its 8 values that hold dim `in` of a step
        const uint32_t qg = F32 ? in % 16 / 4 : in / 8, qt = F32 ? in / 16 * 4 + in % 4 : in % 8;
#pragma unroll
        for (uint32_t i = 0; i < 4 * RT; i++) {
            const uint32_t f = 4 * RT * wave + i, rt = f / 16;
            float scale = 1.f;
            if (!F32) {
                float mx = 0.f;
#pragma unroll
                for (uint32_t j = 0; j < PER; j++) mx = fmaxf(mx, fabsf(qx[i][j]));
                mx = wave_max(mx);
                const int e = top_exponent(mx);
                scale = pow2i(-e);
                if (lane == 0) s_m[0][f] = pow2i(e);
            }
            uint16_t bits[NP][PER];
#pragma unroll
            for (uint32_t j = 0; j < PER; j++) {
                float v = qx[i][j] * scale;
#pragma unroll
                for (uint32_t p = 0; p < NP; p++) {
                    if (F32) {
                        bits[p][j] = (uint16_t)(f2u(v) >> 16);
                        v -= u2f(f2u(v) & 0xFFFF0000u);
                    } else {
                        const _Float16 hv = (_Float16)v;
                        bits[p][j] = __builtin_bit_cast(uint16_t, hv);
                        v -= (float)hv;
                    }
                }
            }
#pragma unroll
            for (uint32_t p = 0; p < NP; p++) {
                uint16_t* at = s_q + (((p * RT + rt) * KS + ks) * 64 + 16 * qg + f % 16) * 8 + qt;
#pragma unroll
                for (uint32_t j = 0; j < PER; j += 2) *(lds_pair*)(at + j) = (uint32_t)bits[p][j] | (uint32_t)bits[p][j + 1] << 16;
            }
        }
    }
    if (drafts) tree_bits(up_of, 0, u.n, s_up, s_kin);
    __syncthreads();
    float q_exp[RT]; // 2^exponent the lane's row was divided by (half caches)
#pragma unroll
    for (uint32_t rt = 0; rt < RT; rt++) q_exp[rt] = F32 ? 1.f : s_m[0][16 * rt + m];
    const lds_u32x4* q_op = (const lds_u32x4*)s_dyn;

    const float qs = AR_LOG2E / sqrtf((float)DH);
    float4v o[RT][NT];
    float m_run[RT], l_run[RT];
#pragma unroll
    for (uint32_t rt = 0; rt < RT; rt++) {
        m_run[rt] = AR_FLOOR;
        l_run[rt] = 0.f;
#pragma unroll
        for (uint32_t t = 0; t < NT; t++) o[rt][t] = float4v{0.f, 0.f, 0.f, 0.f};
    }
    for (uint32_t step = wave; step < n_step; step += 4) {
        const uint32_t key0 = k_begin + SK * step;
        pages(step + 4, pg_next);
        // scores
        float4v s[RT][2 * SUB];
#pragma unroll
        for (uint32_t b = 0; b < 2 * SUB; b++) {
#pragma unroll
            for (uint32_t rt = 0; rt < RT; rt++) s[rt][b] = float4v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (uint32_t ks = 0; ks < KS; ks++) {
                const u32x4* kr = kreg[b / 2][b % 2][ks];
                if constexpr (F32) {
                    float x[8];
#pragma unroll
                    for (uint32_t i = 0; i < 8; i++) x[i] = u2f(kr[i / 4][i % 4]);
                    const Bf3 k3 = split3(x);
#pragma unroll
                    for (uint32_t rt = 0; rt < RT; rt++) {
                        bf16x8 qq[3];
#pragma unroll
                        for (uint32_t p = 0; p < 3; p++) qq[p] = __builtin_bit_cast(bf16x8, u32x4(q_op[((p * RT + rt) * KS + ks) * 64 + lane]));
                        // smallest products first
                        s[rt][b] = mfma16x32(k3.p[2], qq[0], s[rt][b]);
                        s[rt][b] = mfma16x32(k3.p[0], qq[2], s[rt][b]);
                        s[rt][b] = mfma16x32(k3.p[1], qq[1], s[rt][b]);
                        s[rt][b] = mfma16x32(k3.p[1], qq[0], s[rt][b]);
                        s[rt][b] = mfma16x32(k3.p[0], qq[1], s[rt][b]);
                        s[rt][b] = mfma16x32(k3.p[0], qq[0], s[rt][b]);
                    }
                } else {
                    const half8 kh = __builtin_bit_cast(half8, u32x4(kr[0]));
#pragma unroll
                    for (uint32_t rt = 0; rt < RT; rt++) {
                        s[rt][b] = mfma16x32(kh, __builtin_bit_cast(half8, u32x4(q_op[((RT + rt) * KS + ks) * 64 + lane])), s[rt][b]);
                        s[rt][b] = mfma16x32(kh, __builtin_bit_cast(half8, u32x4(q_op[(rt * KS + ks) * 64 + lane])), s[rt][b]);
                    }
                }
                if (ks % 2) __builtin_amdgcn_sched_barrier(0); // the Q operand's reads stay near their use: registers
            }
            if (HALVES) {
                if (b == 0) fetch_v(step, 0, 0, CA, pg);
                else fetch_v(step, 0, CA, NC, pg);
            } else fetch_k(step + 4, b, pg_next);
            __builtin_amdgcn_sched_barrier(0);
        }
        // softmax: this lane's row 16 rt + m, keys 16 b + 4 g + r
        bool whole = key0 + SK <= k_end && key0 + SK <= u.pos + (TREE ? 0u : 1u); // uniform
#pragma unroll
        for (uint32_t b = 0; b < 2 * SUB; b++) whole = whole && pg[b] < a.c.n_page;
        uint32_t seen[RT]; // bit 4 b + r: the row sees that key
        Bf3 p3[RT][SUB];
        Half2 p2[RT][SUB];
#pragma unroll
        for (uint32_t rt = 0; rt < RT; rt++) {
            const float cf = qs * q_exp[rt];
#pragma unroll
            for (uint32_t b = 0; b < 2 * SUB; b++) s[rt][b] *= cf;
            seen[rt] = 0xFFFFu;
            if (!whole) { // uniform
                const uint32_t f = 16 * rt + m, node = min(f, nr - 1) / a.G;
                seen[rt] = 0;
#pragma unroll
                for (uint32_t b = 0; b < 2 * SUB; b++) { // four neighbouring keys at a time
                    const uint32_t key = key0 + 16 * b + 4 * g;
                    const uint32_t stop = pg[b] >= a.c.n_page || f >= nr ? 0u : TREE ? k_end : min(k_end, u.pos + node + 1);
                    uint32_t four = (1u << (stop > key ? min(stop - key, 4u) : 0u)) - 1u;
                    if (drafts) four &= tree_four(s_kin[node], (int32_t)(key - u.pos));
                    seen[rt] |= four << (4 * b);
#pragma unroll
                    for (uint32_t r = 0; r < 4; r++) s[rt][b][r] = (four >> r) & 1u ? s[rt][b][r] : -INFINITY;
                }
            }
            float mx = AR_FLOOR;
#pragma unroll
            for (uint32_t i = 0; i < 8 * SUB; i++) mx = fmaxf(mx, s[rt][i / 4][i % 4]);
            const float m_new = fmaxf(m_run[rt], xor_lanes_max(mx));
            const float corr = __builtin_amdgcn_exp2f(m_run[rt] - m_new);
            m_run[rt] = m_new;
            float sum = 0.f;
#pragma unroll
            for (uint32_t sb = 0; sb < SUB; sb++) {
                float p[8];
#pragma unroll
                for (uint32_t i = 0; i < 8; i++) {
                    p[i] = __builtin_amdgcn_exp2f(s[rt][2 * sb + i / 4][i % 4] - m_new);
                    sum += p[i];
                }
                // weights of a half cache up to 2^14, so that the lo halves of small ones stay normal; undone at the end
                if constexpr (F32) p3[rt][sb] = split3(p);
                else {
#pragma unroll
                    for (uint32_t i = 0; i < 8; i++) p[i] *= 16384.f;
                    p2[rt][sb] = split2(p);
                }
            }
            l_run[rt] = l_run[rt] * corr + sum; // of this lane's keys; the lane groups are added at the end
            if (__builtin_amdgcn_ballot_w64(corr != 1.f)) { // uniform
#pragma unroll
                for (uint32_t t = 0; t < NT; t++) o[rt][t] *= corr;
            }
        }
        // Where not every row sees every key, values that are not finite are taken out of the product (a weight of zero would not
        // keep them out) and added to the rows that do see them.
        uint32_t odd = 0; // bit 8 sb + i: the lane's key i of 8 holds such a value
        auto clean = [&](uint32_t sb, uint32_t c0, uint32_t c1) {
#pragma unroll
            for (uint32_t i = 0; i < 8; i++) {
                bool bad = false;
#pragma unroll
                for (uint32_t c = c0; c < c1; c++)
#pragma unroll
                    for (uint32_t w = 0; w < 4; w++) {
                        const uint32_t x = vreg[sb][c][i][w];
                        if (F32) {
                            const bool b1 = (x & 0x7F800000u) == 0x7F800000u;
                            bad = bad || b1;
                            vreg[sb][c][i][w] = b1 ? 0u : x;
                        } else {
                            const bool b0 = (x & 0x7C00u) == 0x7C00u, b1 = (x & 0x7C000000u) == 0x7C000000u;
                            bad = bad || b0 || b1;
                            vreg[sb][c][i][w] = (b0 ? 0u : x & 0xFFFFu) | (b1 ? 0u : x & 0xFFFF0000u);
                        }
                    }
                const uint64_t who = __builtin_amdgcn_ballot_w64(bad);
                odd |= ((who >> (16 * g)) & 0xFFFFu ? 1u : 0u) << (8 * sb + i);
            }
        };
        auto values = [&](uint32_t sb, uint32_t c0, uint32_t c1) {
#pragma unroll
            for (uint32_t c = c0; c < c1; c++)
#pragma unroll
                for (uint32_t e = 0; e < E; e++) {
                    if constexpr (F32) {
                        float x[8];
#pragma unroll
                        for (uint32_t i = 0; i < 8; i++) x[i] = u2f(vreg[sb][c][i][e]);
                        const Bf3 v3 = split3(x);
#pragma unroll
                        for (uint32_t rt = 0; rt < RT; rt++) {
                            float4v& acc = o[rt][c * E + e];
                            acc = mfma16x32(v3.p[2], p3[rt][sb].p[0], acc);
                            acc = mfma16x32(v3.p[0], p3[rt][sb].p[2], acc);
                            acc = mfma16x32(v3.p[1], p3[rt][sb].p[1], acc);
                            acc = mfma16x32(v3.p[1], p3[rt][sb].p[0], acc);
                            acc = mfma16x32(v3.p[0], p3[rt][sb].p[1], acc);
                            acc = mfma16x32(v3.p[0], p3[rt][sb].p[0], acc);
                        }
                    } else {
                        u32x4 w;
#pragma unroll
                        for (uint32_t i = 0; i < 4; i++) // half e of keys 2 i, 2 i + 1
                            w[i] = __builtin_amdgcn_perm(vreg[sb][c][2 * i + 1][e / 2], vreg[sb][c][2 * i][e / 2], e % 2 ? 0x07060302u : 0x05040100u);
                        const half8 vh = __builtin_bit_cast(half8, w);
#pragma unroll
                        for (uint32_t rt = 0; rt < RT; rt++) {
                            float4v& acc = o[rt][c * E + e];
                            acc = mfma16x32(vh, p2[rt][sb].lo, acc);
                            acc = mfma16x32(vh, p2[rt][sb].hi, acc);
                        }
                    }
                }
        };
        if (HALVES) {
            if (!whole) clean(0, 0, CA);
            values(0, 0, CA);
            __builtin_amdgcn_sched_barrier(0);
            fetch_k(step + 4, 0, pg_next);
            if (!whole) clean(0, CA, NC);
            values(0, CA, NC);
            __builtin_amdgcn_sched_barrier(0);
            fetch_k(step + 4, 1, pg_next);
        } else {
#pragma unroll
            for (uint32_t sb = 0; sb < SUB; sb++) {
                if (!whole) clean(sb, 0, NC);
                values(sb, 0, NC);
                __builtin_amdgcn_sched_barrier(0);
                fetch_v(step + 4, sb, 0, NC, pg_next);
            }
        }
        __builtin_amdgcn_sched_barrier(0);
        if (__builtin_amdgcn_ballot_w64(odd != 0)) { // rare: uniform
            for (uint32_t kk = 0; kk < SK; kk++) {
                const uint32_t kg = kk % 16 / 4, i = kk / 16 * 4 + kk % 4; // lane group and place (bit) of key kk
                const uint32_t flags = (uint32_t)__shfl((int)odd, (int)(16 * kg));
                if (!((flags >> i) & 1u)) continue; // uniform
                const uint32_t key = key0 + kk;
                if (key >= k_end) continue; // uniform (rows behind the range repeat its last one)
                const uint8_t* row = vbase + kv_row(a.c, kv_page(a.c, u.seq, key), kv, key, DH) * ES;
#pragma unroll
                for (uint32_t rt = 0; rt < RT; rt++) {
                    const bool sees = ((uint32_t)__shfl((int)seen[rt], (int)(16 * kg + m)) >> i) & 1u;
#pragma unroll
                    for (uint32_t c = 0; c < NC; c++)
#pragma unroll
                        for (uint32_t e = 0; e < E; e++) {
                            __builtin_amdgcn_sched_barrier(0); // registers: not all loads at once
#pragma unroll
                            for (uint32_t r = 0; r < 4; r++) {
                                const uint32_t d = 16 * E * c + E * (4 * g + r) + e;
                                const float v = F32 ? ((const float*)row)[d] : (float)((const _Float16*)row)[d];
                                if (sees && !(fabsf(v) < INFINITY)) o[rt][c * E + e][r] += v;
                            }
                        }
                }
            }
        }
#pragma unroll
        for (uint32_t b = 0; b < 2 * SUB; b++) pg[b] = pg_next[b];
    }

    // the four waves' partial results: 2, 3 into 0, 1, then 1 into 0
#pragma unroll
    for (uint32_t rt = 0; rt < RT; rt++) l_run[rt] = xor_lanes_sum(l_run[rt]);
    float* s_o = (float*)s_dyn;
#pragma unroll
    for (uint32_t half = 2; half >= 1; half /= 2) {
        __syncthreads(); // the area is free: the Q operand, or the pair before, has been read
        if (wave >= half && wave < 2 * half) {
            const uint32_t at = wave - half;
#pragma unroll
            for (uint32_t rt = 0; rt < RT; rt++) {
                if (g == 0) {
                    s_m[at][16 * rt + m] = m_run[rt];
                    s_l[at][16 * rt + m] = l_run[rt];
                }
#pragma unroll
                for (uint32_t c = 0; c < NC; c++)
#pragma unroll
                    for (uint32_t r = 0; r < 4; r++)
#pragma unroll
                        for (uint32_t e = 0; e < E; e += 4)
                            *(lds_f32x4*)(s_o + ((size_t)at * RT * 16 + 16 * rt + m) * OP + 16 * E * c + E * (4 * g + r) + e) =
                                f32x4{o[rt][c * E + e][r], o[rt][c * E + e + 1][r], o[rt][c * E + e + 2][r], o[rt][c * E + e + 3][r]};
            }
        }
        __syncthreads();
        if (wave < half) {
#pragma unroll
            for (uint32_t rt = 0; rt < RT; rt++) {
                const float mo = s_m[wave][16 * rt + m], lo = s_l[wave][16 * rt + m];
                const float m_new = fmaxf(m_run[rt], mo);
                const float fa = __builtin_amdgcn_exp2f(m_run[rt] - m_new), fb = __builtin_amdgcn_exp2f(mo - m_new);
                m_run[rt] = m_new;
                l_run[rt] = l_run[rt] * fa + lo * fb;
#pragma unroll
                for (uint32_t c = 0; c < NC; c++) {
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (uint32_t r = 0; r < 4; r++)
#pragma unroll
                        for (uint32_t e = 0; e < E; e += 4) {
                            const f32x4 x = *(const lds_f32x4*)(s_o + ((size_t)wave * RT * 16 + 16 * rt + m) * OP + 16 * E * c + E * (4 * g + r) + e);
#pragma unroll
                            for (uint32_t i = 0; i < 4; i++) o[rt][c * E + e + i][r] = o[rt][c * E + e + i][r] * fa + x[i] * fb;
                        }
                }
            }
        }
    }
    if (wave != 0) return;
    constexpr float UNIT = F32 ? 1.f : 1.f / 16384.f; // the weights' factor
#pragma unroll
    for (uint32_t rt = 0; rt < RT; rt++) {
        const uint32_t f = 16 * rt + m;
        if (f >= nr) continue;
        const size_t rh = (size_t)(u.r0 + f / a.G) * a.hQ + kv * a.G + f % a.G;
        const float inv = l_run[rt] == 0.f ? 0.f : UNIT / l_run[rt];
        float* out = a.n_split > 1 ? a.acc + (rh * a.n_split + split) * DH : a.att + rh * DH;
        if (a.n_split > 1 && g == 0) {
            a.ml[2 * (rh * a.n_split + split)] = m_run[rt];
            a.ml[2 * (rh * a.n_split + split) + 1] = l_run[rt];
        }
#pragma unroll
        for (uint32_t c = 0; c < NC; c++)
#pragma unroll
            for (uint32_t r = 0; r < 4; r++)
#pragma unroll
                for (uint32_t e = 0; e < E; e += 4) {
                    const uint32_t d = 16 * E * c + E * (4 * g + r) + e;
                    f32x4 x;
#pragma unroll
                    for (uint32_t i = 0; i < 4; i++) x[i] = o[rt][c * E + e + i][r] * inv;
                    if (a.n_split == 1 && a.qfull) {
                        const f32x4 gt = *(const f32x4*)(a.qfull + rh * 2 * DH + DH + d);
#pragma unroll
                        for (uint32_t i = 0; i < 4; i++) x[i] *= 1.f / (1.f + expf(-gt[i]));
                    }
                    *(f32x4*)(out + d) = x;
                }
    }
}

template <int DH, bool F32, int RT>
static void launch_few(const RunsCall& a, bool tree, hipStream_t st)
{
    constexpr uint32_t q_bytes = (F32 ? 3 : 2) * RT * (DH / 32) * 1024, o_bytes = 2 * RT * 16 * (DH + 4) * 4;
    constexpr uint32_t lds = q_bytes > o_bytes ? q_bytes : o_bytes;
    const dim3 grid(items_of(a.R.n_run, a.slots, a.n_split) * a.c.n_kv), block(256);
    static_assert(lds <= 65536, "more would have to be asked for (allow_lds)");
    if (tree) hipLaunchKernelGGL((attn_few_kernel<DH, F32, RT, true>), grid, block, lds, st, a);
    else hipLaunchKernelGGL((attn_few_kernel<DH, F32, RT, false>), grid, block, lds, st, a);
}

void launch_attn_few(const RunsCall& a, int type, uint32_t dh, bool tree, hipStream_t st)
{
    const bool one = a.R.max_run * a.G <= 16;
    if (dh == 256) {
        if (type == QKK_F32) launch_few<256, true, 1>(a, tree, st);
        else launch_few<256, false, 1>(a, tree, st);
    } else {
        if (type == QKK_F32) one ? launch_few<128, true, 1>(a, tree, st) : launch_few<128, true, 2>(a, tree, st);
        else one ? launch_few<128, false, 1>(a, tree, st) : launch_few<128, false, 2>(a, tree, st);
    }
}

} // namespace qk
