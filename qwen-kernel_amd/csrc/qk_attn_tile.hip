// qk_attn_tile.hip -- attention of runs with MANY query rows (prompts, wide trees) over the paged cache: tiles of 128 query
// rows (positions x heads of one KV head's group), keys staged through LDS as matrix-core operands.
//
// A workgroup takes 128 rows of one run and one KV head, each of its waves 16 (dh 256) or 32 (dh 128) of them from end to end, its
// Q operand and its accumulators in registers: two waves per SIMD, so one's softmax runs beside another's products.  A
// tile of 32 (fp32) or 64 (half) keys goes from the cache to registers while the tile before it is worked on -- half of the waves
// load K, the others V -- and from there to the other one of two LDS buffers:
// Both operands lie in LDS in the order in which the matrix instruction's lanes read them, 64 x 16 bytes per fragment, so reads are
// linear and free of bank conflicts (rows with 16 bytes of padding lost a fifth of the time to them):
//   K    fragments [block of 16 keys][step of 32 dims]; a thread stages pieces of one or two rows;
//   V^T  fragments [block of 16 dims][step of 32 keys]; a thread stages 8 keys x 4 (fp32) or 8 (half) dims, in the order of keys
//        that the weights P have in the registers of the first product, 16 bytes per dim.
// One barrier per tile.  Matrix work per key and row: 4 dh operations times the products of split operands.
//   F16 cache   K and V are operands as they are, Q and P are hi + lo halves: two products.
//   F32 cache   every row of K and V is divided by the power of two that brings its largest value into [2^14, 2^15) and
//               split into hi + lo halves, three products (lo . lo is below 2^-22 of its term): half the matrix work of three
//               bf16 pieces.  The powers of two go back in where they cost little: a key's and a query's, added, into their scores (a
//               product of both as factors would pass fp32's range where the score does not), a value row's into its weight,
//               P V = (P 2^e) (V 2^-e).  The sum is of the weights P alone, against the maximum of the scores alone: with 2^e in
//               it a row of small values beside large ones would fall out of it.  The weights that are multiplied have a power
//               of two of their own per query row, 2^-vx, which follows the largest P 2^e.
// What two halves hold is to 2^-22 exact while the lo half is normal, so everything that is split lies as high in a half's range as it may
// (sums are fp32: 2^15 2^15 times the keys): elements down to 2^-16 of their row's largest are exact to 2^-22, smaller ones to 2^-39
// of that; weights around 2^11, not 1, are to 2^-36 of the row's largest (half caches: the sum has the same factor).
//   Bound by the matrix cores, fed from LDS.  Prompts of 8191 and 3001 rows, fp32, 16 heads on 2 of 256: 1.95 ms, 3 x 320 TFLOP/s
// of products where a large matrix product reaches 1091; three chunks of 777 .. 2048 rows behind up to 6000, half, 32 heads on 8 of 128:
// 0.60 ms, 2 x 418 TFLOP/s.  A tile of 32 fp32 keys takes 2.2 to 2.8 us, 64 half keys 3.4 us.  A call of a few tiles is a
// chain of round trips: 9 us pass before the first product (lengths 2, queries 3, first tile 4).
//   Tried and dropped: staging cut up between the products, which keeps both sides' registers live and spills (4.7 ms).
#include "qk_attn_runs.h"

namespace qk {

typedef u32x4 __attribute__((may_alias)) lds_u32x4;
typedef u32x2 __attribute__((may_alias)) lds_u32x2;
typedef f32x4 __attribute__((may_alias)) lds_f32x4;
typedef int32_t i32x4 __attribute__((ext_vector_type(4)));
typedef i32x4 __attribute__((may_alias)) lds_i32x4;
typedef int32_t __attribute__((may_alias)) lds_i32;

constexpr uint32_t TL_M = AR_TILE_ROWS;
// The running maximum is moved only when a score passes it by more than 2^TL_SLACK: weights stay below 2^(TL_UP + TL_SLACK), inside a
// half's range, and most tiles need neither an exchange between lanes nor a rescaling of the accumulators.  What is left above the maximum is
// lost below it: with 2^13 and 2^2 prompts of 8191 and 3001 rows take 1.05 of the time with 2^6 and 2^8, so 1.03.
constexpr float TL_UP = 11.f, TL_SLACK = 4.f, TL_TOP = 32768.f; // 2^(TL_UP + TL_SLACK)
constexpr int TL_VX = 1000; // vx stays above -TL_VX

template <int DH, bool F32>
struct TileGeom {
    static constexpr uint32_t ES = F32 ? 4 : 2, NH = F32 ? 2 : 1;
    static constexpr uint32_t WAVES = DH / 32;                     // dh 128: 4 waves of 32 rows, two workgroups per CU; 256: 8 waves of 16 rows, one
    static constexpr uint32_t RT = TL_M / WAVES / 16;              // blocks of 16 rows per wave
    static constexpr uint32_t LPR = DH * ES / 16;                  // 16-byte pieces of a row = lanes that load one
    static constexpr uint32_t NB = F32 ? 1 : 2, BN = 32 * NB;      // steps of 32 keys per tile
    static constexpr uint32_t KB = BN * DH * 2, VB = KB;           // bytes of one copy of K, of V^T
    static constexpr uint32_t RL = F32 ? 8 : 16, QL = 64 / RL;     // staging K: rows, and pieces of each, per wave and load
    static constexpr uint32_t PI = LPR / QL, KR = 8 / PI;          // loads per row, rows per thread
    static constexpr uint32_t EXP = F32 ? 2 * BN * 4 : 0;          // per key: exponents of the score and of the value row
    static constexpr uint32_t BUF = NH * (KB + VB) + EXP + 64;     // + flags [4 NB]
    // Operand fragments read ahead of the products, and whether that order is pinned: left to itself the scheduler keeps two in flight,
    // which costs dh 256 4 % and suits halves with dh 128; fp32 with dh 128 has registers for one only.
    static constexpr uint32_t AHEAD = DH == 256 ? 3 : 1;
    static constexpr bool PIN = DH == 256 || F32;
    // half of the waves stage K, the others V: eight pieces per thread
    static_assert(NB * LPR * 4 == WAVES * 32 && WAVES / 2 * RL * KR == BN, "staging");
};

// Maxima of eight rows' magnitudes (as integers, so NaN counts as the largest) over the LPR lanes that hold a row: after the
// first two steps a lane holds two rows' values (row 4 k + lane % 4, k = 0, 1), which the other steps reduce over the lanes
// with the same lane % 4.  Returns both.
template <uint32_t LPR>
__device__ __forceinline__ void rows_max(const uint32_t* v, uint32_t* out)
{
    const uint32_t lane = threadIdx.x & 63u;
    uint32_t a[4];
#pragma unroll
    for (int k = 0; k < 4; k++) {
        const uint32_t keep = lane & 1u ? v[2 * k + 1] : v[2 * k], give = lane & 1u ? v[2 * k] : v[2 * k + 1];
        a[k] = max(keep, (uint32_t)dpp_i<DPP_XOR1>((int)give));
    }
#pragma unroll
    for (int k = 0; k < 2; k++) {
        const uint32_t keep = lane & 2u ? a[2 * k + 1] : a[2 * k], give = lane & 2u ? a[2 * k] : a[2 * k + 1];
        uint32_t b = max(keep, (uint32_t)dpp_i<DPP_XOR2>((int)give));
        b = max(b, (uint32_t)dpp_i<0x124>((int)b)); // row_ror 4
        b = max(b, (uint32_t)dpp_i<0x128>((int)b)); // row_ror 8
        if (LPR > 16) b = max(b, (uint32_t)__shfl_xor((int)b, 16));
        if (LPR > 32) b = max(b, (uint32_t)__shfl_xor((int)b, 32));
        out[k] = b;
    }
}
// value of lane q of the own group of four lanes
template <int Q>
__device__ __forceinline__ float quad_lane(float v)
{
    return dpp_f<Q * 0x55>(v);
}
__device__ __forceinline__ void quad_spread(const float* two, float* eight) // [row 4 k + q] from lane q of the quad
{
#pragma unroll
    for (int k = 0; k < 2; k++) {
        eight[4 * k] = quad_lane<0>(two[k]);
        eight[4 * k + 1] = quad_lane<1>(two[k]);
        eight[4 * k + 2] = quad_lane<2>(two[k]);
        eight[4 * k + 3] = quad_lane<3>(two[k]);
    }
}

template <int DH, bool F32, bool TREE>
__global__ __launch_bounds__((64 * TileGeom<DH, F32>::WAVES), 2) void attn_tile_kernel(RunsCall a)
{
    using T = TileGeom<DH, F32>;
    constexpr uint32_t KS = DH / 32, NT = DH / 16, LPR = T::LPR, NB = T::NB, BN = T::BN, E = F32 ? 4 : 8, NC = LPR / 16, RT = T::RT, WR = 16 * RT;
    QK_DYN_LDS(uint8_t, s_dyn);
    __shared__ int32_t s_up[TREE ? QKK_TREE_MAX : 1];
    __shared__ uint32_t s_kin[TREE ? TL_M : 1][QKK_TREE_MAX / 32];
    const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), m = lane & 15u, g = lane >> 4;

    // workgroup -> KV head (neighbours differ in it: they run on different dies, which then keep one head's cache in their L2), run,
    // block of rows, range of keys
    const uint32_t kv = blockIdx.x % a.c.n_kv;
    uint32_t run, f0, split = 0, chunk = a.c.cap;
    Run u;
    if (a.n_split == 1) {
        // the last (longest) blocks first.  A run's blocks begin at its own first row; run i's first block has the number
        // floor(start G / 128) + i, which leaves every run room for its last, part-filled one.
        const uint32_t blk = gridDim.x / a.c.n_kv - 1 - blockIdx.x / a.c.n_kv;
        auto first_of = [&](uint32_t i) { return (int64_t)((uint64_t)max(a.R.start[i], 0) * a.G / TL_M) + i; };
        run = wave_last_le(a.R.n_run, blk, first_of);
        if (run >= a.R.n_run) return; // the whole workgroup
        u = run_at(a.c, a.R, run);
        f0 = (blk - (uint32_t)first_of(run)) * TL_M;
    } else {
        const Item it = item_of(a, blockIdx.x / a.c.n_kv, TL_M, !TREE);
        if (!it.ok) return; // the whole workgroup
        u = it.u;
        run = it.run;
        f0 = it.block * TL_M;
        split = it.split;
        chunk = it.chunk;
    }
    const uint32_t rows_all = u.n * a.G;
    if (!u.ok || f0 >= rows_all) return; // the whole workgroup
    const uint32_t nr = min(TL_M, rows_all - f0);
    const uint32_t last = (f0 + nr - 1) / a.G; // the block's last position in the run
    const uint32_t end = min(u.pos + last + 1, a.c.cap), k_begin = split * chunk;
    if (k_begin >= end) return; // the whole workgroup
    const uint32_t k_end = min(end, k_begin + chunk), n_tile = (k_end - k_begin + BN - 1) / BN;
    const uint32_t node0 = f0 / a.G;
    if (TREE && k_end > u.pos) tree_bits(tree_parent(a.parent, u), node0, last - node0 + 1, s_up, s_kin);

    const uint32_t wr = WR * wave; // the wave's first row in the block
    const bool has = wr < nr;      // uniform: a wave without rows only stages tiles
    // this lane's rows' positions behind node0 (below 128), 255 for a row that is not there: a byte for each block, so one register
    auto nodes_of = [&](uint32_t col) {
        uint32_t n = 0;
#pragma unroll
        for (uint32_t rt = 0; rt < RT; rt++) n |= (wr + 16 * rt + col < nr ? (f0 + wr + 16 * rt + col) / a.G - node0 : 0xFFu) << (8 * rt);
        return n;
    };
    uint32_t nodes = nodes_of(m);
    const uint32_t first_node = (f0 + min(wr, nr - 1)) / a.G, last_node = (f0 + min(wr + WR, nr) - 1) / a.G;

    // Which of the four keys from `key` on this lane's row of block rt sees, pages aside.
    auto sees = [&](uint32_t rt, uint32_t key) {
        const uint32_t node = nodes >> (8 * rt) & 0xFFu;
        const uint32_t stop = node == 0xFFu ? 0u : TREE ? k_end : min(k_end, u.pos + node0 + node + 1);
        uint32_t four = (1u << (stop > key ? min(stop - key, 4u) : 0u)) - 1u;
        if (TREE && k_end > u.pos) {
            uint32_t at = node & (TL_M - 1);
            asm("" : QK_REG(at), QK_REG(key)); // the row's address is not kept through the loop: registers
            four &= tree_four(s_kin[at], (int32_t)(key - u.pos));
        }
        return four;
    };
    bool odd_values = false; // uniform: some value of this range is not finite

    // Staging: the first half of the waves takes V, the second K, eight 16-byte pieces per thread.
    //   V  (piece, lane group sg of the second product, step st of 32 keys): keys 4 sg + i and 16 + 4 sg + i of the step, i < 4
    //   K  rows RL (KR kw + j) + kr of the tile, j < KR, pieces kq + QL i, i < PI (kw: the wave among those that stage K)
    const bool is_v = wave < T::WAVES / 2; // uniform
    const uint32_t tid = threadIdx.x % (32 * T::WAVES), piece = tid % LPR, sg = tid / LPR % 4, st = tid / LPR / 4;
    const uint32_t kr = lane % T::RL, kq = lane / T::RL, k_row0 = (wave % (T::WAVES / 2)) * T::RL * T::KR + kr;
    // A thread's pieces lie in two groups of four, each at one distance from the next -- V rows 4 sg .. 4 sg + 3 of a block of 16 keys, which
    // are neighbours in their page, or four pieces of one K row -- so a tile takes two full addresses (64-bit products are
    // slow), not eight.  Keys behind the range repeat its last one (masked below).
    u32x4 reg[8];
    const uint8_t* vbase = (const uint8_t*)a.c.v;
    const uint8_t* kbase = (const uint8_t*)a.c.k;
    const uint32_t stride = is_v ? DH * T::ES : 16 * T::QL; // uniform
    auto first_key = [&](uint32_t tile, uint32_t b) {
        uint32_t key = 32 * st + 16 * b + 4 * sg;
        if (!is_v) key = k_row0 + (T::KR == 1 ? 0 : T::RL * b);
        return min(k_begin + BN * tile + key, k_end - 1);
    };
    uint32_t pg[2]; // the groups' page ids, requested a tile ahead of the rows and not looked at before
    auto pages = [&](uint32_t tile) {
#pragma unroll
        for (uint32_t b = 0; b < 2; b++) pg[b] = (uint32_t)*kv_page_at(a.c, a.R.seq + run, u.seq, first_key(tile, b));
    };
    uint32_t bad_pages = 0; // of the tile in registers: bit b, this thread's group b has no page
    auto fetch = [&](uint32_t tile) {
        bad_pages = (pg[0] >= a.c.n_page ? 1u : 0u) | (pg[1] >= a.c.n_page ? 2u : 0u);
#pragma unroll
        for (uint32_t b = 0; b < 2; b++) {
            const uint32_t key = first_key(tile, b), p = pg[b] >= a.c.n_page ? 0u : pg[b]; // without a page: page 0's row, masked
            const size_t at = kv_row(a.c, p, kv, key, DH) * T::ES + 16 * (is_v ? piece : kq + (T::KR == 1 ? 4 * T::QL * b : 0));
            const uint8_t* row = (is_v ? vbase : kbase) + at;
            const uint32_t lim = is_v ? k_end - 1 - key : 3u; // V: rows behind the first that are inside the range
#pragma unroll
            for (uint32_t i = 0; i < 4; i++) reg[4 * b + i] = *(const u32x4*)(row + min(i, lim) * stride);
        }
    };
    // whether every row of the block sees every key of a tile (pages aside)
    auto tile_whole = [&](uint32_t tile) {
        const uint32_t e = k_begin + BN * (tile + 1);
        return e <= k_end && e <= u.pos + (TREE ? 0u : node0 + 1);
    };
    auto stage = [&](uint32_t tile, uint8_t* buf) {
        uint8_t* s_k = buf;
        uint8_t* s_v = buf + T::NH * T::KB;
        float* s_e = (float*)(buf + T::NH * (T::KB + T::VB));
        uint32_t* s_flag = (uint32_t*)(buf + T::NH * (T::KB + T::VB) + T::EXP);
        uint32_t t = threadIdx.x, any = tile;
        asm("" : QK_REG(t), QK_REG(any)); // places of exponents are computed per tile, not kept through the loop: registers
        if (!is_v) {
#pragma unroll
            for (uint32_t j = 0; j < T::KR; j++) {
                const uint32_t row = k_row0 + T::RL * j;
                uint8_t* at = s_k + (row / 16 * KS * 64 + row % 16) * 16;
                if constexpr (F32) {
                    float mx = 0.f; // NaN is passed over here and stays one in its key's scores
#pragma unroll
                    for (uint32_t i = 0; i < T::PI; i++)
#pragma unroll
                        for (uint32_t e = 0; e < 4; e++) mx = fmaxf(mx, fabsf(u2f(reg[T::PI * j + i][e])));
                    mx = fmaxf(mx, dpp_f<0x128>(mx)); // the row's eight lanes: lane % 8 is the row (row_ror 8)
                    mx = xor_lanes_max(mx);
                    const int ex = top_exponent(mx);
                    const float scale = pow2i(-ex);
                    if (kq == 0) s_e[(wave % (T::WAVES / 2)) * T::RL * T::KR + t % T::RL + T::RL * j] = u2f((uint32_t)ex); // row
                    at += kq / 2 * 256 + kq % 2 * 8;
#pragma unroll
                    for (uint32_t i = 0; i < T::PI; i++) { // pieces kq + 8 i: step i of 32 dims
                        const u32x4 x = reg[T::PI * j + i];
                        uint32_t h0, h1, l0, l1;
                        split_pair(u2f(x[0]), u2f(x[1]), scale, true, h0, l0);
                        split_pair(u2f(x[2]), u2f(x[3]), scale, true, h1, l1);
                        *(lds_u32x2*)(at + 1024 * i) = u32x2{h0, h1};
                        *(lds_u32x2*)(at + 1024 * i + T::KB) = u32x2{l0, l1};
                    }
                } else {
#pragma unroll
                    for (uint32_t i = 0; i < T::PI; i++) *(lds_u32x4*)(at + kq * 256 + 1024 * i) = reg[T::PI * j + i];
                }
            }
            return;
        }
        float sc[8];      // what the value rows are multiplied by (fp32)
        uint32_t odd = 0; // bit i: value row i of this thread's eight holds something that is not finite (taken out here, added later)
        if constexpr (F32) {
            uint32_t mx[8], top[2];
#pragma unroll
            for (uint32_t i = 0; i < 8; i++)
                mx[i] = max(max(reg[i][0] & 0x7FFFFFFFu, reg[i][1] & 0x7FFFFFFFu), max(reg[i][2] & 0x7FFFFFFFu, reg[i][3] & 0x7FFFFFFFu));
            rows_max<LPR>(mx, top);
            if (__builtin_amdgcn_ballot_w64(max(top[0], top[1]) >= 0x7F800000u)) { // rare: uniform
#pragma unroll
                for (uint32_t i = 0; i < 8; i++) {
                    mx[i] = 0;
                    bool bad = false;
#pragma unroll
                    for (uint32_t j = 0; j < 4; j++) {
                        const uint32_t x = reg[i][j];
                        const bool nf = (x & 0x7F800000u) == 0x7F800000u;
                        bad = bad || nf;
                        reg[i][j] = nf ? 0u : x;
                        mx[i] = max(mx[i], nf ? 0u : x & 0x7FFFFFFFu);
                    }
                    const uint64_t who = __builtin_amdgcn_ballot_w64(bad) >> (lane - piece % 64);
                    odd |= ((LPR == 64 ? who : who & ((1ull << (LPR % 64)) - 1)) ? 1u : 0u) << i;
                }
                rows_max<LPR>(mx, top);
            }
            float sc2[2];
#pragma unroll
            for (uint32_t k = 0; k < 2; k++) {
                const int e = top_exponent(u2f(top[k]));
                sc2[k] = pow2i(-e);
                if (piece < 4) s_e[BN + 32 * st + 4 * (t / LPR % 4) + 16 * k + piece] = u2f((uint32_t)e); // row 4 k + piece of the eight
            }
            quad_spread(sc2, sc);
        } else if (!tile_whole(tile) || __builtin_amdgcn_ballot_w64(bad_pages != 0)) { // uniform
#pragma unroll
            for (uint32_t i = 0; i < 8; i++) {
                bool bad = false;
#pragma unroll
                for (uint32_t j = 0; j < 4; j++) {
                    const uint32_t x = reg[i][j];
                    const bool b0 = (x & 0x7C00u) == 0x7C00u, b1 = (x & 0x7C000000u) == 0x7C000000u;
                    bad = bad || b0 || b1;
                    reg[i][j] = (b0 ? 0u : x & 0xFFFFu) | (b1 ? 0u : x & 0xFFFF0000u);
                }
                const uint64_t who = __builtin_amdgcn_ballot_w64(bad) >> (lane - piece);
                odd |= ((who & ((1ull << LPR) - 1)) ? 1u : 0u) << i;
            }
        }
        // dim E piece + e is row piece % 16 of block NC e + piece / 16
        const float one = pinned_one();
        uint8_t* at = s_v + (((piece / 16) * NB + st) * 64 + 16 * sg + piece % 16) * 16;
#pragma unroll
        for (uint32_t e = 0; e < E; e++, at += NC * NB * 1024) {
            u32x4 w;
            if constexpr (F32) {
                u32x4 lo;
#pragma unroll
                for (uint32_t i = 0; i < 4; i++) {
                    // two keys, each with its own factor: scaled first
                    uint32_t h, l;
                    split_pair(u2f(reg[2 * i][e]) * sc[2 * i], u2f(reg[2 * i + 1][e]) * sc[2 * i + 1], one, false, h, l);
                    w[i] = h;
                    lo[i] = l;
                }
                *(lds_u32x4*)(at + T::VB) = lo;
            } else {
#pragma unroll
                for (uint32_t i = 0; i < 4; i++) // half e of keys 2 i, 2 i + 1
                    w[i] = __builtin_amdgcn_perm(reg[2 * i + 1][e / 2], reg[2 * i][e / 2], e % 2 ? 0x07060302u : 0x05040100u);
            }
            *(lds_u32x4*)at = w;
        }
        if (piece == 0) s_flag[sg * NB + st] = odd | bad_pages << 8;
    };
    // Q: this wave's rows f0 + WR wave + 16 rt + m, dims 32 ks + 8 g .. + 7, requested in front of the first tile's rows and prepared, divided
    // by the row's power of two, while those arrive
    pages(0);
    // (and multiplied by log2 e / sqrt dh: scores are in the log2 domain)
    half8 qh[RT][KS], ql[RT][KS];
    int xq[RT]; // exponents in one register: the query row's, and above it vx (fp32: o is held divided by 2^(vx - TL_UP))
    auto q_exp = [&](uint32_t rt) { return (int)(int16_t)xq[rt]; };
    auto v_exp = [&](uint32_t rt) { return xq[rt] >> 16; };
    auto set_v_exp = [&](uint32_t rt, int v) { xq[rt] = (v << 16) | (xq[rt] & 0xFFFF); };
    const float qs = AR_LOG2E / sqrtf((float)DH);
    f32x4 qx[RT][KS][2];
#pragma unroll
    for (uint32_t rt = 0; rt < RT; rt++) {
        const uint32_t ff = f0 + min(wr + 16 * rt + m, nr - 1);
        const f32x4* row = (const f32x4*)(a.q + ((size_t)(u.r0 + ff / a.G) * a.hQ + kv * a.G + ff % a.G) * DH);
#pragma unroll
        for (uint32_t ks = 0; ks < KS; ks++)
#pragma unroll
            for (uint32_t i = 0; i < 2; i++) qx[rt][ks][i] = row[8 * ks + 2 * g + i];
    }
    __builtin_amdgcn_sched_barrier(0);
    fetch(0);
    if (n_tile > 1) pages(1);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (uint32_t rt = 0; rt < RT; rt++) {
        float mx = 0.f;
#pragma unroll
        for (uint32_t ks = 0; ks < KS; ks++)
#pragma unroll
            for (uint32_t j = 0; j < 8; j++) mx = fmaxf(mx, fabsf(qx[rt][ks][j / 4][j % 4]));
        xq[rt] = top_exponent(xor_lanes_max(mx) * qs);
        const float scale = pow2i(-xq[rt]);
#pragma unroll
        for (uint32_t ks = 0; ks < KS; ks++) {
            float y[8];
#pragma unroll
            for (uint32_t j = 0; j < 8; j++) y[j] = qx[rt][ks][j / 4][j % 4] * qs * scale;
            const Half2 sp = split2(y);
            qh[rt][ks] = sp.hi;
            ql[rt][ks] = sp.lo;
        }
    }
    float4v o[RT][NT];
    float m_run[RT], l_run[RT];
#pragma unroll
    for (uint32_t rt = 0; rt < RT; rt++) {
        m_run[rt] = AR_FLOOR;
        l_run[rt] = 0.f;
#pragma unroll
        for (uint32_t t = 0; t < NT; t++) o[rt][t] = float4v{0.f, 0.f, 0.f, 0.f};
    }

    // Scores, softmax and values of a tile's 32 keys from 32 sp for this wave.  whole: every row sees every key.
    auto work = [&](uint32_t tile, const uint8_t* buf, bool whole, uint32_t sp) {
        const uint8_t* s_k = buf;
        const uint8_t* s_v = buf + T::NH * T::KB;
        const float* s_e = (const float*)(buf + T::NH * (T::KB + T::VB));
        const uint32_t* s_flag = (const uint32_t*)(buf + T::NH * (T::KB + T::VB) + T::EXP);
        const uint32_t key0 = k_begin + BN * tile + 32 * sp;
        float4v s[RT][2];
#pragma unroll
        for (uint32_t b = 0; b < 2; b++)
#pragma unroll
            for (uint32_t rt = 0; rt < RT; rt++) s[rt][b] = float4v{0.f, 0.f, 0.f, 0.f};
        half8 fh[T::AHEAD], fl[T::AHEAD];
        auto read = [&](const uint8_t* at, uint32_t copy, uint32_t slot) {
            fh[slot] = __builtin_bit_cast(half8, u32x4(*(const lds_u32x4*)at));
            if constexpr (F32) fl[slot] = __builtin_bit_cast(half8, u32x4(*(const lds_u32x4*)(at + copy)));
        };
        const uint8_t* kf_at = s_k + (2 * sp * KS * 64 + lane) * 16;
#pragma unroll
        for (uint32_t i = 0; i < T::AHEAD; i++) read(kf_at + 1024 * i, T::KB, i);
        if (T::PIN) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (uint32_t i = 0; i < 2 * KS; i++) {
            const uint32_t b = i / KS, ks = i % KS, slot = i % T::AHEAD;
            if constexpr (F32) {
#pragma unroll
                for (uint32_t rt = 0; rt < RT; rt++) s[rt][b] = mfma16x32(fl[slot], qh[rt][ks], s[rt][b]);
            }
#pragma unroll
            for (uint32_t rt = 0; rt < RT; rt++) s[rt][b] = mfma16x32(fh[slot], ql[rt][ks], s[rt][b]);
#pragma unroll
            for (uint32_t rt = 0; rt < RT; rt++) s[rt][b] = mfma16x32(fh[slot], qh[rt][ks], s[rt][b]);
            if (i + T::AHEAD < 2 * KS) read(kf_at + 1024 * (i + T::AHEAD), T::KB, slot);
            if (T::PIN) __builtin_amdgcn_sched_barrier(0);
        }
        const uint8_t* vf_at = s_v + (sp * 64 + lane) * 16;
#pragma unroll
        for (uint32_t i = 0; i < T::AHEAD; i++) read(vf_at + 1024 * NB * i, T::VB, i); // the first values arrive during the softmax
        if (T::PIN) __builtin_amdgcn_sched_barrier(0);
        // scores in the log2 domain: this lane's row wr + 16 rt + m, keys 16 b + 4 g + r
#pragma unroll
        for (uint32_t b = 0; b < 2; b++) {
            i32x4 ke;
            if constexpr (F32) ke = *(const lds_i32x4*)(s_e + 32 * sp + 16 * b + 4 * g);
#pragma unroll
            for (uint32_t r = 0; r < 4; r++) {
#pragma unroll
                for (uint32_t rt = 0; rt < RT; rt++) {
                    s[rt][b][r] = __builtin_ldexpf(s[rt][b][r], F32 ? ke[r] + q_exp(rt) : q_exp(rt));
                }
            }
        }
        if (!whole) { // uniform
#pragma unroll
            for (uint32_t rt = 0; rt < RT; rt++) {
#pragma unroll
                for (uint32_t b = 0; b < 2; b++) { // four neighbouring keys at a time
                    const uint32_t key = key0 + 16 * b + 4 * g;
                    const uint32_t bad = s_flag[sp] >> (8 + b) & 1u; // the first lane group's word of this step: its blocks without a page
                    const uint32_t four = bad ? 0u : sees(rt, key);
#pragma unroll
                    for (uint32_t r = 0; r < 4; r++) s[rt][b][r] = (four >> r) & 1u ? s[rt][b][r] : -INFINITY;
                }
            }
        }
        float mx[RT];
        bool over = false;
#pragma unroll
        for (uint32_t rt = 0; rt < RT; rt++) {
            mx[rt] = AR_FLOOR;
#pragma unroll
            for (uint32_t i = 0; i < 8; i++) mx[rt] = fmaxf(mx[rt], s[rt][i / 4][i % 4]);
            over = over || mx[rt] > m_run[rt] + TL_SLACK;
        }
        if (__builtin_amdgcn_ballot_w64(over)) { // uniform: now and then
#pragma unroll
            for (uint32_t rt = 0; rt < RT; rt++) {
                const float top = xor_lanes_max(mx[rt]), m_new = top > m_run[rt] + TL_SLACK ? top : m_run[rt];
                const float step = m_new - m_run[rt];
                float corr = __builtin_amdgcn_exp2f(-step);
                m_run[rt] = m_new;
                l_run[rt] *= corr;
                if constexpr (F32) { // the largest P 2^e need not have moved with the maximum
                    const int was = v_exp(rt), vx = step < 1e30f ? max(was - (int)fminf(step, (float)TL_VX), -TL_VX) : was; // else: the first time
                    set_v_exp(rt, vx);
                    corr = __builtin_amdgcn_exp2f((float)(was - vx) - step);
                }
#pragma unroll
                for (uint32_t n = 0; n < NT; n++) o[rt][n] *= corr;
            }
        }
        half8 ph[RT], pl[RT];
#pragma unroll
        for (uint32_t rt = 0; rt < RT; rt++) {
            float sum = 0.f, p[8];
            if constexpr (F32) {
                float big = 0.f;
                const int up = (int)TL_UP - v_exp(rt);
#pragma unroll
                for (uint32_t b = 0; b < 2; b++) {
                    const i32x4 ve = *(const lds_i32x4*)(s_e + BN + 32 * sp + 16 * b + 4 * g);
#pragma unroll
                    for (uint32_t r = 0; r < 4; r++) {
                        const float x = __builtin_amdgcn_exp2f(s[rt][b][r] - m_run[rt]);
                        sum += x;
                        p[4 * b + r] = __builtin_ldexpf(x, ve[r] + up);
                        big = fmaxf(big, p[4 * b + r]);
                    }
                }
                if (__builtin_amdgcn_ballot_w64(big > 1.01f * TL_TOP)) { // uniform: now and then
                    float top = -(float)TL_VX; // the largest P 2^e, as an exponent
#pragma unroll
                    for (uint32_t i = 0; i < 8; i++) {
                        const int e = ((const lds_i32*)s_e)[BN + 32 * sp + 16 * (i / 4) + 4 * g + i % 4];
                        top = fmaxf(top, s[rt][i / 4][i % 4] - m_run[rt] + (float)e);
                    }
                    top = fminf(xor_lanes_max(top), (float)TL_VX);
                    const int was = v_exp(rt), vx = top > (float)was + TL_SLACK ? (int)__builtin_ceilf(top) : was;
                    set_v_exp(rt, vx);
#pragma unroll
                    for (uint32_t n = 0; n < NT; n++)
#pragma unroll
                        for (uint32_t r = 0; r < 4; r++) o[rt][n][r] = __builtin_ldexpf(o[rt][n][r], was - vx);
#pragma unroll
                    for (uint32_t i = 0; i < 8; i++) {
                        const int e = ((const lds_i32*)s_e)[BN + 32 * sp + 16 * (i / 4) + 4 * g + i % 4];
                        p[i] = __builtin_ldexpf(__builtin_amdgcn_exp2f(s[rt][i / 4][i % 4] - m_run[rt]), e + (int)TL_UP - vx);
                    }
                }
            } else {
                const float top = m_run[rt] - TL_UP;
#pragma unroll
                for (uint32_t i = 0; i < 8; i++) {
                    p[i] = __builtin_amdgcn_exp2f(s[rt][i / 4][i % 4] - top);
                    sum += p[i];
                }
            }
            l_run[rt] += sum; // of this lane's keys; the lane groups are added at the end
            const Half2 p2 = split2(p);
            ph[rt] = p2.hi;
            pl[rt] = p2.lo;
        }
        if (T::PIN) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (uint32_t n = 0; n < NT; n++) {
            const uint32_t slot = n % T::AHEAD;
            if constexpr (F32) {
#pragma unroll
                for (uint32_t rt = 0; rt < RT; rt++) o[rt][n] = mfma16x32(fl[slot], ph[rt], o[rt][n]);
            }
#pragma unroll
            for (uint32_t rt = 0; rt < RT; rt++) o[rt][n] = mfma16x32(fh[slot], pl[rt], o[rt][n]);
#pragma unroll
            for (uint32_t rt = 0; rt < RT; rt++) o[rt][n] = mfma16x32(fh[slot], ph[rt], o[rt][n]);
            if (n + T::AHEAD < NT) read(vf_at + 1024 * NB * (n + T::AHEAD), T::VB, slot);
            if (T::PIN) __builtin_amdgcn_sched_barrier(0);
        }
    };

    stage(0, s_dyn);
    if (n_tile > 1) fetch(1);
    if (n_tile > 2) pages(2);
    __syncthreads();
    if constexpr (F32) { // vx begins at the smallest exponent of the first tile's value rows: no row's weights are made small for the sake of one it does not see
        const float* s_e = (const float*)(s_dyn + T::NH * (T::KB + T::VB));
        const int least = -(int)wave_max(-(float)((const lds_i32*)s_e)[BN + lane % BN]);
#pragma unroll
        for (uint32_t rt = 0; rt < RT; rt++) set_v_exp(rt, least);
    }
    for (uint32_t tile = 0; tile < n_tile; tile++) {
        const uint8_t* buf = s_dyn + (tile & 1u) * T::BUF;
        const uint32_t* s_flag = (const uint32_t*)(buf + T::NH * (T::KB + T::VB) + T::EXP);
        const uint32_t key0 = k_begin + BN * tile;
        // the wave's rows see a prefix up to pos + node: nothing of this tile, all of it, or part
        const uint32_t flag = lane < 4 * NB ? s_flag[min(lane, 4 * NB - 1)] : 0u;
        const bool flagged = __builtin_amdgcn_ballot_w64(flag != 0) != 0;
        if (flagged) odd_values = odd_values || __builtin_amdgcn_ballot_w64((flag & 0xFFu) != 0) != 0;
        const bool whole = !flagged && key0 + BN <= k_end && key0 + BN <= u.pos + (TREE ? 0u : first_node + 1); // uniform
        if (has && key0 <= u.pos + last_node) { // uniform
#pragma unroll
            for (uint32_t sp = 0; sp < NB; sp++) work(tile, buf, whole, sp);
        }
        if (tile + 1 < n_tile) {
            stage(tile + 1, s_dyn + ((tile + 1) & 1u) * T::BUF);
            if (tile + 2 < n_tile) fetch(tile + 2);
            if (tile + 3 < n_tile) pages(tile + 3);
        }
        __syncthreads();
    }
    if (!has) return; // the whole wave; no barrier below
    uint32_t me = threadIdx.x & 15u;
    asm("" : QK_REG(me)); // the rows' places are computed anew from here on, not kept through the loop: registers
    nodes = nodes_of(me);
    if (odd_values) { // rare: values that are not finite were taken out of the products; they reach the rows that see them here
        for (uint32_t key0 = k_begin; key0 < k_end; key0 += 4) { // from a multiple of four: one page
            const uint32_t page = kv_page(a.c, u.seq, key0);
            if (page == KV_NO_PAGE) continue; // uniform
            for (uint32_t k = 0; k < 4 && key0 + k < k_end; k++) {
                const uint8_t* row = vbase + kv_row(a.c, page, kv, key0 + k, DH) * T::ES;
#pragma unroll
                for (uint32_t n = 0; n < NT; n++) {
                    __builtin_amdgcn_sched_barrier(0); // registers: not all loads at once
#pragma unroll
                    for (uint32_t r = 0; r < 4; r++) {
                        const uint32_t d = E * (16 * (n % NC) + 4 * g + r) + n / NC;
                        const float v = F32 ? ((const float*)row)[d] : (float)((const _Float16*)row)[d];
#pragma unroll
                        for (uint32_t rt = 0; rt < RT; rt++)
                            if (!(fabsf(v) < INFINITY) && ((sees(rt, key0) >> k) & 1u)) o[rt][n][r] += v;
                    }
                }
            }
        }
    }
#pragma unroll
    for (uint32_t rt = 0; rt < RT; rt++) {
        const float l = xor_lanes_sum(l_run[rt]);
        const uint32_t f = wr + 16 * rt + me;
        if (f >= nr) continue;
        const size_t rh = (size_t)(u.r0 + (f0 + f) / a.G) * a.hQ + kv * a.G + (f0 + f) % a.G;
        const float inv = l == 0.f ? 0.f : 1.f / l;
        float* out = a.n_split > 1 ? a.acc + (rh * a.n_split + split) * DH : a.att + rh * DH;
        if (a.n_split > 1 && g == 0) {
            a.ml[2 * (rh * a.n_split + split)] = m_run[rt];
            a.ml[2 * (rh * a.n_split + split) + 1] = l;
        }
#pragma unroll
        for (uint32_t c = 0; c < NC; c++)
#pragma unroll
            for (uint32_t r = 0; r < 4; r++)
#pragma unroll
                for (uint32_t e = 0; e < E; e += 4) {
                    const uint32_t d = E * (16 * c + 4 * g + r) + e;
                    f32x4 x;
#pragma unroll
                    for (uint32_t i = 0; i < 4; i++) {
                        x[i] = o[rt][(e + i) * NC + c][r] * inv;
                        if constexpr (F32) x[i] = __builtin_ldexpf(x[i], v_exp(rt) - (int)TL_UP);
                    }
                    if (a.n_split == 1 && a.qfull) {
                        const f32x4 gt = *(const f32x4*)(a.qfull + rh * 2 * DH + DH + d);
#pragma unroll
                        for (uint32_t i = 0; i < 4; i++) x[i] *= 1.f / (1.f + expf(-gt[i]));
                    }
                    *(f32x4*)(out + d) = x;
                }
    }
}

template <int DH, bool F32, bool TREE>
static void launch_tile(const RunsCall& a, hipStream_t st)
{
    constexpr uint32_t lds = 2 * TileGeom<DH, F32>::BUF;
    static_assert(lds <= 160 * 1024, "LDS");
    static std::atomic<uint64_t> asked{0};
    allow_lds((const void*)attn_tile_kernel<DH, F32, TREE>, lds, asked);
    hipLaunchKernelGGL((attn_tile_kernel<DH, F32, TREE>), dim3(items_of(tile_blocks(a.R.n_rows, a.R.n_run, a.G), a.slots, a.n_split) * a.c.n_kv), dim3(64 * TileGeom<DH, F32>::WAVES), lds, st, a);
}

void launch_attn_tile(const RunsCall& a, int type, uint32_t dh, bool tree, hipStream_t st)
{
    if (dh == 256) {
        if (type == QKK_F32) tree ? launch_tile<256, true, true>(a, st) : launch_tile<256, true, false>(a, st);
        else tree ? launch_tile<256, false, true>(a, st) : launch_tile<256, false, false>(a, st);
    } else {
        if (type == QKK_F32) tree ? launch_tile<128, true, true>(a, st) : launch_tile<128, true, false>(a, st);
        else tree ? launch_tile<128, false, true>(a, st) : launch_tile<128, false, false>(a, st);
    }
}

} // namespace qk
