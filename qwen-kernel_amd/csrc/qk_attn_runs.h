// qk_attn_runs.h -- what the kernels of qkk_attn_packed / qkk_attn_tree share (qk_attn_runs.hip, qk_attn_few.hip,
// qk_attn_tile.hip).
//
// Both kernels compute, per KV head, the TRANSPOSED products on the matrix cores (v_mfma_f32_16x16x32, A 16 x 32, B
// 32 x 16, D 16 x 16):
//   S^T[key][row] = K[key][:] . Q[row][:]       A = 16 keys, B = 16 query rows
//   O^T[dim][row] = V^T[dim][:] . P^T[:][row]   A = 16 dims, B = 16 query rows
// so that a lane's outputs all belong to ONE query row (lane % 16): the running maximum, the sum and the rescaling are
// lane-local up to one exchange between the four lane groups, and the weights P leave the first product in the
// registers in which the second one wants them.  With g = lane / 16 a lane holds, after two S^T blocks of 16 keys, the
// keys 4g .. 4g+3 and 16+4g .. 16+4g+3 of a step of 32; the second product contracts its 32 keys in exactly
// that order (contraction order is free as long as A and B agree).
//
// The query rows of a run that share a KV head (positions x heads of the group) are numbered f = position * G + head, so
// any group size fills the 16 columns.
//
// Two halves hold an fp32 value to 2^-22 where the lo half is normal (from 2^-2 up; below it to 2^-25 absolute), three bf16 pieces
// hold it exactly in fp32's own range: products of split operands on the matrix cores (the kernels say which they use and why).
#pragma once
#include "qk_kv.h"
#include "qk_mfma.h"

namespace qk {

constexpr float AR_FLOOR = -3.0e38f;
constexpr float AR_LOG2E = 1.44269504088896341f;

// One call.  With n_split 1 a workgroup takes all keys of its rows and writes att.  Else the keys are cut into ranges, each range's
// result goes to the workspace as if its keys were all there are, with the maximum of its scores and the sum of its weights, and
// attn_join_kernel adds the results up by their share of the whole sum.  How long a range is, is decided on the
// device from the lengths (item_of), a multiple of `grain` and not below `chunk`, of which n_split cover the cache.
struct RunsCall {
    KvView c;
    RunsView R;
    const int32_t* parent;
    const float *q, *qfull;
    float *att, *acc, *ml; // acc [row][head][n_split][dh], ml [row][head][n_split][2] (maximum in the log2 domain, sum)
    uint32_t* chunk_used;  // one word of the workspace
    uint32_t hQ, G, n_split, chunk, grain, slots; // slots: items per KV head that fill the device
};

// The piece of work with number `item` of its KV head: a run, a block of its rows, a range of keys.
struct Item {
    Run u;
    uint32_t run, block, split, chunk;
    bool ok;
};
// The length of a run's ranges, all but the last: as many as `chunk` makes, of one length.
__device__ __forceinline__ uint32_t run_chunk(uint32_t end, uint32_t chunk, uint32_t grain)
{
    const uint32_t splits = max((end + chunk - 1) / chunk, 1u), each = (end + splits - 1) / splits;
    return max((each + grain - 1) / grain, 1u) * grain;
}
// Sequences of a batch differ in length by orders of magnitude, and the lengths live on the device.  Every wave looks all of them
// over (64 runs per round trip, about 2 us), takes the range that cuts the whole of them -- blocks of `rows` rows times keys --
// into as many items as there are places on the device, and finds its own item by a prefix sum; items without work come last
// and end at once.  A run's own ranges are then made equal.  Every workgroup comes to the same result; the join finds the common
// range in the workspace.  (One row for each of sixteen sequences of 1 .. 4096 keys: 25 us, 37 with ranges fixed by the host,
// where three workgroups of four had no work and the others waited behind them.)
//   Packed rows see half of their own run on average: their work is counted so, and ranges that a block of rows does not reach
// end at once.  A block's last range is half empty on average; where that guess makes more items than places, the range is taken
// that cannot: a second round on the device costs more than shorter ranges give.  (Counting a whole range lost per block
// left a tenth of the device idle: trees of 24 nodes on sixteen slots of 1000 .. 4100 fp32 rows took 1.08 of the time so reached, now
// 125 us; two trees on 33,000 and 65,000 half rows 1.03, now 204.)
__device__ __forceinline__ Item item_of(const RunsCall& a, uint32_t item, uint32_t rows, bool causal)
{
    const uint32_t lane = threadIdx.x & 63u;
    auto look = [&](uint32_t i, uint32_t& nb, uint32_t& end, uint32_t& seen) {
        nb = end = seen = 0;
        if (i >= a.R.n_run) return;
        const Run u = run_at(a.c, a.R, i);
        if (!u.ok || !u.n) return;
        nb = (u.n * a.G + rows - 1) / rows;
        end = min(u.pos + u.n, a.c.cap);
        seen = causal ? min(u.pos + (u.n + 1) / 2, end) : end; // at least half of end
    };
    uint32_t nb0, end0, seen0, blocks = 0; // the first 64 runs stay in registers
    uint64_t work = 0;              // in pieces of 64 keys
    look(lane, nb0, end0, seen0);
    for (uint32_t i = lane; i < a.R.n_run; i += 64) {
        uint32_t nb = nb0, end = end0, seen = seen0;
        if (i != lane) look(i, nb, end, seen);
        blocks += nb;
        work += (uint64_t)nb * ((seen + 63) / 64);
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        blocks += __shfl_xor(blocks, d);
        work += __shfl_xor(work, d);
    }
    auto range_for = [&](uint32_t places) {
        const uint64_t want = ((work + places - 1) / places * 64 + a.grain - 1) / a.grain * a.grain;
        return (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)min(max(want, (uint64_t)a.chunk), (uint64_t)1 << 30));
    };
    const uint32_t least = max(a.slots / 2, 1u);
    uint32_t chunk = range_for(max(a.slots - min(blocks / 2, a.slots), least));
    if (!causal) {
        uint32_t made = 0;
        for (uint32_t i = lane; i < a.R.n_run; i += 64) {
            uint32_t nb = nb0, end = end0, seen = seen0;
            if (i != lane) look(i, nb, end, seen);
            made += nb * ((end + chunk - 1) / chunk);
        }
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) made += __shfl_xor(made, d);
        if (made > a.slots) chunk = range_for(max(a.slots - min(blocks, a.slots), least)); // uniform
    }
    Item it;
    if (blockIdx.x == 0 && threadIdx.x == 0 && a.n_split > 1) *a.chunk_used = chunk;
    it.ok = false;
    uint32_t before = 0;
    for (uint32_t i0 = 0; i0 < a.R.n_run; i0 += 64) {
        uint32_t nb = nb0, end = end0, seen = seen0;
        if (i0) look(i0 + lane, nb, end, seen);
        const uint32_t mine = nb * ((end + chunk - 1) / chunk), incl = before + wave_incl_scan_u32(mine);
        const uint64_t past = __builtin_amdgcn_ballot_w64(incl > item);
        if (past) {
            const uint32_t at = (uint32_t)__builtin_ctzll(past);
            const uint32_t first = (uint32_t)__shfl((int)(incl - mine), (int)at), last = (uint32_t)__shfl((int)end, (int)at);
            const uint32_t splits = (last + chunk - 1) / chunk;
            it.run = __builtin_amdgcn_readfirstlane(i0 + at);
            it.block = __builtin_amdgcn_readfirstlane((item - first) / splits);
            it.split = __builtin_amdgcn_readfirstlane((item - first) % splits);
            it.chunk = __builtin_amdgcn_readfirstlane(run_chunk(last, chunk, a.grain));
            it.u = run_at(a.c, a.R, it.run);
            it.ok = true;
            return it;
        }
        before = (uint32_t)__shfl((int)incl, 63);
    }
    return it;
}

__device__ __forceinline__ float xor_lanes_max(float v) // over the four lane groups: lanes with the same lane % 16
{
    v = fmaxf(v, __shfl_xor(v, 16));
    return fmaxf(v, __shfl_xor(v, 32));
}
__device__ __forceinline__ float xor_lanes_sum(float v)
{
    v += __shfl_xor(v, 16);
    return v + __shfl_xor(v, 32);
}

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ float4v mfma16x32(bf16x8 a, bf16x8 b, float4v c)
{
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

__device__ __forceinline__ uint32_t f2u(float x) { return __builtin_bit_cast(uint32_t, x); }
__device__ __forceinline__ float u2f(uint32_t x) { return __builtin_bit_cast(float, x); }

// Eight floats as three bf16 vectors whose sum they are, exactly (8 bits each, truncated): infinities and NaN become NaN.
struct Bf3 {
    bf16x8 p[3];
};
__device__ __forceinline__ Bf3 split3(const float* x)
{
    u32x4 o[3];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        float a = x[2 * i], b = x[2 * i + 1];
#pragma unroll
        for (int j = 0; j < 3; j++) {
            o[j][i] = __builtin_amdgcn_perm(f2u(b), f2u(a), 0x07060302u); // upper halves of a, b
            if (j < 2) {
                a -= u2f(f2u(a) & 0xFFFF0000u);
                b -= u2f(f2u(b) & 0xFFFF0000u);
            }
        }
    }
    Bf3 r;
#pragma unroll
    for (int j = 0; j < 3; j++) r.p[j] = __builtin_bit_cast(bf16x8, o[j]);
    return r;
}

// Eight floats as hi + lo halves, both rounded to nearest: exact to 2^-22 of x from |x| = 2^-2 up to a half's largest, below to 2^-25.  Two values
// take three instructions: one packs both hi halves, and the rest x * s - hi is formed and rounded by one mixed-precision
// multiply-add each.  The pinned register keeps the compiler from converting every value a second time on its own, the pinned
// factor 1 from turning the multiply-add into a subtraction of converted values.
struct Half2 {
    half8 hi, lo;
};
__device__ __forceinline__ uint32_t pack_half(float a, float b) { return __builtin_bit_cast(uint32_t, half2v{(_Float16)a, (_Float16)b}); }
__device__ __forceinline__ float pinned_one()
{
    float one = 1.f;
    asm("" : QK_REG(one));
    return one;
}
__device__ __forceinline__ void split_pair(float a, float b, float s, bool scaled, uint32_t& hi, uint32_t& lo)
{
    uint32_t top = scaled ? pack_half(a * s, b * s) : pack_half(a, b);
    asm("" : QK_REG(top));
    const half2v h = __builtin_bit_cast(half2v, top);
    hi = top;
    lo = __builtin_bit_cast(uint32_t, half2v{(_Float16)__builtin_fmaf(a, s, -(float)h[0]), (_Float16)__builtin_fmaf(b, s, -(float)h[1])});
}
__device__ __forceinline__ Half2 split2(const float* x)
{
    u32x4 h, l;
    const float one = pinned_one();
#pragma unroll
    for (int i = 0; i < 4; i++) {
        uint32_t hi, lo;
        split_pair(x[2 * i], x[2 * i + 1], one, false, hi, lo);
        h[i] = hi;
        l[i] = lo;
    }
    return Half2{__builtin_bit_cast(half8, h), __builtin_bit_cast(half8, l)};
}

// Exponent of the power of two that a row is divided by, so that its largest magnitude m comes into [2^14, 2^15): as high as a
// half allows, since elements below 2^-2 lose bits.  Not below -126, so that the power and its reciprocal are normal.
__device__ __forceinline__ int top_exponent(float m)
{
    return max((int)(f2u(m) >> 23) - 127 - 14, -126);
}
__device__ __forceinline__ float pow2i(int e) { return u2f((uint32_t)(e + 127) << 23); }

// Ancestors of the nodes node0 .. node0 + n - 1 of a run as bits, kin[n][QKK_TREE_MAX / 32] in LDS; s_up: the run's parents
// (QKK_TREE_MAX entries), thread i brings node i's (requested early: tree_parent).  The whole workgroup, at least QKK_TREE_MAX
// threads, calls it (two barriers).
__device__ __forceinline__ int32_t tree_parent(const int32_t* __restrict__ parent, const Run& u)
{
    return threadIdx.x < u.n ? parent[u.r0 + threadIdx.x] : -1;
}
__device__ __forceinline__ void tree_bits(int32_t up_of, uint32_t node0, uint32_t n, int32_t* s_up, uint32_t (*kin)[QKK_TREE_MAX / 32])
{
    if (threadIdx.x < QKK_TREE_MAX) s_up[threadIdx.x] = up_of;
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < n; i += blockDim.x) {
        uint32_t w[QKK_TREE_MAX / 32] = {};
#pragma unroll
        for (uint32_t b = 0; b < QKK_TREE_MAX / 32; b++) w[b] = 0;
        int32_t a = (int32_t)(node0 + i);
        while (true) { // ends: a parent lies below its node
#pragma unroll
            for (uint32_t b = 0; b < QKK_TREE_MAX / 32; b++) w[b] |= (uint32_t)(a >> 5) == b ? 1u << (a & 31) : 0u;
            const int32_t up = s_up[a];
            if (up < 0 || up >= a) break;
            a = up;
        }
#pragma unroll
        for (uint32_t b = 0; b < QKK_TREE_MAX / 32; b++) kin[i][b] = w[b];
    }
    __syncthreads();
}

// rows x heads of a run that fit the kernel for few rows: one block of 16, for dh 128 two (at dh 256 a second block's accumulators
// do not fit the registers)
constexpr uint32_t few_rows(uint32_t dh) { return dh == 128 ? 32 : 16; }

// Which of four neighbouring keys, the first `rel` rows behind the tree's first row (negative: in front of the tree), a node sees.
__device__ __forceinline__ uint32_t tree_four(const uint32_t* kin, int32_t rel)
{
    constexpr uint32_t W = QKK_TREE_MAX / 32;
    const uint32_t before = (uint32_t)min(max(-rel, 0), 4), at = (uint32_t)max(rel, 0), w = min(at >> 5, W - 1); // no branches
    const uint32_t lo = kin[w], hi = kin[min(w + 1, W - 1)];
    const uint64_t both = ((uint64_t)(w + 1 < W ? hi : 0u) << 32) | lo;
    const uint32_t bits = at < QKK_TREE_MAX ? (uint32_t)(both >> (at & 31u)) : 0u;
    return ((bits << before) | ((1u << before) - 1u)) & 15u;
}

// query rows (positions x heads of a group) per workgroup of the kernel for many rows, and its blocks of them: a run's blocks begin
// at its own first row, so every run may have one that is not full
constexpr uint32_t AR_TILE_ROWS = 128;
inline uint32_t tile_blocks(uint32_t n_rows, uint32_t n_run, uint32_t G) { return (uint32_t)((uint64_t)n_rows * G / AR_TILE_ROWS) + n_run; }

// Items of one KV head that a launch has to have room for, `blocks` the blocks of rows at most.  item_of cuts what is seen, at least half
// of what it counts out, into no more than `slots` full ranges, and every block may have one that is not full.  One per block where
// the keys are not cut.
inline uint32_t items_of(uint32_t blocks, uint32_t slots, uint32_t n_split)
{
    const uint64_t all = (uint64_t)blocks * n_split, made = 2ull * slots + blocks;
    return (uint32_t)(n_split == 1 ? blocks : all < made ? all : made);
}

void launch_attn_few(const RunsCall& call, int type, uint32_t dh, bool tree, hipStream_t st);
void launch_attn_tile(const RunsCall& call, int type, uint32_t dh, bool tree, hipStream_t st);

} // namespace qk
