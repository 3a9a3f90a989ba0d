// Attention of one query token per sequence over a paged pool, for any number of kv heads, 1..8 query heads per kv head,
// head_dim 64 or 128, F16 or E4M3 blocks: the part that the scored decode attention and the shared-prefix attention have in
// common (the latter runs it over the tokens behind the prefix).
//
//   x[t] = scale * log2(e) * k_scale * (q . k_t),   m >= max x - 6,   l = sum 2^(x[t] - m),   O = sum 2^(x[t] - m) * v_t
//
// and (m, l, O) of a token range is one partial result; ranges are joined by a second kernel.
//
// Bound: every cached K and V byte is read once, 2 x head_dim multiply-adds per query head and byte pair, so HBM sets the pace and
// what matters is bytes in flight and few instructions per byte.  A warp works alone: one kv head, one contiguous share of the
// batch's cached blocks, an 8 KB x 3 ring of its own that its lanes fill with 16-byte cp.async and read back lane by lane (every
// lane copies the pieces that its own MMA fragments need, so the ring needs no barrier and no swizzle).  The eight warps of a CTA
// are eight kv heads of the same tokens where the pool has eight, so the copies of a CTA cover whole pool rows.  The order of the
// dims inside a contraction is free, which is what lets a lane's fragment be a 16-byte run of a row: the four lanes of a token take
// neighbouring 16-byte pieces of K (64-byte runs), the eight lanes of four tokens neighbouring pieces of V (128-byte runs).
// Both contractions run on mma.sync m16n8k16 with the tokens (K) or the dims (V) as the 16 rows and the query heads as the 8
// columns; the maximum is only raised, for all lanes at once after a vote, when a score exceeds it by 2^6, so the common step has
// no shuffle in it.
//
// Work split: the batch's blocks, sequence after sequence, are cut into `parts` equal shares that may span sequences; part p and
// sequence s meet in partial slot p + s, which is unique because both only grow along the batch.
#pragma once
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <stdint.h>

namespace tkv_rows {

constexpr int BS = 16;                       // tokens per block
constexpr int WARPS = 8;
constexpr int STAGES = 3;
constexpr int STAGE_DATA = 8192, STAGE_BYTES = STAGE_DATA + 64;
constexpr uint32_t SEQ_CACHE = 1024;         // sequences whose ranges a CTA keeps in shared memory (more are looked up again)
constexpr float RAISE = 6.0f;                // log2: probabilities reach 2^6, far inside F16

struct Args {
    const char *k_base, *v_base;             // layer tensors
    const float *k_scales, *v_scales;        // [total_blocks][n_kv_heads], or null
    const void* q;                           // f16 or f32 [n_seqs][n_q_heads][D]
    const uint32_t *tables, *kv_lens;
    const uint32_t *group_starts, *prefix_lens;   // shared-prefix groups, or null: ranges begin at token 0
    float *part_o, *part_ml;                 // [slot][n_q_heads][D], [slot][n_q_heads][2]
    float* logits;                           // [n_seqs][n_q_heads][logit_stride], or null
    uint32_t* plan;                          // [0] blocks per part, [1 + s] blocks before sequence s (n_seqs + 1 entries)
    uint32_t* status;
    uint64_t block_stride;
    uint32_t row_stride, n_seqs, n_groups, n_q_heads, n_kv_heads, group, table_stride, max_kv_len, max_prefix_len, total_blocks, parts, min_share,
        logit_stride;
    float scale_log2;
};

__device__ __forceinline__ void report(uint32_t* status, uint32_t code) {
    if (status) atomicCAS(status, 0u, code);
}
__device__ __forceinline__ float exp2_fast(float x) {          // 2^x, relative error 2^-22, 2^-inf = 0
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ uint32_t h2_bits(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }
__device__ __forceinline__ uint32_t e4m3x2_h2(uint32_t two_bytes) {
    uint32_t r;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"((unsigned short)two_bytes));
    return r;
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {   // an 8 x 8 matrix of 16-bit values, two to a lane
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
    return r;
}
__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <int BYTES> __device__ __forceinline__ void copy_async(uint32_t dst, const void* src, bool ok) {   // zeros where !ok
    if (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(ok ? 16u : 0u) : "memory");
    if (BYTES == 8) asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(dst), "l"(src), "r"(ok ? 8u : 0u) : "memory");
    if (BYTES == 4) asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(ok ? 4u : 0u) : "memory");
}

// The group table is device memory that the host has not seen: it is used only if its starts ascend and end inside the batch and
// its prefixes are whole blocks within the host's bound.
__device__ __forceinline__ bool groups_bad(const uint32_t* starts, const uint32_t* prefix, uint32_t n_groups, uint32_t n_seqs, uint32_t max_prefix,
                                           uint32_t tid, uint32_t n_threads) {
    bool bad = false;
    for (uint32_t g = tid; g < n_groups; g += n_threads) {
        const uint32_t lo = starts[g], hi = starts[g + 1], p = prefix[g];
        bad |= lo > hi || hi > n_seqs || (p % BS) != 0 || p > max_prefix;
    }
    return bad;
}
// the group of sequence s, or n_groups where it is in none (a batch padded behind its last sequence)
__device__ __forceinline__ uint32_t group_of(const uint32_t* starts, uint32_t n_groups, uint32_t s) {
    if (!n_groups || s < starts[0] || s >= starts[n_groups]) return n_groups;
    uint32_t lo = 0, hi = n_groups;          // starts[lo] <= s < starts[hi]
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) >> 1;
        if (starts[mid] <= s) lo = mid;
        else hi = mid;
    }
    return lo;
}

// tokens [x, y) of sequence s that the rows kernel attends to; x is a whole number of blocks
__device__ __forceinline__ uint2 own_range(const Args& a, uint32_t s) {
    const uint32_t len = min(a.kv_lens[s], a.max_kv_len);
    if (!a.group_starts) return make_uint2(0u, len);
    const uint32_t g = group_of(a.group_starts, a.n_groups, s);
    if (g == a.n_groups) return make_uint2(0u, 0u);
    const uint32_t begin = a.prefix_lens[g];
    return begin < len ? make_uint2(begin, len) : make_uint2(0u, 0u);
}
__device__ __forceinline__ uint32_t blocks_of(uint2 r) { return (r.y + BS - 1) / BS - r.x / BS; }

template <int D, bool FP8> struct Shape {
    static constexpr int ES = FP8 ? 1 : 2;
    static constexpr int KB = D / 4 * ES, VB = D / 8 * ES;     // bytes of a K token per lane (4 lanes share it), of a V token (8 lanes)
    static constexpr int KP = KB / 16;                          // 16-byte pieces of a K token per lane
    static constexpr int VPB = VB >= 16 ? 16 : 8, VP = VB / VPB;
    static constexpr int LANE_BLOCK = 2 * KB + 4 * VB;          // a lane holds 2 tokens of K and 4 of V
    static constexpr int NB = STAGE_DATA / 32 / LANE_BLOCK;     // blocks per stage: 1 (F16, 128 dims) .. 4 (E4M3, 64 dims)
    static constexpr int KS = D / 16, MT = D / 16;              // k-steps of Q.K, row tiles of V^T.P
};

// a position in a part's stream of blocks
struct Cursor {
    uint32_t seq, block, left;                                  // block of the sequence; blocks left in it for this part
    uint32_t len;                                               // tokens of the sequence
    uint32_t rest;                                              // blocks left for this part behind this sequence
};

// F32: q and out are F32, q is used as two F16 terms (22 bits) and the probabilities too; else q and out are F16 and a probability is
// one F16 (2^-12 of its own value at most, below the rounding of the output).
template <int D, bool FP8, bool F32>
__global__ void __launch_bounds__(WARPS * 32, 1) rows_attn(const Args a) {
    using S = Shape<D, FP8>;
    constexpr int NB = S::NB, KS = S::KS, MT = S::MT;
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u, grp = lane >> 2, j = lane & 3u;
    extern __shared__ __align__(128) unsigned char smem[];
    uint2* seq_info = reinterpret_cast<uint2*>(smem + WARPS * STAGES * STAGE_BYTES);            // [SEQ_CACHE]
    __shared__ uint32_t cum[WARPS * 32 + 1], warp_sum[WARPS];

    if (a.group_starts) {
        const bool bad = groups_bad(a.group_starts, a.prefix_lens, a.n_groups, a.n_seqs, a.max_prefix_len, tid, WARPS * 32);
        if (__syncthreads_or(bad)) {
            if (tid == 0) {
                report(a.status, 2u);
                if (blockIdx.x == 0) a.plan[0] = 0;             // nothing was computed
            }
            return;
        }
    }
    // ---- blocks before every run of `per` sequences ----
    const uint32_t per = (a.n_seqs + WARPS * 32 - 1) / (WARPS * 32);
    uint32_t mine = 0;
    for (uint32_t i = 0; i < per; i++) {
        const uint32_t s = tid * per + i;
        if (s < a.n_seqs) {
            const uint2 r = own_range(a, s);
            if (s < SEQ_CACHE) seq_info[s] = r;
            mine += blocks_of(r);
            if (blockIdx.x == 0 && a.kv_lens[s] > a.max_kv_len) report(a.status, 2u);
        }
    }
    uint32_t incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t v = __shfl_up_sync(0xFFFFFFFFu, incl, o);
        if (lane >= (uint32_t)o) incl += v;
    }
    if (lane == 31) warp_sum[warp] = incl;
    __syncthreads();
    uint32_t before = 0;
#pragma unroll
    for (int w = 0; w < WARPS; w++) before += w < (int)warp ? warp_sum[w] : 0u;
    cum[tid] = before + incl - mine;
    if (tid == WARPS * 32 - 1) cum[WARPS * 32] = before + incl;
    __syncthreads();
    const uint32_t total = cum[WARPS * 32];
    const uint32_t share = max((total + a.parts - 1) / a.parts, a.min_share);
    auto range_of = [&](uint32_t s) { return s < SEQ_CACHE ? seq_info[s] : own_range(a, s); };
    if (blockIdx.x == 0) {                                      // the joining kernel finds a sequence's parts from these
        uint32_t at = cum[tid];
        for (uint32_t i = 0; i < per; i++) {
            const uint32_t s = tid * per + i;
            if (s < a.n_seqs) {
                a.plan[1 + s] = at;
                at += blocks_of(range_of(s));
            }
        }
        if (tid == 0) {
            a.plan[0] = share;
            a.plan[1 + a.n_seqs] = total;
        }
    }
    const uint32_t stream = blockIdx.x * WARPS + warp, kvh = stream % a.n_kv_heads, part = stream / a.n_kv_heads;
    if (part >= a.parts || (uint64_t)part * share >= total) return;
    const uint32_t first = part * share, n_mine = min(share, total - first);

    // ---- the first sequence of this part ----
    Cursor c;
    {
        uint32_t lo = 0, hi = WARPS * 32;                       // cum[lo] <= first < cum[hi]
        while (hi - lo > 1) {
            const uint32_t mid = (lo + hi) >> 1;
            if (cum[mid] <= first) lo = mid;
            else hi = mid;
        }
        uint32_t s = lo * per, at = cum[lo];
        uint2 r = range_of(s);
        while (at + blocks_of(r) <= first) {
            at += blocks_of(r);
            r = range_of(++s);
        }
        c.seq = s;
        c.block = r.x / BS + (first - at);
        c.left = min(blocks_of(r) - (first - at), n_mine);
        c.len = r.y;
        c.rest = n_mine - c.left;
    }
    auto next_sequence = [&](Cursor& x) {                       // called with left == 0 and rest > 0: a later sequence has blocks
        uint2 r;
        do r = range_of(++x.seq);
        while (blocks_of(r) == 0);
        x.block = r.x / BS;
        x.left = min(blocks_of(r), x.rest);
        x.len = r.y;
        x.rest -= x.left;
    };

    // ---- the ring ----
    unsigned char* ring = smem + (size_t)warp * STAGES * STAGE_BYTES;
    const uint32_t ring_addr = (uint32_t)__cvta_generic_to_shared(ring);
    const size_t head_off = (size_t)kvh * D * S::ES;
    Cursor f = c;                                               // what is fetched next
    bool f_done = false;
    auto ids_at = [&](const Cursor& x, bool done) -> uint32_t { // lane b: block id of block b of the stage at x
        uint32_t id = 0;
        if (!done && lane < (uint32_t)NB && lane < x.left) {
            id = __ldg(a.tables + (size_t)x.seq * a.table_stride + x.block + lane);
            if (id >= a.total_blocks) {                         // never dereferenced: block 0 is read instead and the launch reports it
                report(a.status, 2u);
                id = 0;
            }
        }
        return id;
    };
    uint32_t ids = ids_at(f, false);
    auto fetch = [&](uint32_t slot) {
        if (!f_done) {
            const uint32_t base = ring_addr + slot * STAGE_BYTES;
            const uint32_t n = min(f.left, (uint32_t)NB);
#pragma unroll
            for (int b = 0; b < NB; b++) {
                const uint32_t id = __shfl_sync(0xFFFFFFFFu, ids, b);
                const uint32_t t0 = (f.block + b) * BS;
                const uint32_t live = b < (int)n ? min((uint32_t)BS, f.len - t0) : 0u;
                const char* kb = a.k_base + (uint64_t)id * a.block_stride + head_off;
                const char* vb = a.v_base + (uint64_t)id * a.block_stride + head_off;
                const uint32_t kd = base + b * (S::LANE_BLOCK * 32) + lane * 16, vd = base + b * (S::LANE_BLOCK * 32) + 2 * S::KB * 32 + lane * S::VPB;
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const uint32_t tok = grp + 8 * h;
                    const bool ok = tok < live;
                    const char* row = kb + (size_t)(ok ? tok : 0u) * a.row_stride + j * 16;
#pragma unroll
                    for (int i = 0; i < S::KP; i++) copy_async<16>(kd + (h * S::KP + i) * 512, row + i * 64, ok);
                }
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const uint32_t tok = 2 * j + (i & 1) + 8 * (i >> 1);
                    const bool ok = tok < live;
                    const char* row = vb + (size_t)(ok ? tok : 0u) * a.row_stride + grp * S::VPB;
#pragma unroll
                    for (int p = 0; p < S::VP; p++) copy_async<S::VPB>(vd + (i * S::VP + p) * (32 * S::VPB), row + p * 128, ok);
                }
            }
            if (FP8 && a.k_scales) {                            // lane 2b: K scale of block b, lane 2b + 1: V scale
                const uint32_t id = __shfl_sync(0xFFFFFFFFu, ids, (lane >> 1) & (NB - 1));
                if (lane < 2u * NB) copy_async<4>(base + STAGE_DATA + lane * 4, ((lane & 1u) ? a.v_scales : a.k_scales) + (size_t)id * a.n_kv_heads + kvh, true);
            }
            f.block += n;
            f.left -= n;
            if (f.left == 0) {
                if (f.rest) next_sequence(f);
                else f_done = true;
            }
            ids = ids_at(f, f_done);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");   // one group per step, empty past the end
    };
#pragma unroll
    for (int i = 0; i < STAGES - 1; i++) fetch(i);

    uint32_t q_hi[KS][2], q_lo[F32 ? KS : 1][2];
    auto load_q = [&](uint32_t seq) {
        const size_t at = ((size_t)seq * a.n_q_heads + kvh * a.group + (grp < a.group ? grp : 0u)) * D;
        const bool live = grp < a.group;
#pragma unroll
        for (int s = 0; s < KS; s++) {
            const int dim = FP8 ? (4 * (s >> 2) + (int)j) * 16 + (s & 3) * 4 : (4 * (s >> 1) + (int)j) * 8 + (s & 1) * 4;
            if (F32) {
                const float4 x = live ? *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(a.q) + at + dim) : make_float4(0, 0, 0, 0);
                const __half2 h0 = __floats2half2_rn(x.x, x.y), h1 = __floats2half2_rn(x.z, x.w);
                const float2 f0 = __half22float2(h0), f1 = __half22float2(h1);
                q_hi[s][0] = h2_bits(h0);
                q_hi[s][1] = h2_bits(h1);
                q_lo[F32 ? s : 0][0] = h2_bits(__floats2half2_rn(x.x - f0.x, x.y - f0.y));
                q_lo[F32 ? s : 0][1] = h2_bits(__floats2half2_rn(x.z - f1.x, x.w - f1.y));
            } else {
                const uint2 x = live ? *reinterpret_cast<const uint2*>(reinterpret_cast<const __half*>(a.q) + at + dim) : make_uint2(0, 0);
                q_hi[s][0] = x.x;
                q_hi[s][1] = x.y;
            }
        }
    };

    float o[MT][4], m2[2], l2[2], v_ref, v_inv;                // o[t]: dims 2t, 2t + 1 of this lane's run, query heads 2j, 2j + 1; in units of v_ref
    auto begin_sequence = [&](uint32_t seq) {
        load_q(seq);
#pragma unroll
        for (int t = 0; t < MT; t++) o[t][0] = o[t][1] = o[t][2] = o[t][3] = 0.0f;
        m2[0] = m2[1] = -INFINITY;
        l2[0] = l2[1] = 0.0f;
        v_ref = FP8 ? 0x1p-100f : 1.0f;                         // a power of two above every V scale met so far: P x scale / v_ref stays in F16's range
        v_inv = FP8 ? 0x1p+100f : 1.0f;
    };
    begin_sequence(c.seq);

    for (uint32_t step = 0;; step++) {
        fetch((step + STAGES - 1) % STAGES);                    // into the stage that the step before this one has read
        asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 1) : "memory");
        __syncwarp();
        const unsigned char* stage = ring + (step % STAGES) * STAGE_BYTES;
        const uint32_t n = min(c.left, (uint32_t)NB);

        // scores
        float x[NB][4], vs[NB];
#pragma unroll
        for (int b = 0; b < NB; b++) {
            const uint4* kp = reinterpret_cast<const uint4*>(stage + b * (S::LANE_BLOCK * 32)) + lane;
            float even[4] = {0.0f, 0.0f, 0.0f, 0.0f}, odd[4] = {0.0f, 0.0f, 0.0f, 0.0f};   // two chains
#pragma unroll
            for (int i = 0; i < S::KP; i++) {
                const uint4 lo = kp[i * 32], hi = kp[(S::KP + i) * 32];
                const uint32_t wl[4] = {lo.x, lo.y, lo.z, lo.w}, wh[4] = {hi.x, hi.y, hi.z, hi.w};
#pragma unroll
                for (int u = 0; u < (FP8 ? 4 : 2); u++) {
                    const int s = FP8 ? 4 * i + u : 2 * i + u;
                    uint32_t a0, a1, a2, a3;
                    if (FP8) {
                        a0 = e4m3x2_h2(wl[u] & 0xFFFFu);
                        a2 = e4m3x2_h2(wl[u] >> 16);
                        a1 = e4m3x2_h2(wh[u] & 0xFFFFu);
                        a3 = e4m3x2_h2(wh[u] >> 16);
                    } else {
                        a0 = wl[2 * u];
                        a2 = wl[2 * u + 1];
                        a1 = wh[2 * u];
                        a3 = wh[2 * u + 1];
                    }
                    mma16816((u & 1) ? odd : even, a0, a1, a2, a3, q_hi[s][0], q_hi[s][1]);
                    if (F32) mma16816((u & 1) ? odd : even, a0, a1, a2, a3, q_lo[F32 ? s : 0][0], q_lo[F32 ? s : 0][1]);
                }
            }
            float ks = a.scale_log2;
            vs[b] = 1.0f;
            if (FP8 && a.k_scales) {
                const float2 sc = *reinterpret_cast<const float2*>(stage + STAGE_DATA + b * 8);
                ks *= sc.x;
                vs[b] = b < (int)n ? sc.y : 0.0f;
            }
            const uint32_t live = b < (int)n ? min((uint32_t)BS, c.len - (c.block + b) * BS) : 0u;
#pragma unroll
            for (int i = 0; i < 4; i++) x[b][i] = grp + 8 * (i >> 1) < live ? (even[i] + odd[i]) * ks : -INFINITY;   // x[b][2 * (token half) + head]
            if (a.logits) {
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const uint32_t head = 2 * j + (i & 1), tok = grp + 8 * (i >> 1);
                    if (head < a.group && tok < live)
                        a.logits[((size_t)c.seq * a.n_q_heads + kvh * a.group + head) * a.logit_stride + (c.block + b) * BS + tok] = x[b][i];
                }
            }
        }
        // the maxima in use are raised, for all lanes together, once a score is 2^6 above
        bool over = false;
        float v_top = 0.0f;
#pragma unroll
        for (int b = 0; b < NB; b++) {
#pragma unroll
            for (int i = 0; i < 4; i++) over |= x[b][i] > m2[i & 1] + RAISE;
            v_top = fmaxf(v_top, vs[b]);
        }
        if (__any_sync(0xFFFFFFFFu, over)) {
#pragma unroll
            for (int h = 0; h < 2; h++) {
                float mx = m2[h];
#pragma unroll
                for (int b = 0; b < NB; b++) mx = fmaxf(mx, fmaxf(x[b][h], x[b][2 + h]));
                mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, 4));
                mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, 8));
                mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, 16));
                const float keep = m2[h] == -INFINITY ? 0.0f : exp2_fast(m2[h] - mx);
                m2[h] = mx;
                l2[h] *= keep;
#pragma unroll
                for (int t = 0; t < MT; t++) {
                    o[t][h] *= keep;
                    o[t][2 + h] *= keep;
                }
            }
        }
        if (FP8 && v_top > v_ref) {                             // the same in every lane
            const float up = __uint_as_float(min((__float_as_uint(v_top) >> 23) + 1u, 253u) << 23);
            const float keep = v_ref / up;
            v_ref = up;
            v_inv = 1.0f / up;
#pragma unroll
            for (int t = 0; t < MT; t++)
#pragma unroll
                for (int i = 0; i < 4; i++) o[t][i] *= keep;
        }
        const float sub0 = m2[0] == -INFINITY ? 0.0f : m2[0], sub1 = m2[1] == -INFINITY ? 0.0f : m2[1];
        // probabilities and O += V^T P
#pragma unroll
        for (int b = 0; b < NB; b++) {
            float p[4];
            p[0] = exp2_fast(x[b][0] - sub0);
            p[1] = exp2_fast(x[b][1] - sub1);
            p[2] = exp2_fast(x[b][2] - sub0);
            p[3] = exp2_fast(x[b][3] - sub1);
            l2[0] += p[0] + p[2];
            l2[1] += p[1] + p[3];
            if (FP8) {
                const float vn = vs[b] * v_inv;
#pragma unroll
                for (int i = 0; i < 4; i++) p[i] *= vn;
            }
            const __half2 pl = __floats2half2_rn(p[0], p[1]), ph = __floats2half2_rn(p[2], p[3]);
            const uint32_t b0 = transpose8(h2_bits(pl)), b1 = transpose8(h2_bits(ph));   // rows: tokens 2j, 2j + 1 (+ 8); column: head grp
            uint32_t c0 = 0, c1 = 0;
            if (F32) {
                const float2 fl = __half22float2(pl), fh = __half22float2(ph);
                c0 = transpose8(h2_bits(__floats2half2_rn(p[0] - fl.x, p[1] - fl.y)));
                c1 = transpose8(h2_bits(__floats2half2_rn(p[2] - fh.x, p[3] - fh.y)));
            }
            const unsigned char* vp = stage + b * (S::LANE_BLOCK * 32) + 2 * S::KB * 32 + lane * S::VPB;
#pragma unroll
            for (int pc = 0; pc < S::VP; pc++) {
                uint32_t w[4][S::VPB / 4];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const unsigned char* at = vp + (i * S::VP + pc) * (32 * S::VPB);
                    if (S::VPB == 16) {
                        const uint4 v = *reinterpret_cast<const uint4*>(at);
                        w[i][0] = v.x;
                        w[i][1] = v.y;
                        w[i][S::VPB / 4 - 2] = v.z;
                        w[i][S::VPB / 4 - 1] = v.w;
                    } else {
                        const uint2 v = *reinterpret_cast<const uint2*>(at);
                        w[i][0] = v.x;
                        w[i][1] = v.y;
                    }
                }
                constexpr int TILES = S::VPB / S::ES / 2;       // two dims of the run per row tile
#pragma unroll
                for (int t = 0; t < TILES; t++) {
                    uint32_t a0, a1, a2, a3;
                    if (FP8) {
                        const uint32_t lo = 2u * (t & 1), sel0 = lo | ((4u + lo) << 4), sel1 = (lo + 1u) | ((5u + lo) << 4);
                        a0 = e4m3x2_h2(__byte_perm(w[0][t >> 1], w[1][t >> 1], sel0));
                        a1 = e4m3x2_h2(__byte_perm(w[0][t >> 1], w[1][t >> 1], sel1));
                        a2 = e4m3x2_h2(__byte_perm(w[2][t >> 1], w[3][t >> 1], sel0));
                        a3 = e4m3x2_h2(__byte_perm(w[2][t >> 1], w[3][t >> 1], sel1));
                    } else {
                        a0 = __byte_perm(w[0][t], w[1][t], 0x5410u);
                        a1 = __byte_perm(w[0][t], w[1][t], 0x7632u);
                        a2 = __byte_perm(w[2][t], w[3][t], 0x5410u);
                        a3 = __byte_perm(w[2][t], w[3][t], 0x7632u);
                    }
                    mma16816(o[pc * TILES + t], a0, a1, a2, a3, b0, b1);
                    if (F32) mma16816(o[pc * TILES + t], a0, a1, a2, a3, c0, c1);
                }
            }
        }
        c.block += n;
        c.left -= n;
        if (c.left) continue;

        // ---- the sequence's blocks of this part are done ----
        const uint32_t slot = part + c.seq;
#pragma unroll
        for (int h = 0; h < 2; h++) {
            float l = l2[h];
            l += __shfl_xor_sync(0xFFFFFFFFu, l, 4);
            l += __shfl_xor_sync(0xFFFFFFFFu, l, 8);
            l += __shfl_xor_sync(0xFFFFFFFFu, l, 16);
            const uint32_t head = 2 * j + h;
            if (head < a.group) {
                const size_t row = (size_t)slot * a.n_q_heads + kvh * a.group + head;
                if (grp == 0) *reinterpret_cast<float2*>(a.part_ml + row * 2) = make_float2(m2[h], l);
                float* dst = a.part_o + row * D;
#pragma unroll
                for (int t = 0; t < MT; t++) {
                    constexpr int RUN = S::VPB / S::ES;         // dims of a piece
                    const int e = 2 * t, dim = (e / RUN) * (8 * RUN) + (int)grp * RUN + e % RUN;
                    *reinterpret_cast<float2*>(dst + dim) = make_float2(o[t][h] * v_ref, o[t][2 + h] * v_ref);
                }
            }
        }
        if (!c.rest) break;
        next_sequence(c);
        begin_sequence(c.seq);
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
}

// ---- host side -------------------------------------------------------------------------------------------------------------
struct Split {
    uint32_t parts, min_share, grid;
};
// Parts for a batch of at most `blocks` cached blocks: one warp per part and kv head, one CTA per SM, and no part shorter than
// MIN_SHARE blocks (a part costs the joining kernel a partial result per query head).
constexpr uint32_t MIN_SHARE = 4;
inline Split split_for(uint64_t blocks, uint32_t n_kv_heads, uint32_t sms) {
    Split s;
    s.min_share = MIN_SHARE;
    const uint64_t most = (uint64_t)sms * WARPS / n_kv_heads, want = (blocks + MIN_SHARE - 1) / MIN_SHARE;
    s.parts = (uint32_t)(most < 1 ? 1 : want < 1 ? 1 : want < most ? want : most);
    s.grid = (uint32_t)(((uint64_t)s.parts * n_kv_heads + WARPS - 1) / WARPS);
    return s;
}
constexpr size_t SMEM_BYTES = (size_t)WARPS * STAGES * STAGE_BYTES + SEQ_CACHE * sizeof(uint2);
static_assert(SMEM_BYTES + 2048 <= 227 * 1024, "shared memory of one CTA");

template <int D, bool FP8, bool F32> cudaError_t launch_one(const Args& a, uint32_t grid, cudaStream_t st) {
    auto kernel = rows_attn<D, FP8, F32>;
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)SMEM_BYTES);
    if (e != cudaSuccess) return e;
    kernel<<<grid, WARPS * 32, SMEM_BYTES, st>>>(a);
    return cudaGetLastError();
}
inline cudaError_t launch_rows(uint32_t head_dim, bool fp8, bool f32, const Args& a, uint32_t grid, cudaStream_t st) {
    if (head_dim == 128) {
        if (fp8) return f32 ? launch_one<128, true, true>(a, grid, st) : launch_one<128, true, false>(a, grid, st);
        return f32 ? launch_one<128, false, true>(a, grid, st) : launch_one<128, false, false>(a, grid, st);
    }
    if (fp8) return f32 ? launch_one<64, true, true>(a, grid, st) : launch_one<64, true, false>(a, grid, st);
    return f32 ? launch_one<64, false, true>(a, grid, st) : launch_one<64, false, false>(a, grid, st);
}

}  // namespace tkv_rows
