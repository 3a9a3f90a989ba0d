// Attention of one query token per sequence over a paged pool, for any number of kv heads, 1..8 query heads per kv head,
// head_dim 64 or 128, F16 or E4M3 blocks: the part that the scored decode attention and the shared-prefix attention have in
// common (the latter runs it over the tokens behind the prefix).
//
//   x[t] = scale * log2(e) * k_scale * (q . k_t),   m >= max x - 14,   l = sum 2^(x[t] - m),   O = sum 2^(x[t] - m) * v_t
//
// and (m, l, O) of a token range is one partial result; ranges are joined by a second kernel.
//
// Bound: every cached K and V byte is read once, 2 x head_dim multiply-adds per query head and byte pair, so HBM sets the pace and
// what matters is bytes in flight, large copies, and few instructions per byte.  A stream is a run of up to eight kv heads over a
// contiguous share of the batch's cached blocks: a producer warp keeps a ring of whole blocks in flight with bulk copies, and
// consumer warps, one kv head each, read their fragments out of the stage and hand it back.  A CTA holds 8 / heads streams, so
// pools with few kv heads keep as many warps busy.  A block arrives as four runs of four tokens, 32 bytes apart from a multiple of 128
// in shared memory (one copy per token cost 50 ns each: 1.6 us per block against 0.7 us that HBM needs for an E4M3 block; one copy
// per block leaves four-way bank conflicts).  With token(j, i) = 4 * (i odd ? j ^ 2 : j) + i as the i-th token of the four lanes j, the
// 16-byte fragment reads of K (four lanes side by side in each of two tokens) and of V (two lanes side by side in each of four tokens)
// are free of bank conflicts.  The order of the dims inside a contraction is free too: a lane's fragment is a 16-byte run.
// Both contractions run on mma.sync m16n8k16 with the tokens (K) or the dims (V) as the 16 rows and the query heads as the 8
// columns; the reference m lies 8 below a maximum that it is set from and is only raised, for all lanes at once after a vote, when a score
// exceeds it by 14, so the common step has no shuffle in it.  Probabilities are used as two F16 terms: with up to four query heads per kv
// head the second term rides in the four spare columns of the same MMAs, else it is a second set of them.  Between 2^8 (or more) for the
// largest and F16's smallest step of 2^-24 they keep 22 bits down to 2^-10 of the largest and are off by 2^-33 of it below.
// In a scaled E4M3 pool what the MMA takes is 2^(x - m) * v_scale * unit, with a power of two `unit` per query head that holds the largest such
// product met so far (not the largest scale: a block that is large but not attended to must not push the others among F16's subnormals)
// where the largest probability would be.
//
// A block costs a consumer a chain of dependent steps (wait, fragments, eight MMAs, exp2, transposes, eight MMAs).  For an F16 block the
// chain is shorter than the time in which HBM delivers the block (131 071 tokens of 8 heads: 92 us, 5.9 TB/s).  An E4M3 block has half the bytes
// and a conversion in the chain: 64 sequences of up to 4 096 tokens take 54 us (4.9 TB/s), one context of 131 071 the same, of which delivery alone
// is 46 to 47 (consumers that only hand their stages back; 5.8 TB/s, the rate of F16 blocks) and 7 to 8 the arithmetic that the ring does not
// hide.  The scales are not it (53 us without).  Two consumers per head on alternate blocks did not help: the same 71 us for the whole call, and
// 91 against 75 us for one context of 131 071 tokens.
//
// Work split: the batch's blocks, sequence after sequence, are cut into `parts` equal shares that may span sequences; part p and
// sequence s meet in partial slot p + s, which is unique because both only grow along the batch.
#pragma once
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <stdint.h>

#include <atomic>

namespace tkv_rows {

constexpr int BS = 16;                       // tokens per block
constexpr int WARPS = 8;                     // consumer warps of a share of the blocks
constexpr int THREADS = (WARPS + 1) * 32;    // and the producer
constexpr int MAX_STAGES = 8;
constexpr uint32_t PAD = 32;                 // bytes between runs of four tokens
constexpr uint32_t SCALE_BYTES = 2 * WARPS * 4;
constexpr uint32_t RING_BYTES = 208 * 1024;  // of all streams of a CTA
constexpr uint32_t SEQ_CACHE = 1024;         // sequences whose ranges a CTA keeps in shared memory (more are looked up again)
constexpr float HEAD = 8.0f, RAISE = 14.0f;  // log2: what is largest is put at 2^8 and may grow to 2^14 (F16 ends below 2^16) before it is put there again
constexpr float UNIT_MOST = 0x1p+100f;
// of a power of two
__device__ __forceinline__ float log2_of_power(float u) { return (float)((int)(__float_as_uint(u) >> 23) - 127); }
__device__ __forceinline__ float inverse_of_power(float u) { return __uint_as_float(0x7F000000u - __float_as_uint(u)); }
// The unit of a row whose reference was just raised by `up`; `top` is the largest probability times V scale at hand as a power of two (-inf: none).
// Measured absolutely a unit only falls, as a maximum only rises.  (up <= 126: what O is multiplied by stays a number.)
__device__ __forceinline__ float next_unit(float unit, float up, float top) {
    const float e = fminf(log2_of_power(unit) + fminf(up, 126.0f), HEAD - top);
    return __uint_as_float((uint32_t)((int)floorf(fminf(fmaxf(e, -110.0f), 100.0f)) + 127) << 23);
}

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
    uint32_t heads, streams, head_groups, stages;   // kv heads per stream, streams per CTA, streams per part, ring depth
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
__device__ __forceinline__ float log2_fast(float x) {
    float r;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
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
__device__ __forceinline__ uint32_t smem_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ bool bar_test(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    return ok != 0;
}
// bounded: gives up after 2^17 polls (a few seconds: a poll may sleep for some 45 us), or as soon as another warp of the CTA has recorded a failure
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity, const volatile uint32_t* fail) {
    for (uint32_t it = 0; it < (1u << 17); it++) {
        if (bar_test(bar, parity)) return true;
        if ((it & 15u) == 15u && *fail) return false;
    }
    return false;
}

__device__ __forceinline__ void shared_read16(uint32_t at, uint32_t (&w)[4]) {
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(at));
}
__device__ __forceinline__ float shared_read4(uint32_t at) {
    float v;
    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(at));
    return v;
}
__device__ __forceinline__ void shared_read8(uint32_t at, uint32_t (&w)[4]) {
    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(at));
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

// Tokens [x, y) of sequence s that the rows kernel attends to; x is a whole number of blocks.  A member that ends inside its group's
// prefix comes here whole (x = SHORT), with the table row that names the prefix: in the matrix product over the prefix the tokens
// behind its end would be zeros times V, and 0 x infinity and 0 x NaN are NaN.
constexpr uint32_t SHORT = 1;                // below a block: x / BS is 0
__device__ __forceinline__ uint2 own_range(const Args& a, uint32_t s) {
    const uint32_t len = min(a.kv_lens[s], a.max_kv_len);
    if (!a.group_starts) return make_uint2(0u, len);
    const uint32_t g = group_of(a.group_starts, a.n_groups, s);
    if (g == a.n_groups) return make_uint2(0u, 0u);
    const uint32_t begin = a.prefix_lens[g];
    return begin < len ? make_uint2(begin, len) : begin == len ? make_uint2(0u, 0u) : make_uint2(SHORT, len);
}
// the table row of a sequence with that range
__device__ __forceinline__ uint32_t table_row(const Args& a, uint2 range, uint32_t s) {
    return range.x == SHORT ? a.group_starts[group_of(a.group_starts, a.n_groups, s)] : s;
}
__device__ __forceinline__ uint32_t blocks_of(uint2 r) { return (r.y + BS - 1) / BS - r.x / BS; }

template <int D, bool FP8> struct Shape {
    static constexpr int ES = FP8 ? 1 : 2, ROW = D * ES;       // bytes of one kv head's row
    static constexpr int KP = ROW / 64;                         // 16-byte pieces of a K token per lane (4 lanes share it)
    static constexpr int VB = ROW / 8, VPB = VB >= 16 ? 16 : 8, VP = VB / VPB;   // bytes of a V token per lane (8 lanes), and its pieces
    static constexpr int KS = D / 16, MT = D / 16;              // k-steps of Q.K, row tiles of V^T.P
};

// a position in a part's run of blocks
struct Cursor {
    uint32_t seq, block, left;                                  // block of the sequence; blocks left in it for this part
    uint32_t len;                                               // tokens of the sequence
    uint32_t row;                                               // of the block table
    uint32_t rest;                                              // blocks left for this part behind this sequence
};

// F32: q and out are F32 and q is used as two F16 terms (22 bits); else both are F16.
// WIDE: more than four query heads per kv head (the second term of the probabilities then takes MMAs of its own).
template <int D, bool FP8, bool F32, bool WIDE>
__global__ void __launch_bounds__(THREADS, 1) rows_attn(const Args a) {
    using S = Shape<D, FP8>;
    constexpr int NWARPS = THREADS / 32;
    constexpr int KS = S::KS, MT = S::MT;
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u;
    extern __shared__ __align__(128) unsigned char ring[];
    __shared__ uint2 seq_info[SEQ_CACHE];
    __shared__ uint32_t cum[THREADS + 1], warp_sum[NWARPS], fail;
    __shared__ uint64_t full[WARPS][MAX_STAGES], empty[WARPS][MAX_STAGES];   // [stream][stage]

    if (a.group_starts) {
        const bool bad = groups_bad(a.group_starts, a.prefix_lens, a.n_groups, a.n_seqs, a.max_prefix_len, tid, THREADS);
        if (__syncthreads_or(bad)) {
            if (tid == 0) {
                report(a.status, 2u);
                if (blockIdx.x == 0) a.plan[0] = 0;             // nothing was computed
            }
            asm volatile("griddepcontrol.wait;" ::: "memory");
            return;
        }
    }
    // ---- blocks before every run of `per` sequences ----
    const uint32_t per = (a.n_seqs + THREADS - 1) / THREADS;
    uint32_t mine = 0;
    for (uint32_t i = 0; i < per; i++) {
        const uint32_t s = tid * per + i;
        if (s < a.n_seqs) {
            const uint2 r = own_range(a, s);
            if (s < SEQ_CACHE) seq_info[s] = r;
            mine += blocks_of(r);
            if (blockIdx.x == 0 && a.kv_lens[s] > a.max_kv_len && (!a.group_starts || group_of(a.group_starts, a.n_groups, s) < a.n_groups)) report(a.status, 2u);
        }
    }
    uint32_t incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t v = __shfl_up_sync(0xFFFFFFFFu, incl, o);
        if (lane >= (uint32_t)o) incl += v;
    }
    if (lane == 31) warp_sum[warp] = incl;
    if (tid < WARPS) {                                          // the streams' barriers; the last run of heads may be short
        const uint32_t hg = (blockIdx.x * a.streams + tid) % a.head_groups, n = min(a.heads, a.n_kv_heads - hg * a.heads);
        for (uint32_t i = 0; i < (uint32_t)MAX_STAGES; i++) {
            // the producer's own arrival and, for scales, one per lane when its copy has landed
            asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_addr(&full[tid][i])), "r"(FP8 && a.k_scales ? 33u : 1u));
            asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_addr(&empty[tid][i])), "r"(n));
        }
        if (tid == 0) fail = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    uint32_t before = 0;
#pragma unroll
    for (int w = 0; w < NWARPS; w++) before += w < (int)warp ? warp_sum[w] : 0u;
    cum[tid] = before + incl - mine;
    if (tid == THREADS - 1) cum[THREADS] = before + incl;
    __syncthreads();
    const uint32_t total = cum[THREADS];
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
    // blocks of part p, and where it starts
    auto part_blocks = [&](uint32_t p) -> uint32_t { return p < a.parts && (uint64_t)p * share < total ? min(share, total - p * share) : 0u; };
    auto part_start = [&](uint32_t p, uint32_t n) -> Cursor {
        const uint32_t first = p * share;
        uint32_t lo = 0, hi = THREADS;                          // cum[lo] <= first < cum[hi]
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
        Cursor c;
        c.seq = s;
        c.block = r.x / BS + (first - at);
        c.left = min(blocks_of(r) - (first - at), n);
        c.len = r.y;
        c.row = table_row(a, r, s);
        c.rest = n - c.left;
        return c;
    };
    auto next_sequence = [&](Cursor& x) {                       // called with left == 0 and rest > 0: a later sequence has blocks
        uint2 r;
        do r = range_of(++x.seq);
        while (blocks_of(r) == 0);
        x.block = r.x / BS;
        x.left = min(blocks_of(r), x.rest);
        x.len = r.y;
        x.row = table_row(a, r, x.seq);
        x.rest -= x.left;
    };
    // a table entry; it is checked where it is used, a few blocks later, so that nothing waits for the load here
    auto table_entry = [&](const Cursor& x, uint32_t i) -> uint32_t { return __ldg(a.tables + (size_t)x.row * a.table_stride + x.block + i); };
    auto checked = [&](uint32_t id) -> uint32_t {
        if (id < a.total_blocks) return id;
        report(a.status, 2u);                                   // never dereferenced: block 0 is read instead and the launch reports it
        return 0u;
    };
    asm volatile("griddepcontrol.launch_dependents;");          // the joining kernel may take its place; it waits for this grid's end by itself
    const uint32_t row_smem = a.heads * S::ROW, run_smem = 4 * row_smem + PAD, plane = 4 * run_smem;
    const uint32_t stage_bytes = 2 * plane + (FP8 ? SCALE_BYTES : 0);    // K, V, scales of K and of V per head

    if (warp == NWARPS - 1) {
        // ---- producer: the streams in step, block k of each; lane x keeps the place in stream x.  A run of tokens is one copy where the
        // stream has all heads of the pool, else its tokens are copied one by one: lane 16 * (V) + token, lanes without a copy idle ----
        const uint32_t stream = blockIdx.x * a.streams + lane, hg_l = stream % a.head_groups;
        const uint32_t n_l = lane < a.streams ? part_blocks(stream / a.head_groups) : 0u;
        Cursor f{};
        if (n_l) f = part_start(stream / a.head_groups, n_l);
        bool done = n_l == 0;
        uint32_t id[4], live[4], id_next[4], live_next[4];
        auto look_up = [&](uint32_t (&ids)[4], uint32_t (&lives)[4]) {    // the next four blocks of lane x's stream
#pragma unroll
            for (int u = 0; u < 4; u++) {
                ids[u] = lives[u] = 0;
                if (!done) {
                    ids[u] = table_entry(f, 0);
                    lives[u] = min((uint32_t)BS, f.len - f.block * BS);
                    f.block++;
                    if (--f.left == 0) {
                        if (f.rest) next_sequence(f);
                        else done = true;
                    }
                }
            }
        };
        look_up(id, live);
        const uint32_t n_max = __reduce_max_sync(0xFFFFFFFFu, n_l);
        const bool whole = a.heads == a.n_kv_heads;
        const uint32_t row = lane & 15u, per_copy = whole ? 4u : 1u;
        const bool copies = row % per_copy == 0;
        const char* base = ((lane >> 4) ? a.v_base : a.k_base) + (size_t)row * a.row_stride;
        const uint32_t dst0 = smem_addr(ring) + (lane >> 4) * plane + (row >> 2) * run_smem + (row & 3u) * row_smem;
        uint64_t policy;                                        // read once: the scores and partial results are what L2 should keep
        asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(policy));
        uint32_t issued = 0;                                    // lane x: blocks of stream x asked for
        uint32_t slot = 0, phase = 1;                           // phase of `empty` that block k waits for; the first round waits for nothing
        bool ok = true;
        for (uint32_t k0 = 0; k0 < n_max && ok; k0 += 4) {
            look_up(id_next, live_next);
#pragma unroll
            for (int u = 0; u < 4; u++) {
                if (k0 + u < n_max && ok) {
                    for (uint32_t x = 0; x < a.streams; x++) {
                        const uint32_t entry = __shfl_sync(0xFFFFFFFFu, id[u], x), rows = __shfl_sync(0xFFFFFFFFu, live[u], x);
                        const uint32_t hg = __shfl_sync(0xFFFFFFFFu, hg_l, x);
                        if (rows == 0 || !ok) continue;         // this stream has ended
                        if (k0 + u >= a.stages) ok = bar_wait(smem_addr(&empty[x][slot]), phase, &fail);
                        ok = __all_sync(0xFFFFFFFFu, ok);
                        if (!ok) continue;
                        const uint32_t bytes = min(a.heads, a.n_kv_heads - hg * a.heads) * S::ROW, bar = smem_addr(&full[x][slot]);
                        if (lane == 0)
                            asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(2u * rows * bytes) : "memory");
                        __syncwarp();
                        const uint32_t block = checked(entry);
                        if (lane == x) issued++;
                        const uint32_t stage = (x * a.stages + slot) * stage_bytes;
                        if (FP8 && a.k_scales) {                // 4-byte copies that arrive on the same barrier
                            const uint32_t head = hg * a.heads + row;
                            if (row < a.heads && head < a.n_kv_heads)
                                asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_addr(ring) + stage + 2 * plane + ((lane >> 4) * WARPS + row) * 4),
                                             "l"(((lane >> 4) ? a.v_scales : a.k_scales) + (size_t)block * a.n_kv_heads + head) : "memory");
                            asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
                        }
                        if (copies && row < rows)
                            asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1], %2, [%3], %4;"
                                         ::"r"(dst0 + stage),
                                         "l"(base + (uint64_t)block * a.block_stride + (size_t)hg * a.heads * S::ROW), "r"(bytes * min(per_copy, rows - row)),
                                         "r"(bar), "l"(policy) : "memory");
                    }
                    if (++slot == a.stages) {
                        slot = 0;
                        phase ^= 1u;
                    }
                }
            }
#pragma unroll
            for (int u = 0; u < 4; u++) {
                id[u] = id_next[u];
                live[u] = live_next[u];
            }
        }
        if (!ok && lane == 0) {
            atomicCAS(&fail, 0u, 4u);
            report(a.status, 4u);
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
        // Whatever happens to the consumers, no copy is in flight when the CTA's shared memory goes: the last copy into every stage is waited for.
        for (uint32_t x = 0; x < a.streams; x++) {
            const uint32_t n = __shfl_sync(0xFFFFFFFFu, issued, x);
            for (uint32_t k = n > a.stages ? n - a.stages : 0u; k < n; k++)
                for (uint32_t it = 0; it < (1u << 17); it++)
                    if (bar_test(smem_addr(&full[x][k % a.stages]), (k / a.stages) & 1u)) break;
        }
        // Launched beside the kernel before it (shared-prefix attention), this grid ends after that one: whoever waits for this grid has both.
        asm volatile("griddepcontrol.wait;" ::: "memory");
        return;
    }

    // ---- consumer: one kv head of one stream ----
    const uint32_t x_stream = warp / a.heads, h = warp % a.heads, stream = blockIdx.x * a.streams + x_stream;
    const uint32_t part = stream / a.head_groups, kvh = (stream % a.head_groups) * a.heads + h;
    if (x_stream >= a.streams || kvh >= a.n_kv_heads) return;
    const uint32_t n_mine = part_blocks(part);
    if (n_mine == 0) return;
    const uint32_t grp = lane >> 2, j = lane & 3u;
    Cursor c = part_start(part, n_mine);
    const uint32_t run_k = (grp & 1u) ? (grp >> 1) ^ 2u : grp >> 1, tok_k = 4 * run_k + (grp & 1u);   // tokens of MMA rows grp, grp + 8: tok_k, tok_k + 2
    const uint32_t tok_v0 = 4 * j, tok_v1 = 4 * (j ^ 2u) + 1;   // of k indices 2j, 2j + 1; of 2j + 8, 2j + 9: two more

    const bool scaled = FP8 && a.k_scales != nullptr;
    uint32_t slot = 0, phase = 0;                               // ring stage of the next block
    const uint32_t ring_base = smem_addr(ring) + x_stream * a.stages * stage_bytes;
    const uint32_t k_off = ring_base + h * S::ROW + run_k * run_smem + (grp & 1u) * row_smem + j * 16, half = 2 * row_smem;
    const uint32_t v_off = ring_base + plane + h * S::ROW + grp * S::VPB;
    const uint32_t v_at0 = v_off + j * run_smem, v_at1 = v_off + (j ^ 2u) * run_smem + row_smem;
    const uint32_t sc_off = ring_base + 2 * plane + 4 * h;
    const bool col0 = 2 * j < a.group, col1 = 2 * j + 1 < a.group;

    for (;;) {                                                  // the sequences of this part
        uint32_t q_hi[KS][2], q_lo[F32 ? KS : 1][2];
        {
            const uint32_t head = WIDE ? grp : (grp & 3u);      // columns 4..7 repeat heads 0..3 where the spare columns carry second terms
            const bool in = head < a.group;
            const size_t at = ((size_t)c.seq * a.n_q_heads + kvh * a.group + (in ? head : 0u)) * D;
#pragma unroll
            for (int s = 0; s < KS; s++) {
                const int dim = FP8 ? (4 * (s >> 2) + (int)j) * 16 + (s & 3) * 4 : (4 * (s >> 1) + (int)j) * 8 + (s & 1) * 4;
                if (F32) {
                    const float4 v = in ? *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(a.q) + at + dim) : make_float4(0, 0, 0, 0);
                    const __half2 h0 = __floats2half2_rn(v.x, v.y), h1 = __floats2half2_rn(v.z, v.w);
                    const float2 f0 = __half22float2(h0), f1 = __half22float2(h1);
                    q_hi[s][0] = h2_bits(h0);
                    q_hi[s][1] = h2_bits(h1);
                    q_lo[F32 ? s : 0][0] = h2_bits(__floats2half2_rn(v.x - f0.x, v.y - f0.y));
                    q_lo[F32 ? s : 0][1] = h2_bits(__floats2half2_rn(v.z - f1.x, v.w - f1.y));
                } else {
                    const uint2 v = in ? *reinterpret_cast<const uint2*>(reinterpret_cast<const __half*>(a.q) + at + dim) : make_uint2(0, 0);
                    q_hi[s][0] = v.x;
                    q_hi[s][1] = v.y;
                }
            }
        }
        float o[MT][4], m2[2] = {-INFINITY, -INFINITY}, l2[2] = {0.0f, 0.0f};   // o[t]: dims 2t, 2t + 1 of this lane's run, columns 2j, 2j + 1
#pragma unroll
        for (int t = 0; t < MT; t++) o[t][0] = o[t][1] = o[t][2] = o[t][3] = 0.0f;
        float unit[2] = {scaled ? UNIT_MOST : 1.0f, scaled ? UNIT_MOST : 1.0f};   // O is in units of 1 / unit
        float* lg = a.logits ? a.logits + ((size_t)c.seq * a.n_q_heads + kvh * a.group + 2 * j) * a.logit_stride + c.block * BS + tok_k : nullptr;
        const uint32_t n = c.left;
        for (uint32_t turn = 0; turn < n; turn++) {
            if (!bar_wait(smem_addr(&full[x_stream][slot]), phase, &fail)) {
                if (lane == 0) {
                    atomicCAS(&fail, 0u, 4u);
                    report(a.status, 4u);
                }
                return;
            }
            __syncwarp();
            const uint32_t stage = slot * stage_bytes;
            const uint32_t live = min((uint32_t)BS, c.len - (c.block + turn) * BS);

            // scores
            float even[4] = {0.0f, 0.0f, 0.0f, 0.0f}, odd[4] = {0.0f, 0.0f, 0.0f, 0.0f};   // two chains
#pragma unroll
            for (int i = 0; i < S::KP; i++) {
                uint32_t wl[4], wh[4];
                shared_read16(stage + k_off + i * 64, wl);
                shared_read16(stage + k_off + half + i * 64, wh);
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
                        a0 = wl[2 * (u & 1)];
                        a2 = wl[2 * (u & 1) + 1];
                        a1 = wh[2 * (u & 1)];
                        a3 = wh[2 * (u & 1) + 1];
                    }
                    mma16816((u & 1) ? odd : even, a0, a1, a2, a3, q_hi[s][0], q_hi[s][1]);
                    if (F32) mma16816((u & 1) ? odd : even, a0, a1, a2, a3, q_lo[F32 ? s : 0][0], q_lo[F32 ? s : 0][1]);
                }
            }
            float ks = a.scale_log2, vs = 1.0f;
            if (scaled) {
                ks *= shared_read4(stage + sc_off);
                vs = shared_read4(stage + sc_off + 4 * WARPS);
            }
            float x[4];                                         // x[2 * (token half) + column]
#pragma unroll
            for (int i = 0; i < 4; i++) x[i] = (even[i] + odd[i]) * ks;
            if (live < (uint32_t)BS) {
#pragma unroll
                for (int i = 0; i < 4; i++) x[i] = tok_k + 2 * (i >> 1) < live ? x[i] : -INFINITY;
            }
            if (lg) {
                float* at = lg + turn * BS;
                const bool lo = tok_k < live, hi = tok_k + 2 < live;
                if (col0 && lo) at[0] = x[0];
                if (col0 && hi) at[2] = x[2];
                at += a.logit_stride;
                if (col1 && lo) at[0] = x[1];
                if (col1 && hi) at[2] = x[3];
            }
            // the references in use are raised, for all lanes together, once a score (or a score and its V scale) is too far above
            float room[2] = {RAISE, RAISE}, vs_log2 = 0.0f;
            if (FP8 && scaled) {
                vs_log2 = log2_fast(fabsf(vs));
                room[0] -= fmaxf(vs_log2 + log2_of_power(unit[0]), 0.0f);
                room[1] -= fmaxf(vs_log2 + log2_of_power(unit[1]), 0.0f);
            }
            const bool over = fmaxf(x[0], x[2]) > m2[0] + room[0] || fmaxf(x[1], x[3]) > m2[1] + room[1];
            if (__any_sync(0xFFFFFFFFu, over)) {
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    float mx = fmaxf(x[e], x[2 + e]);
                    mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, 4));
                    mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, 8));
                    mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, 16));
                    const float m_new = fmaxf(m2[e], mx - HEAD);
                    const float up = m_new - m2[e];
                    float keep = m2[e] == -INFINITY ? 0.0f : exp2_fast(-up);
                    m2[e] = m_new;
                    l2[e] *= keep;
                    if (FP8 && scaled) {
                        const float u = next_unit(unit[e], up, mx == -INFINITY ? mx : mx - m_new + vs_log2);
                        keep *= u * inverse_of_power(unit[e]);
                        unit[e] = u;
                    }
#pragma unroll
                    for (int t = 0; t < MT; t++) {
                        o[t][e] *= keep;
                        o[t][2 + e] *= keep;
                    }
                }
            }
            const float sub0 = m2[0] == -INFINITY ? 0.0f : m2[0], sub1 = m2[1] == -INFINITY ? 0.0f : m2[1];
            // probabilities, and O += V^T P
            float p[4];
            p[0] = exp2_fast(x[0] - sub0);
            p[1] = exp2_fast(x[1] - sub1);
            p[2] = exp2_fast(x[2] - sub0);
            p[3] = exp2_fast(x[3] - sub1);
            l2[0] += p[0] + p[2];
            l2[1] += p[1] + p[3];
            if (FP8 && scaled) {
                const float vn[2] = {vs * unit[0], vs * unit[1]};
#pragma unroll
                for (int i = 0; i < 4; i++) p[i] *= vn[i & 1];
            }
            __half2 pl = __floats2half2_rn(p[0], p[1]), ph = __floats2half2_rn(p[2], p[3]);
            const float2 fl = __half22float2(pl), fh = __half22float2(ph);
            const __half2 rl = __floats2half2_rn(p[0] - fl.x, p[1] - fl.y), rh = __floats2half2_rn(p[2] - fh.x, p[3] - fh.y);
            if (!WIDE && j >= 2) {                              // columns 4..7: the second terms of heads 0..3
                pl = rl;
                ph = rh;
            }
            const uint32_t b0 = transpose8(h2_bits(pl)), b1 = transpose8(h2_bits(ph));   // rows: k indices 2j, 2j + 1 (+ 8); column grp
            uint32_t c0 = 0, c1 = 0;
            if (WIDE) {
                c0 = transpose8(h2_bits(rl));
                c1 = transpose8(h2_bits(rh));
            }
#pragma unroll
            for (int pc = 0; pc < S::VP; pc++) {
                uint32_t w[4][4];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const uint32_t at = stage + ((i & 1) ? v_at1 : v_at0) + (i >> 1) * half + pc * 128;
                    if (S::VPB == 16) shared_read16(at, w[i]);
                    else shared_read8(at, w[i]);
                }
                if (live < (uint32_t)BS) {                      // rows that were not copied hold an older block's bytes: 0 x NaN must not reach O
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const uint32_t tok = ((i & 1) ? tok_v1 : tok_v0) + 2 * (i >> 1);
#pragma unroll
                        for (int e = 0; e < S::VPB / 4; e++) w[i][e] = tok < live ? w[i][e] : 0u;
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
                    if (WIDE) mma16816(o[pc * TILES + t], a0, a1, a2, a3, c0, c1);
                }
            }
            __syncwarp();                                       // every lane's reads of the stage are done
            if (lane == 0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_addr(&empty[x_stream][slot])) : "memory");
            if (++slot == a.stages) {
                slot = 0;
                phase ^= 1u;
            }
        }

        // ---- partial results of (part, sequence) ----
        const size_t at_slot = (size_t)part + c.seq;
        if (!WIDE) {                                            // first and second terms of a head together
#pragma unroll
            for (int t = 0; t < MT; t++)
#pragma unroll
                for (int i = 0; i < 4; i++) o[t][i] += __shfl_xor_sync(0xFFFFFFFFu, o[t][i], 2);
        }
#pragma unroll
        for (int e = 0; e < 2; e++) {
            float l = l2[e];
            l += __shfl_xor_sync(0xFFFFFFFFu, l, 4);
            l += __shfl_xor_sync(0xFFFFFFFFu, l, 8);
            l += __shfl_xor_sync(0xFFFFFFFFu, l, 16);
            const uint32_t head = 2 * j + e;
            const float inv_unit = inverse_of_power(unit[e]);
            if (head < a.group) {
                const size_t row = at_slot * a.n_q_heads + kvh * a.group + head;
                if (grp == 0) *reinterpret_cast<float2*>(a.part_ml + row * 2) = make_float2(m2[e], l);
                float* dst = a.part_o + row * D;
#pragma unroll
                for (int t = 0; t < MT; t++) {
                    constexpr int RUN = S::VPB / S::ES;         // dims of a piece
                    const int i = 2 * t, dim = (i / RUN) * (8 * RUN) + (int)grp * RUN + i % RUN;
                    *reinterpret_cast<float2*>(dst + dim) = make_float2(o[t][e] * inv_unit, o[t][2 + e] * inv_unit);
                }
            }
        }
        if (!c.rest) break;
        next_sequence(c);
    }
}

// ---- host side -------------------------------------------------------------------------------------------------------------
struct Split {
    uint32_t heads, streams, head_groups;    // of a stream, of a CTA, of a part
    uint32_t parts, min_share, grid;
};
// Streams of at most eight kv heads, as even as they come; parts for a batch of at most `blocks` cached blocks: one CTA per SM, and no
// part shorter than MIN_SHARE blocks (a part costs the joining kernel a partial result per query head; scored attention of one sequence of 200 tokens:
// 12.3 us with 2, 14.3 with 4, 16.4 with 8, and no difference for batches that fill the machine).
constexpr uint32_t MIN_SHARE = 2;
inline Split split_for(uint64_t blocks, uint32_t n_kv_heads, uint32_t ctas) {
    Split s;
    s.head_groups = (n_kv_heads + WARPS - 1) / WARPS;
    s.heads = (n_kv_heads + s.head_groups - 1) / s.head_groups;
    s.head_groups = (n_kv_heads + s.heads - 1) / s.heads;
    s.streams = WARPS / s.heads;
    s.min_share = MIN_SHARE;
    const uint64_t most = (uint64_t)ctas * s.streams / s.head_groups, want = (blocks + MIN_SHARE - 1) / MIN_SHARE;
    s.parts = (uint32_t)(most < 1 ? 1 : want < 1 ? 1 : want < most ? want : most);
    s.grid = (uint32_t)(((uint64_t)s.parts * s.head_groups + s.streams - 1) / s.streams);
    return s;
}

// beside: the launch does not wait for the kernel before it on the stream, which has to be one that this one does not read from
template <int D, bool FP8, bool F32, bool WIDE> cudaError_t launch_one(Args a, const Split& sp, bool beside, cudaStream_t st) {
    using S = Shape<D, FP8>;
    a.heads = sp.heads;
    a.streams = sp.streams;
    a.head_groups = sp.head_groups;
    a.parts = sp.parts;
    a.min_share = sp.min_share;
    const uint32_t stage = 2 * (BS * sp.heads * S::ROW + 4 * PAD) + (FP8 ? SCALE_BYTES : 0), fit = RING_BYTES / (sp.streams * stage);
    a.stages = fit < (uint32_t)MAX_STAGES ? fit : (uint32_t)MAX_STAGES;   // at least 3 (eight heads of 128 F16 dims: 65 KB each)
    const size_t smem = (size_t)sp.streams * a.stages * stage;
    auto kernel = rows_attn<D, FP8, F32, WIDE>;
    static std::atomic<uint64_t> granted{0};                    // devices on which this kernel may use the ring's shared memory
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    const uint64_t bit = dev < 64 ? 1ull << dev : 0ull;
    if (!(granted.load(std::memory_order_relaxed) & bit)) {
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)RING_BYTES);
        if (e != cudaSuccess) return e;
        granted.fetch_or(bit, std::memory_order_relaxed);
    }
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(sp.grid);
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = beside ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kernel, a);
}
template <int D, bool FP8> cudaError_t launch_type(bool f32, const Args& a, const Split& sp, bool beside, cudaStream_t st) {
    const bool wide = a.group > 4;
    if (f32) return wide ? launch_one<D, FP8, true, true>(a, sp, beside, st) : launch_one<D, FP8, true, false>(a, sp, beside, st);
    return wide ? launch_one<D, FP8, false, true>(a, sp, beside, st) : launch_one<D, FP8, false, false>(a, sp, beside, st);
}
inline cudaError_t launch_rows(uint32_t head_dim, bool fp8, bool f32, const Args& a, const Split& sp, bool beside, cudaStream_t st) {
    if (head_dim == 128) return fp8 ? launch_type<128, true>(f32, a, sp, beside, st) : launch_type<128, false>(f32, a, sp, beside, st);
    return fp8 ? launch_type<64, true>(f32, a, sp, beside, st) : launch_type<64, false>(f32, a, sp, beside, st);
}

}  // namespace tkv_rows
