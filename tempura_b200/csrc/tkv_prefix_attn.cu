// Decode attention of a batch whose sequences share prefixes: the shared tokens of a group are attended to once for all its members.
//
// Over the prefix every (member, query head) of a group and kv head is one row of a matrix product, so
//
//     S[rows][128 tokens] = Q . K_tile^T,   P = 2^(scale * S - m),   O[rows][dims] += P . V_tile
//
// runs on the fifth-generation tensor cores (tcgen05, accumulators in tensor memory) and K and V of the prefix are read once
// per group instead of once per sequence.  The tokens behind the prefix go through rows_attn, and a third kernel joins the partial
// results (m, l, O) of both: out = sum 2^(m_i - M) O_i / sum 2^(m_i - M) l_i.
//
// A CTA works on up to 256 rows of one (group, kv head) as two streams of 128 with their own S, P and O that read the same cached tiles; with
// up to 128 rows the second stream issues nothing.  (Letting both streams take the same rows on halves of every tile doubles the partial results:
// 30 sequences on 2 048 tokens 38 us against 33, 16 on 8 192 45 against 36, 8 on 16 384 of an E4M3 pool 55 against 44; only with many tiles per
// CTA it is ahead: 45 in 7 groups, E4M3, 86 against 91.)  A stream goes 64 cached tokens at a time through two S buffers: the scores of the next
// step are there when the softmax of this one ends.  (One buffer of 128 tokens per stream left the softmax warps waiting for two products per
// tile: 4 800 cycles per tile of both streams.)  A softmax thread owns a row: no exchange between threads.  P goes back to tensor memory, over
// the S it was made from, as the A operand of the second product, so shared memory holds Q and the K and V tiles only.  The row maximum in use
// is raised, and O rescaled, only when a score is 14 above a reference that lies 8 below the maximum it was set from.
// Measured: 128 sequences on 16 384 tokens, 64 query heads: 131 us for the call, 529 TFLOP/s of useful products (0.32 of the measured bf16 rate; with
// the second terms counted 0.48).  A step of 64 tokens takes both streams some 2 100 cycles, of which the products are 1 790 (N = 64 from shared
// memory 48 cycles each, with A in tensor memory 64) and the rest hand-offs between softmax and issuers.
// An F16 pool's tiles arrive as tensor-map boxes, in the 128-byte swizzle the MMA reads.  An E4M3 pool's tiles are widened to F16
// on the way by four warps (exact); K's block scale multiplies the scores, V's the probabilities, in units of a power of two per row that goes by
// the largest probability times scale met so far (tkv_rows_attn.cuh).  Both operands of both products are then F16 and the products exact.  A
// probability is two F16 terms (22 bits), the second with products of its own: 0.21e-3 off 64 bits, which is the rounding of the output alone, against 0.29e-3
// with one term.  That costs 118 -> 131 us on that case and nothing where the products are not the bound.
//
// Work split: the cached tiles of all (group, kv head, row block) items, one after another, in equal shares, one per CTA; a share may
// begin and end inside an item.  The partial rows of item i and share c start at (rows before item i) + 256 * c, which keeps them
// apart because both only grow along the work.
#include <cuda.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstdio>
#include <stdint.h>
#include <type_traits>

#include "../../include/tkv.h"
#include "tkv_rows_attn.cuh"
#include "tkv_tc_common.cuh"

namespace tkv_internal {
int32_t set_error(int32_t code, int32_t cuda_code, const char* text);
}

namespace {

using namespace tkv_tc;
using tkv_rows::bar_wait;

constexpr uint32_t CTAS = 148;               // one per SM of the part this is built for; partial results are sized by it
constexpr int BS = 16, KT = 128, ST = 64;    // tokens of a block, of a cached tile, of a step
constexpr int GROUP_BYTES = 128 * 128;       // a [128 rows][128 B] swizzled column group of an operand tile
using tkv_rows::HEAD;
using tkv_rows::RAISE;
// Cached tiles of a share: at least two where there are shares for more than half of the SMs, so that the kernel for the tokens behind the prefix
// finds SMs beside this one (64 sequences on 2 048 tokens: 41 us with 2, 53 with 1), else one (3 on 48: 14 us, 18 with 2).
__host__ __device__ __forceinline__ uint32_t min_share(uint64_t tiles) { return 2 * tiles > CTAS ? 2u : 1u; }

struct Args {
    const uint32_t *tables, *kv_lens, *group_starts, *prefix_lens;
    const __half* q;
    const char *k8, *v8;                     // layer tensors of an E4M3 pool
    const float *k_scales, *v_scales;
    float *part_o, *part_ml;                 // [row][D], [row][2]
    uint32_t *plan, *status;                 // [0] cached tiles per share, [1 + g] tiles before group g (n_groups + 1 entries)
    uint64_t block_stride;
    uint32_t row_stride, n_seqs, n_groups, n_q_heads, n_kv_heads, group, table_stride, max_kv_len, max_prefix_len, total_blocks, parts;
    uint32_t q_sign;                         // 0x80008000 for a negative scale: its sign is moved to q
    float scale_log2;                        // not negative
};

__host__ __device__ constexpr int softmax_warps() { return 8; }
__host__ __device__ constexpr int feed_warps(bool fp8) { return fp8 ? 4 : 1; }
__host__ __device__ constexpr int threads_of(bool fp8) { return (softmax_warps() + feed_warps(fp8) + 2) * 32; }   // and an MMA issuer per stream

struct Control {
    uint64_t k_full[2], k_empty[2], v_full[2], v_empty[2];
    uint64_t q_ready[2], s_full[2][2], p_full[2][2], pv_done[2][2], drained[2];   // [stream][S buffer]
    uint32_t tmem, fail;
    float scales[4][24];                     // per cached tile (mod 4): of its 8 blocks K scale x scale_log2, V scale, log2 of V scale
};
constexpr uint32_t CTRL_BYTES = 1024;
static_assert(sizeof(Control) <= CTRL_BYTES, "control block");

// one tile of one item
struct Item {
    uint32_t first_seq, rows, row0, block_rows;   // of the group: first sequence, rows; of the row block: first row, rows (at most 256)
    uint32_t kvh, prefix, tile, n_tiles;          // tiles [tile, tile + n_tiles) of the prefix
    uint64_t out_row;                             // first partial row
};
__device__ __forceinline__ uint32_t row_blocks(uint32_t rows) { return (rows + 255) / 256; }

__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) { mma<false>(d, a, b, idesc, acc); }
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t* r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};"
                 ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]) : "memory");
}
__device__ __forceinline__ bool elect_one() {
    uint32_t yes;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xFFFFFFFF;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(yes));
    return yes != 0;
}
// A operand from tensor memory: lane = row, two F16 of the row per column
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a_tmem, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
                 ::"r"(d), "r"(a_tmem), "l"(b), "r"(idesc), "r"(acc) : "memory");
}

template <int D, bool FP8>
__global__ void __launch_bounds__(threads_of(FP8), 1)
prefix_attn_tc(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const Args a) {
    constexpr int NCG = D / 64;                                 // column groups of 64 F16 dims
    constexpr int TILE = NCG * GROUP_BYTES;                     // Q, K or V tile of 128 rows
    constexpr int KSTEPS = D / 16;
    constexpr int THREADS = threads_of(FP8), SM = softmax_warps(), FEED = feed_warps(FP8);
    constexpr uint32_t IDESC_QK = instr_desc2(0u, 0u, 0u, 0u, (uint32_t)ST), IDESC_PV = instr_desc2(0u, 0u, 0u, 1u, (uint32_t)D);   // B = V, MN-major
    constexpr uint64_t DESC_HI = ((uint64_t)(1024u >> 4) << 32) | (1ull << 46) | (2ull << 61);
    constexpr uint64_t DESC_K = DESC_HI | ((uint64_t)1u << 16);
    constexpr uint64_t DESC_V = DESC_HI | ((uint64_t)(GROUP_BYTES >> 4) << 16);        // the second 64 dims one column group further
    constexpr uint32_t TM_S = 0, TM_O = 256;                    // tensor memory columns: S (and P over it) of stream x, buffer b at 128 x + 64 b, O at 256 + 128 x

    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u;
    extern __shared__ __align__(1024) unsigned char smem[];
    Control* c = reinterpret_cast<Control*>(smem);
    unsigned char* q_tile = smem + CTRL_BYTES;                  // two
    unsigned char* k_ring = q_tile + 2 * TILE;                  // two
    unsigned char* v_ring = k_ring + 2 * TILE;                  // two
    const volatile uint32_t* fail = &c->fail;
    uint32_t* cum = reinterpret_cast<uint32_t*>(q_tile);        // [THREADS + 1], until the first item
    uint32_t* warp_sum = cum + THREADS + 1;                     // [THREADS / 32]

    if (__syncthreads_or(tkv_rows::groups_bad(a.group_starts, a.prefix_lens, a.n_groups, a.n_seqs, a.max_prefix_len, tid, THREADS))) {
        if (tid == 0) {
            tkv_rows::report(a.status, 2u);
            if (blockIdx.x == 0) a.plan[0] = 0;                 // nothing was computed
        }
        return;
    }
    // ---- cached tiles before every run of `per` groups ----
    auto tiles_of = [&](uint32_t g) -> uint32_t {               // a group's tiles times its (kv head, row block) items
        const uint32_t rows = (a.group_starts[g + 1] - a.group_starts[g]) * a.group;
        return row_blocks(rows) * a.n_kv_heads * ((a.prefix_lens[g] + KT - 1) / KT);
    };
    const uint32_t per = (a.n_groups + THREADS - 1) / THREADS;
    uint32_t mine = 0;
    for (uint32_t i = 0; i < per; i++)
        if (tid * per + i < a.n_groups) mine += tiles_of(tid * per + i);
    uint32_t incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t v = __shfl_up_sync(0xFFFFFFFFu, incl, o);
        if (lane >= (uint32_t)o) incl += v;
    }
    if (lane == 31) warp_sum[warp] = incl;
    if (tid == 0) {
        for (int i = 0; i < 2; i++) {
            mbar_init(c->k_full + i, FP8 ? FEED : 1);
            mbar_init(c->v_full + i, FP8 ? FEED : 1);
            mbar_init(c->k_empty + i, 2);
            mbar_init(c->v_empty + i, 2);
            mbar_init(c->q_ready + i, SM / 2);
            for (int b = 0; b < 2; b++) {
                mbar_init(&c->s_full[i][b], 1);
                mbar_init(&c->p_full[i][b], SM / 2);
                mbar_init(&c->pv_done[i][b], 1);
            }
        }
        mbar_init(c->drained, 1);
        mbar_init(c->drained + 1, 1);
        c->fail = (smem_u32(smem) & 1023u) ? 2u : 0u;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    uint32_t before = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 32; w++) before += w < (int)warp ? warp_sum[w] : 0u;
    cum[tid] = before + incl - mine;
    if (tid == THREADS - 1) cum[THREADS] = before + incl;
    __syncthreads();
    const uint32_t total = cum[THREADS], share = max((total + a.parts - 1) / a.parts, min_share(total));
    if (blockIdx.x == 0) {
        uint32_t at = cum[tid];
        for (uint32_t i = 0; i < per; i++)
            if (tid * per + i < a.n_groups) {
                a.plan[1 + tid * per + i] = at;
                at += tiles_of(tid * per + i);
            }
        if (tid == 0) {
            a.plan[0] = share;
            a.plan[1 + a.n_groups] = total;
        }
    }
    asm volatile("griddepcontrol.launch_dependents;");          // the kernel for the tokens behind the prefixes may start where SMs are free
    if ((uint64_t)blockIdx.x * share >= total) return;
    const uint32_t u_begin = blockIdx.x * share, u_end = min(total, u_begin + share);

    if (warp == SM + FEED) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&c->tmem)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = 0;                                    // all 512 columns are this CTA's: they begin at 0
    if (tid == 0 && c->tmem != 0) c->fail = 2u;

    // ---- the group of the first tile ----
    uint32_t g, at;                                             // tiles before group g
    {
        uint32_t lo = 0, hi = THREADS;                          // cum[lo] <= u_begin < cum[hi]
        while (hi - lo > 1) {
            const uint32_t mid = (lo + hi) >> 1;
            if (cum[mid] <= u_begin) lo = mid;
            else hi = mid;
        }
        g = lo * per;
        at = cum[lo];
    }
    __syncthreads();                                            // Q goes where the sums were
    uint32_t tiles_done = 0;                                    // cached tiles of this CTA before the item at hand: places in the rings
    uint32_t n_steps = 0;                                       // steps of each stream before the item at hand: phases of its barriers
    uint32_t issued[2] = {0, 0};                                // F16 producer: tiles of K, of V asked for
    bool ok = true;
    for (uint32_t u = u_begin, item_no = 0; u < u_end; item_no++) {
        while (at + tiles_of(g) <= u) at += tiles_of(g++);
        Item it;
        {
            it.first_seq = a.group_starts[g];
            it.rows = (a.group_starts[g + 1] - it.first_seq) * a.group;
            it.prefix = a.prefix_lens[g];
            const uint32_t nt = (it.prefix + KT - 1) / KT, rbs = row_blocks(it.rows), item = (u - at) / nt;
            it.kvh = item / rbs;
            it.row0 = (item % rbs) * 256;
            it.block_rows = min(256u, it.rows - it.row0);
            it.tile = (u - at) % nt;
            it.n_tiles = min(nt - it.tile, u_end - u);
            it.out_row = (uint64_t)(it.first_seq - a.group_starts[0]) * a.group * a.n_kv_heads + (uint64_t)it.kvh * it.rows + it.row0 + 256ull * blockIdx.x;
        }
        const bool few = it.block_rows <= 128;                  // nothing for the second stream
        const uint32_t* table = a.tables + (size_t)it.first_seq * a.table_stride;
        const uint32_t n_blocks = it.prefix / BS;
        auto blocks_in = [&](uint32_t i) { return min(8u, n_blocks - (it.tile + i) * 8u); };   // of the item's i-th tile
        auto steps_in = [&](uint32_t i) { return blocks_in(i) > 4u ? 2u : 1u; };

        if (warp >= SM + FEED) {
            // ---- MMA issuers, a warp per stream.  Waits sleep in hardware (a polling issuer took issue slots from the softmax warps of its
            // scheduler and held the tile up by 1 000 cycles), and the warp issues together through an elected lane.  The scores run two
            // steps ahead of the second product. ----
            // Broadcast from one lane, what selects operands is known to be the warp's own: addresses then are computed once per warp.
            auto uni = [](uint32_t v) { return __shfl_sync(0xFFFFFFFFu, v, 0); };
            const uint32_t x = uni(warp - (SM + FEED)), s_x = uni(n_steps), n_t = uni(it.n_tiles);
            const uint32_t done = uni(tiles_done), n_left = uni(n_blocks - it.tile * 8u);
            const bool idle = uni(few ? 1u : 0u) != 0 && x != 0;   // a stream without rows
            auto blocks_at = [&](uint32_t i) { return min(8u, n_left - i * 8u); };
            const uint32_t q_lo = (smem_u32(q_tile) >> 4) + x * (TILE >> 4), k_lo = smem_u32(k_ring) >> 4, v_lo = smem_u32(v_ring) >> 4;
            const uint32_t ts = TM_S + x * 128, to = TM_O + x * 128;
            auto wait = [&](uint64_t* bar, uint32_t parity) {
                if (ok) ok = bar_wait(smem_u32(bar), parity & 1u, fail);
            };
            if (elect_one()) {
            wait(c->q_ready + x, item_no);
            auto steps_at = [&](uint32_t i) { return blocks_at(i) > 4u ? 2u : 1u; };
            uint32_t iq = 0, hq = 0, nq = s_x;                   // tile, step in it and number of the next scores
            uint32_t ip = 0, hp = 0, np = s_x;                   // of the next product
            while (ok && ip < n_t) {
                // The scores run up to two steps ahead, but a tile that is not there yet holds up no product: that would hold up its V's place, too.
                const uint32_t tq = done + iq, sq = tq & 1u;
                bool ahead = iq < n_t && nq - np < 2;
                if (ahead && hq == 0) {
                    if (np == nq) wait(c->k_full + sq, tq >> 1);
                    else ahead = mbar_test(c->k_full + sq, (tq >> 1) & 1u);
                }
                if (ahead) {
                    const uint32_t b = nq & 1u;
                    if (nq >= 2) wait(&c->pv_done[x][b], (nq >> 1) - 1u);  // the buffer is free when the product that read P over it is done
                    if (!ok) break;
                    tc_fence_after();
                    const bool last = hq + 1 == steps_at(iq);
                    if (!idle) {
#pragma unroll
                        for (int ks = 0; ks < KSTEPS; ks++) {
                            const uint32_t off = (ks / 4) * (GROUP_BYTES >> 4) + (ks % 4) * 2;
                            mma_ss(ts + b * ST, DESC_K | (q_lo + off), DESC_K | (k_lo + sq * (TILE >> 4) + hq * (ST * 128u >> 4) + off), IDESC_QK, ks > 0 ? 1u : 0u);
                        }
                    }
                    tc_commit(&c->s_full[x][b]);
                    if (last) tc_commit(c->k_empty + sq);                  // a tile goes back when both streams have read it
                    nq++;
                    hq = last ? 0 : 1;
                    iq += last ? 1 : 0;
                } else {
                    const uint32_t t = done + ip, st = t & 1u, b = np & 1u, nb = min(4u, blocks_at(ip) - 4u * hp);
                    wait(&c->p_full[x][b], np >> 1);
                    if (hp == 0) wait(c->v_full + st, t >> 1);
                    if (!ok) break;
                    tc_fence_after();
                    const bool last = hp + 1 == steps_at(ip);
                    if (!idle) {
                        const uint64_t v_desc = DESC_V | (v_lo + st * (TILE >> 4) + 4 * hp * (2048u >> 4));
#pragma unroll
                        for (uint32_t ks = 0; ks < 4; ks++)                // a block is one k-step: blocks behind the prefix are left out
                            if (ks < nb) mma_ts(to, ts + b * ST + ks * 8, v_desc + ks * (2048u >> 4), IDESC_PV, (np > s_x || ks > 0) ? 1u : 0u);
#pragma unroll
                        for (uint32_t ks = 0; ks < 4; ks++)                // the second terms of the probabilities
                            if (ks < nb) mma_ts(to, ts + b * ST + 32 + ks * 8, v_desc + ks * (2048u >> 4), IDESC_PV, 1u);
                    }
                    tc_commit(&c->pv_done[x][b]);
                    if (last) tc_commit(c->v_empty + st);
                    np++;
                    hp = last ? 0 : 1;
                    ip += last ? 1 : 0;
                }
            }
            if (!ok) atomicCAS(&c->fail, 0u, 4u);
            }
            __syncwarp();
            ok = *fail == 0;
        } else if (warp >= SM) {
            if (!FP8) {
                // ---- producer: eight lanes, a block each ----
                for (uint32_t i = 0; i < it.n_tiles && ok; i++) {
                    const uint32_t t = tiles_done + i, st = t & 1u, nb = blocks_in(i);
                    uint32_t blk = 0;
                    if (lane < nb) blk = table[(it.tile + i) * 8u + lane];
                    if (__any_sync(0xFFFFFFFFu, blk >= a.total_blocks)) {          // a stale or foreign id is never turned into an address
                        if (lane == 0) atomicCAS(&c->fail, 0u, 2u);
                        ok = false;
                        break;
                    }
#pragma unroll
                    for (int kv = 0; kv < 2; kv++) {
                        uint64_t* full = (kv ? c->v_full : c->k_full) + st;
                        if (t >= 2) ok = __all_sync(0xFFFFFFFFu, bar_wait(smem_u32((kv ? c->v_empty : c->k_empty) + st), ((t >> 1) - 1u) & 1u, fail));
                        if (!ok) break;
                        issued[kv] = t + 1;
                        if (lane == 0) mbar_expect_tx(full, nb * BS * 128u * NCG);
                        __syncwarp();
                        if (lane < nb) {
                            const uint32_t dst = smem_u32((kv ? v_ring : k_ring) + st * TILE) + lane * (BS * 128u);
#pragma unroll
                            for (int cg = 0; cg < NCG; cg++)
                                tma_head_rows(dst + cg * GROUP_BYTES, kv ? &map_v : &map_k, cg * 128, (int32_t)it.kvh, (int32_t)(blk * BS), full);
                        }
                    }
                }
                if (!ok && lane == 0) atomicCAS(&c->fail, 0u, 4u);
            } else {
                // ---- widening: 128 threads, 16 bytes of a token at a time.  The bytes arrive a tile ahead by asynchronous copies; a thread copies
                // what it will widen, so its own wait is enough.  (In registers they did not fit beside the softmax's share of them.) ----
                constexpr int CPR = D / 16, PER = 128 * CPR / 128;             // 16-byte pieces of a row; per thread and tile
                const uint32_t t128 = tid - SM * 32;
                const uint32_t raw[2] = {smem_u32(v_ring + 2 * TILE) + t128 * 16, smem_u32(v_ring + 2 * TILE) + 128 * D + t128 * 16};
                // block ids a tile ahead of the copies that use them; an id outside the pool is remembered, without a branch that would wait
                uint32_t id[PER], sc_id = 0;
                bool foreign = false;
                float sc = 1.0f;
                auto look_up = [&](uint32_t i) {
                    const uint32_t nb = i < it.n_tiles ? blocks_in(i) : 0u;
#pragma unroll
                    for (int e = 0; e < PER; e++) {
                        const uint32_t b = (e * 128 + t128) / CPR / BS;
                        id[e] = b < nb ? table[(it.tile + i) * 8u + b] : ~0u;
                    }
                    sc_id = (t128 & 7u) < nb ? table[(it.tile + i) * 8u + (t128 & 7u)] : ~0u;
                };
                auto copy = [&](int kv, uint32_t i) {                          // nothing but the group's mark behind the item's last tile
                    if (i < it.n_tiles) {
                        const char* base = (kv ? a.v8 : a.k8) + (size_t)it.kvh * D;
                        const uint32_t nb = blocks_in(i);
#pragma unroll
                        for (int e = 0; e < PER; e++) {
                            const uint32_t n = e * 128 + t128, row = n / CPR, ch = n % CPR;   // a warp's pieces: whole rows
                            const bool in = id[e] < a.total_blocks;
                            foreign |= !in && row / BS < nb;
                            const char* src = base + (uint64_t)(in ? id[e] : 0u) * a.block_stride + (size_t)(row % BS) * a.row_stride + ch * 16;
                            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(raw[kv] + e * 2048u), "l"(src), "r"(in ? 16u : 0u) : "memory");
                        }
                    }
                    asm volatile("cp.async.commit_group;" ::: "memory");
                };
                auto load_scales = [&]() {
                    sc = 1.0f;
                    if (t128 < 16 && a.k_scales) sc = sc_id < a.total_blocks ? __ldg((t128 < 8 ? a.k_scales : a.v_scales) + (size_t)sc_id * a.n_kv_heads + it.kvh) : 0.0f;
                };
                auto widen = [&](unsigned char* tile, int kv) {
                    asm volatile("cp.async.wait_group 1;" ::: "memory");       // all but the other tensor's, asked for last
#pragma unroll
                    for (int e = 0; e < PER; e++) {
                        const uint32_t n = e * 128 + t128, row = n / CPR, ch = n % CPR;
                        uint32_t w[4], h[8];
                        tkv_rows::shared_read16(raw[kv] + e * 2048u, w);
#pragma unroll
                        for (int k = 0; k < 4; k++) {
                            h[2 * k] = tkv_rows::e4m3x2_h2(w[k] & 0xFFFFu);
                            h[2 * k + 1] = tkv_rows::e4m3x2_h2(w[k] >> 16);
                        }
                        unsigned char* base = tile + (ch / 4) * GROUP_BYTES;   // 16 dims = two 16-byte chunks of F16
                        *reinterpret_cast<uint4*>(base + swz(row, (ch % 4) * 2)) = make_uint4(h[0], h[1], h[2], h[3]);
                        *reinterpret_cast<uint4*>(base + swz(row, (ch % 4) * 2 + 1)) = make_uint4(h[4], h[5], h[6], h[7]);
                    }
                    fence_async_smem();
                    __syncwarp();
                };
                look_up(0);
                load_scales();
                copy(0, 0);
                copy(1, 0);
                look_up(1);
                for (uint32_t i = 0; i < it.n_tiles && ok; i++) {
                    const uint32_t t = tiles_done + i, st = t & 1u;
                    if (t >= 2) ok = __all_sync(0xFFFFFFFFu, bar_wait(smem_u32(c->k_empty + st), ((t >> 1) - 1u) & 1u, fail));
                    if (!ok) break;
                    if (t128 < 16) c->scales[t & 3u][t128] = t128 < 8 ? sc * a.scale_log2 : sc;
                    if (t128 >= 8 && t128 < 16) c->scales[t & 3u][t128 + 8] = fast_log2(fabsf(sc));
                    widen(k_ring + st * TILE, 0);
                    if (lane == 0) mbar_arrive(c->k_full + st);
                    load_scales();
                    copy(0, i + 1);
                    if (t >= 2) ok = __all_sync(0xFFFFFFFFu, bar_wait(smem_u32(c->v_empty + st), ((t >> 1) - 1u) & 1u, fail));
                    if (!ok) break;
                    widen(v_ring + st * TILE, 1);
                    if (lane == 0) mbar_arrive(c->v_full + st);
                    copy(1, i + 1);
                    look_up(i + 2);
                    if (*fail) ok = false;
                }
                asm volatile("cp.async.wait_all;" ::: "memory");
                if (foreign) atomicCAS(&c->fail, 0u, 2u);
                if (!ok && lane == 0) atomicCAS(&c->fail, 0u, 4u);
            }
        } else {
            // ---- softmax: one row per thread ----
            const uint32_t x = warp >> 2, s_x = n_steps, r = (warp & 3u) * 32u + lane;
            const uint32_t row = it.row0 + x * 128u + r;        // of the group and kv head
            const bool live = x * 128u + r < it.block_rows;
            const bool warp_live = __any_sync(0xFFFFFFFFu, live);
            const uint32_t seq = it.first_seq + (live ? row / a.group : 0u), head = it.kvh * a.group + (live ? row % a.group : 0u);
            const uint32_t limit = live && min(a.kv_lens[seq], a.max_kv_len) >= it.prefix ? it.prefix : 0u;   // shorter members: rows_attn
            {
                // Q rows of the warp, whole rows per load (a row per thread took 8 000 cycles)
                constexpr int CPR = D / 8, RPL = 32 / CPR;      // 16-byte chunks of a row; rows per load
                const uint32_t q_row = seq * a.n_q_heads + head, alive = __ballot_sync(0xFFFFFFFFu, live), ch = lane % CPR;
                unsigned char* qt = q_tile + x * TILE + (ch / 8) * GROUP_BYTES;
#pragma unroll
                for (int r0 = 0; r0 < 32; r0 += RPL) {
                    const uint32_t o = r0 + lane / CPR, from = __shfl_sync(0xFFFFFFFFu, q_row, o);
                    uint4 v = (alive >> o) & 1u ? __ldg(reinterpret_cast<const uint4*>(a.q + (size_t)from * D) + ch) : make_uint4(0, 0, 0, 0);
                    v = make_uint4(v.x ^ a.q_sign, v.y ^ a.q_sign, v.z ^ a.q_sign, v.w ^ a.q_sign);
                    *reinterpret_cast<uint4*>(qt + swz((warp & 3u) * 32u + o, ch % 8)) = v;
                }
                fence_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(c->q_ready + x);
            }
            const uint32_t lanes = ((warp & 3u) * 32u) << 16, ts = tmem + TM_S + x * 128 + lanes, to = tmem + TM_O + x * 128 + lanes;
            float m = -INFINITY, l = 0.0f, unit = FP8 ? tkv_rows::UNIT_MOST : 1.0f;   // O is in units of 1 / unit
            uint32_t n = s_x;                                   // steps of this stream so far
            for (uint32_t i = 0; i < it.n_tiles && ok; i++) {
                const uint32_t slot = (tiles_done + i) & 3u, h_end = steps_in(i);
                for (uint32_t h = 0; h < h_end; h++, n++) {
                    const uint32_t t0 = (it.tile + i) * KT + h * ST, b = n & 1u;
                    ok = __all_sync(0xFFFFFFFFu, bar_wait(smem_u32(&c->s_full[x][b]), (n >> 1) & 1u, fail));
                    if (!ok) break;
                    if (warp_live) {
                        tc_fence_after();
                        const int left = (int)min(limit > t0 ? limit - t0 : 0u, (uint32_t)ST);   // tokens of the step that the row attends to
                        const uint32_t tb = ts + b * ST;
                        const float* sc = c->scales[slot] + 4 * h;
                        auto step = [&](auto masked_type) {
                            constexpr bool MASKED = decltype(masked_type)::value;
                            constexpr int NB = ST / BS;
                            uint32_t v[NB][16];
#pragma unroll
                            for (int q = 0; q < NB; q++) tmem_ld16(tb + q * 16, v[q]);
                            tmem_wait_ld();
                            float mx = -INFINITY, mv = -INFINITY;   // no scale is negative: the maximum commutes with them; mv: with V's scale
#pragma unroll
                            for (int q = 0; q < NB; q++) {      // a block
                                float top = -INFINITY;
#pragma unroll
                                for (int k = 0; k < 16; k++) top = fmaxf(top, MASKED && q * 16 + k >= left ? -INFINITY : __uint_as_float(v[q][k]));
                                if (FP8) {
                                    top *= sc[q];               // -inf x 0 is NaN, which no maximum takes
                                    mv = fmaxf(mv, top + sc[16 + q]);
                                }
                                mx = fmaxf(mx, top);
                            }
                            if (!FP8) mx = mx == -INFINITY ? mx : mx * a.scale_log2;
                            // ---- a raised reference rescales the row of O, once the product of the step before is done ----
                            float factor = 1.0f;
                            if (mx > m + RAISE || (FP8 && mv + tkv_rows::log2_of_power(unit) > m + RAISE)) {
                                const float m_new = fmaxf(m, mx - HEAD);
                                const float up = m_new - m;
                                factor = m == -INFINITY ? 0.0f : fast_exp2(-up);
                                m = m_new;
                                l *= factor;
                                if (FP8) {
                                    const float u = tkv_rows::next_unit(unit, up, mv == -INFINITY ? mv : mv - m);
                                    factor *= u * tkv_rows::inverse_of_power(unit);
                                    unit = u;
                                }
                            }
                            if (n > s_x && __any_sync(0xFFFFFFFFu, factor != 1.0f)) {
                                ok = __all_sync(0xFFFFFFFFu, bar_wait(smem_u32(&c->pv_done[x][b ^ 1u]), ((n - 1) >> 1) & 1u, fail));
                                tc_fence_after();
#pragma unroll 1
                                for (uint32_t c0 = 0; c0 < (uint32_t)D; c0 += 16) {
                                    uint32_t o[16];
                                    tmem_ld16(to + c0, o);
                                    tmem_wait_ld();
#pragma unroll
                                    for (int k = 0; k < 16; k++) o[k] = __float_as_uint(__uint_as_float(o[k]) * factor);
                                    tmem_st16(to + c0, o);
                                }
                                tmem_wait_st();
                            }
                            // ---- probabilities, as F16 pairs over the scores ----
                            const float sub = m == -INFINITY ? 0.0f : -m;
                            float sum = 0.0f;
#pragma unroll
                            for (int q = 0; q < NB; q++) {
                                const float ks = FP8 ? sc[q] : a.scale_log2, vn = FP8 ? sc[8 + q] * unit : 1.0f;
                                uint32_t first[8], second[8];
#pragma unroll
                                for (int k = 0; k < 16; k += 2) {
                                    float p0 = fast_exp2(__fmaf_rn(__uint_as_float(v[q][k]), ks, sub));
                                    float p1 = fast_exp2(__fmaf_rn(__uint_as_float(v[q][k + 1]), ks, sub));
                                    if (MASKED) {
                                        p0 = q * 16 + k < left ? p0 : 0.0f;
                                        p1 = q * 16 + k + 1 < left ? p1 : 0.0f;
                                    }
                                    sum += p0 + p1;
                                    if (FP8) {
                                        p0 *= vn;
                                        p1 *= vn;
                                    }
                                    const __half2 hp = __floats2half2_rn(p0, p1);
                                    first[k / 2] = *reinterpret_cast<const uint32_t*>(&hp);
                                    const float2 fp = __half22float2(hp);
                                    const __half2 lp = __floats2half2_rn(p0 - fp.x, p1 - fp.y);
                                    second[k / 2] = *reinterpret_cast<const uint32_t*>(&lp);
                                }
                                tmem_st8(tb + q * 8, first);
                                tmem_st8(tb + 32 + q * 8, second);
                            }
                            tmem_wait_st();
                            l += sum;
                        };
                        const bool masked = __any_sync(0xFFFFFFFFu, left < ST);
                        if (masked) step(std::true_type{});
                        else step(std::false_type{});
                        tc_fence_before();
                    }
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&c->p_full[x][b]);
                }
            }
            // ---- partial result of the row ----
            const bool any = n > s_x;
            const uint64_t dst = it.out_row + x * 128u + r;
            if (ok && any) ok = __all_sync(0xFFFFFFFFu, bar_wait(smem_u32(&c->pv_done[x][(n - 1) & 1u]), ((n - 1) >> 1) & 1u, fail));
            if (ok && warp_live) {
                tc_fence_after();
                if (live) *reinterpret_cast<float2*>(a.part_ml + dst * 2) = any ? make_float2(m, l) : make_float2(-INFINITY, 0.0f);
                if (any) {
                    // through the stream's Q tile, which no product reads any more, half of the dims at a time: the rows of a warp follow one
                    // another in memory, so a store covers whole half rows (a row per thread took 9 000 cycles)
                    constexpr int DH = D / 2, CH = DH / 4;      // dims of a pass; its 16-byte chunks per row
                    unsigned char* stage = q_tile + x * TILE + (warp & 3u) * (TILE / 4);
                    const uint32_t n_live = (uint32_t)__popc(__ballot_sync(0xFFFFFFFFu, live));
                    const float inv_unit = tkv_rows::inverse_of_power(unit);
                    float* rows_out = a.part_o + (dst - lane) * D;             // (the warp's first row is alive if any is)
#pragma unroll 1
                    for (int d0 = 0; d0 < D; d0 += DH) {
#pragma unroll
                        for (int c0 = 0; c0 < DH; c0 += 32) {
                            uint32_t o[32];
                            tmem_ld32(to + d0 + c0, o);
                            tmem_wait_ld();
#pragma unroll
                            for (int k = 0; k < 8; k++)
                                *reinterpret_cast<float4*>(stage + lane * (DH * 4) + (((c0 / 4 + k) ^ (lane % CH)) * 16)) =
                                    make_float4(__uint_as_float(o[4 * k]) * inv_unit, __uint_as_float(o[4 * k + 1]) * inv_unit, __uint_as_float(o[4 * k + 2]) * inv_unit,
                                                __uint_as_float(o[4 * k + 3]) * inv_unit);
                        }
                        __syncwarp();
#pragma unroll 8
                        for (uint32_t n16 = lane; n16 < n_live * CH; n16 += 32) {
                            const uint32_t o = n16 / CH, k = n16 % CH;
                            *reinterpret_cast<float4*>(rows_out + (size_t)o * D + d0 + 4 * k) = *reinterpret_cast<const float4*>(stage + o * (DH * 4) + ((k ^ (o % CH)) * 16));
                        }
                        __syncwarp();
                    }
                }
            }
            if (!ok && lane == 0) atomicCAS(&c->fail, 0u, 4u);
            tc_fence_before();
        }
        __syncthreads();                                        // the next item's Q overwrites this one's
        tc_fence_after();
        if (*fail) break;                                       // the same for all threads: nobody writes it between the two barriers
        __syncthreads();
        tiles_done += it.n_tiles;
        const uint32_t cut = 2 - steps_in(it.n_tiles - 1);      // only a prefix's last tile may hold one half
        n_steps += 2 * it.n_tiles - cut;
        u += it.n_tiles;
    }
    if (!FP8 && warp == SM && *fail) {                          // whichever role gave up, no copy is in flight when the CTA's shared memory goes
#pragma unroll
        for (int kv = 0; kv < 2; kv++)                          // the last two of each ring
            for (uint32_t t = issued[kv] > 2 ? issued[kv] - 2 : 0u; t < issued[kv]; t++)
                for (uint32_t n = 0; n < (1u << 20) && !mbar_test((kv ? c->v_full : c->k_full) + (t & 1u), (t >> 1) & 1u); n++) {}
    }
    if (warp >= SM + FEED && elect_one()) {                     // (the lane that issued) whatever ended the loop, no product is under way when tensor memory goes back
        uint64_t* bar = c->drained + (warp - (SM + FEED));
        tc_commit(bar);
        for (uint32_t i = 0; i < (1u << 22) && !mbar_test(bar, 0u); i++) {}
    }
    __syncthreads();
    if (warp == SM + FEED) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    }
    if (tid == 0 && c->fail) tkv_rows::report(a.status, c->fail);
}

// ---- joining ----------------------------------------------------------------------------------------------------------------------
struct JoinArgs {
    const float *pre_o, *pre_ml, *own_o, *own_ml;   // partial results over the prefixes, over the tokens behind them
    const uint32_t *pre_plan, *own_plan, *group_starts, *prefix_lens;
    __half* out;
    uint32_t n_seqs, n_groups, n_q_heads, n_kv_heads, group;
};

// WPR warps join the partial results of one (sequence, query head): one where there are rows enough to fill the machine, eight where
// few rows have many parts (960 rows: 38 us for the whole call with eight, 42 with one; 8 192 rows: 136 and 117).  Bound by latency and L2.
template <int D, int WPR> __global__ void __launch_bounds__(256) prefix_join(const JoinArgs a) {
    // what the caller wrote is read while the kernels before this one still run
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
    const uint64_t row = WPR == 1 ? (uint64_t)blockIdx.x * 8 + warp : blockIdx.x;
    const bool in = row < (uint64_t)a.n_seqs * a.n_q_heads;
    const uint32_t s = in ? (uint32_t)(row / a.n_q_heads) : 0u, head = in ? (uint32_t)(row % a.n_q_heads) : 0u;
    const uint32_t g = tkv_rows::group_of(a.group_starts, a.n_groups, s), g_in = min(g, a.n_groups - 1);
    const uint32_t base = a.group_starts[0], s0 = a.group_starts[g_in], s1 = a.group_starts[g_in + 1], prefix = a.prefix_lens[g_in];
    asm volatile("griddepcontrol.wait;" ::: "memory");          // launched ahead of the second kernel's end, which comes after the first one's
    const uint32_t share_t = a.pre_plan[0], share_b = a.own_plan[0], tiles_before = a.pre_plan[1 + g_in], lo = a.own_plan[1 + s], hi = a.own_plan[2 + s];
    if (!in || share_t == 0 || share_b == 0 || g == a.n_groups) return;   // (all warps of a row alike) refused, or a row behind the last sequence
    // parts of the prefix
    const uint32_t rows = (s1 - s0) * a.group, kvh = head / a.group, r = (s - s0) * a.group + head % a.group;
    const uint32_t rb = r / 256, nt = (prefix + KT - 1) / KT;
    const uint32_t t0 = tiles_before + (kvh * row_blocks(rows) + rb) * nt, c0 = nt ? t0 / share_t : 0u;
    const uint32_t n_pre = nt ? (t0 + nt - 1) / share_t - c0 + 1 : 0u;
    const uint64_t first = (uint64_t)(s0 - base) * a.group * a.n_kv_heads + (uint64_t)kvh * rows + r + 256ull * c0;
    // parts of the tokens behind it
    const uint32_t p0 = hi > lo ? lo / share_b : 0u;
    const uint32_t n_own = hi > lo ? (hi - 1) / share_b - p0 + 1 : 0u, n = n_pre + n_own;
    auto part = [&](uint32_t i, const float*& o, const float*& ml) {
        if (i < n_pre) {
            const uint64_t at = first + i * 256ull;
            o = a.pre_o + at * D;
            ml = a.pre_ml + at * 2;
        } else {
            const uint64_t at = ((uint64_t)(p0 + s) + (i - n_pre)) * a.n_q_heads + head;
            o = a.own_o + at * D;
            ml = a.own_ml + at * 2;
        }
    };
    // maximum and sum of the row, every warp by itself
    float m = -INFINITY, l = 0.0f;
    for (uint32_t i0 = 0; i0 < n; i0 += 128) {
        float2 v[4];
#pragma unroll
        for (int q = 0; q < 4; q++) {
            const uint32_t i = i0 + 32 * q + lane;
            v[q] = make_float2(-INFINITY, 0.0f);
            if (i < n) {
                const float *o, *ml;
                part(i, o, ml);
                v[q] = *reinterpret_cast<const float2*>(ml);
            }
        }
#pragma unroll
        for (int q = 0; q < 4; q++) {
            const float mm = fmaxf(m, v[q].x);
            l = mm == -INFINITY ? l + v[q].y : l * fast_exp2(m - mm) + v[q].y * fast_exp2(v[q].x - mm);
            m = mm;
        }
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) {
        const float m_o = __shfl_xor_sync(0xFFFFFFFFu, m, off), l_o = __shfl_xor_sync(0xFFFFFFFFu, l, off);
        const float mm = fmaxf(m, m_o);
        l = mm == -INFINITY ? l + l_o : l * fast_exp2(m - mm) + l_o * fast_exp2(m_o - mm);
        m = mm;
    }
    const float top = m == -INFINITY ? 0.0f : m, inv = l == 0.0f ? 0.0f : 1.0f / l;   // an empty row: 0
    constexpr int PER = D / 32;
    float acc[PER];
#pragma unroll
    for (int d = 0; d < PER; d++) acc[d] = 0.0f;
#pragma unroll 8
    for (uint32_t i = WPR == 1 ? 0u : warp; i < n; i += WPR) {
        const float *o, *ml;
        part(i, o, ml);
        const float2 v = *reinterpret_cast<const float2*>(ml);
        const float f = fast_exp2(v.x - top);
        float x[PER];
#pragma unroll
        for (int d = 0; d < PER; d++) x[d] = o[d * 32 + lane];
#pragma unroll
        for (int d = 0; d < PER; d++) acc[d] = v.x != -INFINITY || v.y != 0.0f ? __fmaf_rn(f, x[d], acc[d]) : acc[d];   // an empty part's O counts for nothing
    }
    __half* out = a.out + row * D;
    if (WPR == 1) {
#pragma unroll
        for (int d = 0; d < PER; d++) out[d * 32 + lane] = __float2half_rn(acc[d] * inv);
    } else {
        __shared__ float sum[8][D];
#pragma unroll
        for (int d = 0; d < PER; d++) sum[warp][d * 32 + lane] = acc[d];
        __syncthreads();
        if (threadIdx.x < D) {
            float v = 0.0f;
#pragma unroll
            for (int w = 0; w < 8; w++) v += sum[w][threadIdx.x];
            out[threadIdx.x] = __float2half_rn(v * inv);
        }
    }
}

// ---- host side --------------------------------------------------------------------------------------------------------------------
int32_t fail(int32_t code, const char* fmt, unsigned long long x = 0, unsigned long long y = 0) {
    char buf[256];
    snprintf(buf, sizeof buf, fmt, x, y);
    return tkv_internal::set_error(code, 0, buf);
}
uint64_t up(uint64_t x, uint64_t to) { return (x + to - 1) / to * to; }

// An F16 layer tensor as bytes [token][kv head][2 D], boxes of [16 tokens][1 head][128 B]: one column group of a head's rows of a block.
bool make_map(CUtensorMap* map, uint64_t base, uint32_t total_blocks, uint32_t n_kv_heads, uint32_t head_dim) {
    EncodeTiledFn fn = encode_tiled();
    if (!fn) return false;
    const cuuint64_t dims[3] = {2ull * head_dim, n_kv_heads, (cuuint64_t)total_blocks * BS};
    const cuuint64_t strides[2] = {2ull * head_dim, 2ull * head_dim * n_kv_heads};
    const cuuint32_t box[3] = {128u, 1u, (cuuint32_t)BS}, elem[3] = {1u, 1u, 1u};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, reinterpret_cast<void*>(base), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

struct Layout {
    tkv_rows::Split own;                     // of the tokens behind the prefixes
    uint32_t parts;                          // of the prefixes
    uint64_t pre_ml, pre_o, own_plan, own_ml, own_o, bytes;   // offsets; the prefixes' plan is at 0
};
Layout layout_of(uint32_t n_seqs, uint32_t n_groups, uint32_t n_q_heads, uint32_t n_kv_heads, uint32_t head_dim, uint32_t max_kv_len, uint32_t max_prefix_len) {
    Layout l;
    const uint64_t group = n_q_heads / n_kv_heads, nt = (max_prefix_len + KT - 1ull) / KT;
    const uint64_t tiles = (n_groups + (uint64_t)n_seqs * group / 256) * n_kv_heads * nt;      // at most: every group ends in a row block of its own
    l.parts = (uint32_t)std::max<uint64_t>(1, std::min<uint64_t>(CTAS, tiles));
    l.own = tkv_rows::split_for((uint64_t)n_seqs * ((max_kv_len + 15ull) / 16), n_kv_heads, CTAS);
    const uint64_t rows = (uint64_t)n_seqs * n_q_heads + 256ull * l.parts, slots = (uint64_t)l.own.parts + n_seqs;
    l.pre_ml = up(4ull * (n_groups + 2ull), 256);
    l.pre_o = l.pre_ml + up(rows * 8, 256);
    l.own_plan = l.pre_o + up(rows * head_dim * 4, 256);
    l.own_ml = l.own_plan + up(4ull * (n_seqs + 2ull), 256);
    l.own_o = l.own_ml + up(slots * n_q_heads * 8, 256);
    l.bytes = l.own_o + slots * n_q_heads * head_dim * 4;
    return l;
}

template <int D, bool FP8> cudaError_t launch_prefix(const CUtensorMap& mk, const CUtensorMap& mv, const Args& a, cudaStream_t st) {
    constexpr size_t smem = CTRL_BYTES + 6 * (size_t)(D / 64) * GROUP_BYTES + (FP8 ? 2 * 128 * (size_t)D : 0);
    static_assert(smem <= 227 * 1024, "shared memory of one CTA");
    auto kernel = prefix_attn_tc<D, FP8>;
    static std::atomic<uint64_t> granted{0};                    // devices on which this kernel may use that much shared memory
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    const uint64_t bit = dev < 64 ? 1ull << dev : 0ull;
    if (!(granted.load(std::memory_order_relaxed) & bit)) {
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return e;
        granted.fetch_or(bit, std::memory_order_relaxed);
    }
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(a.parts);
    cfg.blockDim = dim3(threads_of(FP8));
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    return cudaLaunchKernelEx(&cfg, kernel, mk, mv, a);
}
template <int D> cudaError_t launch_join(const JoinArgs& a, cudaStream_t st) {
    const uint64_t rows = (uint64_t)a.n_seqs * a.n_q_heads;
    const bool few = rows <= 8ull * CTAS;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(few ? rows : (rows + 7) / 8));
    cfg.blockDim = dim3(256);
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    return few ? cudaLaunchKernelEx(&cfg, prefix_join<D, 8>, a) : cudaLaunchKernelEx(&cfg, prefix_join<D, 1>, a);
}

}  // namespace

extern "C" {

uint64_t tkv_prefix_attn_scratch_bytes(uint32_t n_seqs, uint32_t n_groups, uint32_t n_q_heads, uint32_t n_kv_heads, uint32_t head_dim, uint32_t max_kv_len,
                                       uint32_t max_prefix_len) {
    if (!n_seqs || !n_groups || !n_kv_heads || n_q_heads < n_kv_heads || max_kv_len > 0xFFFFFFF0u || max_prefix_len > 0xFFFFFFF0u) return 0;
    return layout_of(n_seqs, n_groups, n_q_heads, n_kv_heads, head_dim, max_kv_len, max_prefix_len).bytes;
}

int32_t tkv_prefix_attn_enqueue(const TkvPool* pool, const TkvPrefixAttn* p, void* stream) {
    if (!pool || !p) return fail(TKV_ERR_INVALID_CONFIG, "NULL argument");
    if (pool->dtype != TKV_DTYPE_F16 && pool->dtype != TKV_DTYPE_E4M3)
        return fail(TKV_ERR_INVALID_CONFIG, "shared-prefix attention reads F16 or E4M3 pools (dtype %llu)", (unsigned long long)pool->dtype);
    if (pool->head_dim != 64 && pool->head_dim != 128)
        return fail(TKV_ERR_DIMENSION_MISMATCH, "dimension mismatch: expected %llu, got %llu (shared-prefix attention is built for head_dim 64 and 128)", 128,
                    pool->head_dim);
    if (pool->block_size != BS)
        return fail(TKV_ERR_DIMENSION_MISMATCH, "dimension mismatch: expected %llu, got %llu (tokens per block)", BS, pool->block_size);
    if (p->layer >= pool->n_layers) return fail(TKV_ERR_INVALID_CONFIG, "layer %llu outside the pool (%llu layers)", p->layer, pool->n_layers);
    if (!pool->n_kv_heads || !p->n_q_heads || p->n_q_heads % pool->n_kv_heads || p->n_q_heads / pool->n_kv_heads > 8)
        return fail(TKV_ERR_DIMENSION_MISMATCH, "dimension mismatch: expected %llu, got %llu (query heads must be 1..8 times the kv heads)",
                    pool->n_kv_heads, p->n_q_heads);
    if (pool->n_kv_heads > CTAS * tkv_rows::WARPS) return fail(TKV_ERR_INVALID_CONFIG, "at most %llu kv heads (%llu)", CTAS * tkv_rows::WARPS, pool->n_kv_heads);
    if ((pool->k_scales == 0) != (pool->v_scales == 0)) return fail(TKV_ERR_INVALID_CONFIG, "k_scales and v_scales must both be set or both be 0");
    if (pool->k_scales && pool->dtype != TKV_DTYPE_E4M3) return fail(TKV_ERR_INVALID_CONFIG, "only an E4M3 pool carries scales");
    const float scale_log2 = p->sm_scale * 1.4426950408889634f;
    if (!std::isfinite(scale_log2)) return fail(TKV_ERR_INVALID_CONFIG, "sm_scale x log2(e) is not finite");
    if (p->n_seqs == 0 || p->n_groups == 0) return TKV_OK;
    if (!p->q || !p->out || !p->tables || !p->kv_lens || !p->group_starts || !p->prefix_lens || !pool->k_layer_ptrs || !pool->v_layer_ptrs || !pool->total_blocks)
        return fail(TKV_ERR_INVALID_CONFIG, "NULL buffer");
    if (p->max_kv_len > 0xFFFFFFF0u || p->max_prefix_len > 0xFFFFFFF0u) return fail(TKV_ERR_INVALID_CONFIG, "length bounds above 2^32 - 16");
    const uint64_t own_blocks = (uint64_t)p->n_seqs * ((p->max_kv_len + 15ull) / 16), group = p->n_q_heads / pool->n_kv_heads;
    const uint64_t tiles = (p->n_groups + (uint64_t)p->n_seqs * group / 256) * pool->n_kv_heads * ((p->max_prefix_len + KT - 1ull) / KT);
    if (own_blocks >= 0x7FFFFFFFull || tiles >= 0x7FFFFFFFull || (uint64_t)p->n_seqs * p->n_q_heads >= 0x7FFFFFFFull)
        return fail(TKV_ERR_INVALID_CONFIG, "%llu sequences of %llu tokens: batch too large", p->n_seqs, p->max_kv_len);
    if (std::max((p->max_kv_len + 15ull) / 16, (p->max_prefix_len + 15ull) / 16) > p->table_stride)
        return fail(TKV_ERR_DIMENSION_MISMATCH, "dimension mismatch: expected %llu, got %llu (table_stride below the blocks of max_kv_len or max_prefix_len)",
                    std::max((p->max_kv_len + 15ull) / 16, (p->max_prefix_len + 15ull) / 16), p->table_stride);
    const bool fp8 = pool->dtype == TKV_DTYPE_E4M3;
    if (!fp8 && (uint64_t)pool->total_blocks * BS >= 0x7FFFFFFFull) return fail(TKV_ERR_INVALID_CONFIG, "an F16 pool of %llu blocks is too large", pool->total_blocks);
    const uint64_t kp = pool->k_layer_ptrs[p->layer], vp = pool->v_layer_ptrs[p->layer];
    if (!kp || !vp) return fail(TKV_ERR_INVALID_CONFIG, "NULL buffer");
    if ((kp | vp | p->q | p->out) % 16 || p->scratch % 256) return fail(TKV_ERR_INVALID_CONFIG, "layer tensors, q and out must be 16-byte aligned, scratch 256-byte");
    if ((p->tables | p->kv_lens | p->group_starts | p->prefix_lens | p->status | pool->k_scales | pool->v_scales) % 4)
        return fail(TKV_ERR_INVALID_CONFIG, "tables, lengths, groups, scales and status must be 4-byte aligned");
    const Layout l = layout_of(p->n_seqs, p->n_groups, p->n_q_heads, pool->n_kv_heads, pool->head_dim, p->max_kv_len, p->max_prefix_len);
    if (!p->scratch || p->scratch_bytes < l.bytes)
        return fail(TKV_ERR_DIMENSION_MISMATCH, "dimension mismatch: expected %llu, got %llu (scratch bytes)", l.bytes, p->scratch ? p->scratch_bytes : 0);

    const uint32_t es = fp8 ? 1u : 2u;
    const size_t layer_scales = (size_t)p->layer * pool->total_blocks * pool->n_kv_heads;
    Args a{};
    a.tables = reinterpret_cast<const uint32_t*>(p->tables);
    a.kv_lens = reinterpret_cast<const uint32_t*>(p->kv_lens);
    a.group_starts = reinterpret_cast<const uint32_t*>(p->group_starts);
    a.prefix_lens = reinterpret_cast<const uint32_t*>(p->prefix_lens);
    a.q = reinterpret_cast<const __half*>(p->q);
    a.k8 = reinterpret_cast<const char*>(kp);
    a.v8 = reinterpret_cast<const char*>(vp);
    a.k_scales = pool->k_scales ? reinterpret_cast<const float*>(pool->k_scales) + layer_scales : nullptr;
    a.v_scales = pool->v_scales ? reinterpret_cast<const float*>(pool->v_scales) + layer_scales : nullptr;
    a.plan = reinterpret_cast<uint32_t*>(p->scratch);
    a.part_ml = reinterpret_cast<float*>(p->scratch + l.pre_ml);
    a.part_o = reinterpret_cast<float*>(p->scratch + l.pre_o);
    a.status = reinterpret_cast<uint32_t*>(p->status);
    a.row_stride = pool->n_kv_heads * pool->head_dim * es;
    a.block_stride = (uint64_t)BS * a.row_stride;
    a.n_seqs = p->n_seqs;
    a.n_groups = p->n_groups;
    a.n_q_heads = p->n_q_heads;
    a.n_kv_heads = pool->n_kv_heads;
    a.group = (uint32_t)group;
    a.table_stride = p->table_stride;
    a.max_kv_len = p->max_kv_len;
    a.max_prefix_len = p->max_prefix_len;
    a.total_blocks = pool->total_blocks;
    a.parts = l.parts;
    a.q_sign = scale_log2 < 0.0f ? 0x80008000u : 0u;
    a.scale_log2 = std::fabs(scale_log2);

    tkv_rows::Args r{};
    r.k_base = a.k8;
    r.v_base = a.v8;
    r.k_scales = a.k_scales;
    r.v_scales = a.v_scales;
    r.q = a.q;
    r.tables = a.tables;
    r.kv_lens = a.kv_lens;
    r.group_starts = a.group_starts;
    r.prefix_lens = a.prefix_lens;
    r.plan = reinterpret_cast<uint32_t*>(p->scratch + l.own_plan);
    r.part_ml = reinterpret_cast<float*>(p->scratch + l.own_ml);
    r.part_o = reinterpret_cast<float*>(p->scratch + l.own_o);
    r.status = a.status;
    r.block_stride = a.block_stride;
    r.row_stride = a.row_stride;
    r.n_seqs = a.n_seqs;
    r.n_groups = a.n_groups;
    r.n_q_heads = a.n_q_heads;
    r.n_kv_heads = a.n_kv_heads;
    r.group = a.group;
    r.table_stride = a.table_stride;
    r.max_kv_len = a.max_kv_len;
    r.max_prefix_len = a.max_prefix_len;
    r.total_blocks = a.total_blocks;
    r.scale_log2 = scale_log2;

    JoinArgs j{};
    j.pre_o = a.part_o;
    j.pre_ml = a.part_ml;
    j.own_o = r.part_o;
    j.own_ml = r.part_ml;
    j.pre_plan = a.plan;
    j.own_plan = r.plan;
    j.group_starts = a.group_starts;
    j.prefix_lens = a.prefix_lens;
    j.out = reinterpret_cast<__half*>(p->out);
    j.n_seqs = a.n_seqs;
    j.n_groups = a.n_groups;
    j.n_q_heads = a.n_q_heads;
    j.n_kv_heads = a.n_kv_heads;
    j.group = a.group;

    CUtensorMap mk{}, mv{};
    if (!fp8 && (!make_map(&mk, kp, pool->total_blocks, pool->n_kv_heads, pool->head_dim) || !make_map(&mv, vp, pool->total_blocks, pool->n_kv_heads, pool->head_dim)))
        return fail(TKV_ERR_CUDA, "shared-prefix attention: cannot describe the layer tensors to the copy engine");
    int prev = -1;
    cudaError_t e = cudaGetDevice(&prev);
    if (e == cudaSuccess && prev != pool->device) e = cudaSetDevice(pool->device);
    if (e == cudaSuccess) {
        cudaStream_t st = static_cast<cudaStream_t>(stream);
        if (pool->head_dim == 128) e = fp8 ? launch_prefix<128, true>(mk, mv, a, st) : launch_prefix<128, false>(mk, mv, a, st);
        else e = fp8 ? launch_prefix<64, true>(mk, mv, a, st) : launch_prefix<64, false>(mk, mv, a, st);
        if (e == cudaSuccess) e = tkv_rows::launch_rows(pool->head_dim, fp8, false, r, l.own, true, st);
        if (e == cudaSuccess) e = pool->head_dim == 128 ? launch_join<128>(j, st) : launch_join<64>(j, st);
    }
    if (prev >= 0 && prev != pool->device) cudaSetDevice(prev);
    if (e != cudaSuccess) {
        cudaGetLastError();                                     // reported here, not by whoever asks next
        char buf[256];
        snprintf(buf, sizeof buf, "shared-prefix attention launch: %s (cuda error %d)", cudaGetErrorString(e), (int)e);
        return tkv_internal::set_error(TKV_ERR_CUDA, (int32_t)e, buf);
    }
    return TKV_OK;
}

}  // extern "C"
