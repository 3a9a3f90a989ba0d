// Cutting a cache to a budget by accumulated attention weight: which tokens of every (layer, sequence, kv head) stay, and the move of
// their rows to the front of the sequence's blocks.
//
// Select.  Of a row of `len` tokens the first `protect`, the last `recent` and the best-scored others stay, together
//     new_len = min(len, max(budget, protect + recent)),
// ties to the lower index.  Scores become 32-bit keys that compare like the numbers (NaN below everything, -0 = +0); the key that
// the last kept token has is found by histograms over 11, 11 and 10 bits of it, each over the tokens whose higher bits agree with what is
// known; once these are few, a thread ranks each of them against all.  A last pass writes the indices in ascending order (ballots inside a
// warp, prefix sums across warps and CTAs).  Scores are read once into shared memory; the bound is instruction issue for many rows (4 096
// rows of up to 4 096 tokens: 56 us for 52.6 MB, 45 million warp instructions) and latency for few (88 rows of 512: 6.1 us).  A long row
// is split over a thread-block cluster, whose CTAs add their histograms through distributed shared memory.
//
// Compact.  Row j takes what row kept[j] >= j holds, in place.  A CTA owns one row set (layer, sequence, kv head, K or V) and
// walks it in tiles: it reads all rows of a tile, waits, then stores them.  A row that a tile overwrites can only be the source of
// rows at or before it, which are in this tile or an earlier one, so nothing is lost and no second buffer is needed.  Bound by HBM: a moved
// row is read and written once (2.19 GB of F16 rows in 356 us, 6.15 TB/s).  Rows of half the size keep fewer bytes in flight per tile, and nothing
// of the next tile: 526 MB of E4M3 rows take 103 us (5.1 TB/s) without scales and 124 (4.2 TB/s) with them, where they are re-encoded.
// Rows that stay are not touched, protected (shared) blocks among them.
// A block of a scaled E4M3 pool has one scale: it becomes the largest of its new rows' scales.  Rows that had it keep their bytes; the others
// are multiplied by scale / new scale <= 1 and rounded to E4M3 once more (half a step, 2^-4 relative, and flushed to zero below
// 2^-6 as every writer of this pool does).  Taking the rows' absolute maximum instead would round every row again at every eviction.
#include <cooperative_groups.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdio>
#include <stdint.h>

#include "../../include/tkv.h"

namespace tkv_internal {
int32_t set_error(int32_t code, int32_t cuda_code, const char* text);
}

namespace {

namespace cg = cooperative_groups;

constexpr int BS = 16;
constexpr int BINS = 2048;
constexpr int FEW = 256;                     // tokens that are ranked against one another: at most one per thread
constexpr uint32_t STAGE_TOKENS = 49152;     // tokens of a row that a CTA keeps in shared memory; longer slices are read again in every pass
constexpr uint32_t MAX_CLUSTER = 8;

__device__ __forceinline__ void report_bad(uint32_t* status) {
    if (status) atomicCAS(status, 0u, (uint32_t)TKV_ERR_INVALID_CONFIG);
}

struct SelectArgs {
    const float* scores;
    const uint32_t *kv_lens, *protect;
    uint32_t *kept, *new_lens, *status;
    uint32_t n_seqs, n_kv_heads, max_kv_len, score_stride, kept_stride, budget, recent;
    uint32_t staged;                         // the slice fits the CTA's shared memory
};

// tokens that stay of `len`, of which `protect` + `recent` always do
__device__ __forceinline__ uint32_t kept_of(uint32_t len, uint32_t protect, uint32_t recent, uint32_t budget) {
    const uint64_t always = (uint64_t)protect + recent;
    return always >= len || budget >= len ? len : max(budget, (uint32_t)always);
}

__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t u = __float_as_uint(x);
    if ((u & 0x7FFFFFFFu) > 0x7F800000u) return 0u;             // NaN
    if (u == 0x80000000u) return 0x80000000u;                   // -0 like +0
    return u ^ ((u >> 31) ? 0xFFFFFFFFu : 0x80000000u);
}

template <int THREADS> __global__ void __launch_bounds__(THREADS, 1536 / THREADS) evict_select(const SelectArgs a) {
    constexpr int WARPS = THREADS / 32, PER_THREAD = BINS / THREADS;
    static_assert(BINS % (4 * THREADS) == 0, "every thread clears the same number of bins");
    cg::cluster_group cluster = cg::this_cluster();
    const uint32_t parts = cluster.num_blocks(), rank = cluster.block_rank();
    const uint32_t row = blockIdx.x / parts, s = (row / a.n_kv_heads) % a.n_seqs;
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u, below = (1u << lane) - 1u;
    extern __shared__ uint32_t keys[];
    __shared__ __align__(16) uint32_t hist[BINS];
    __shared__ uint32_t warp_sum[WARPS], chosen[4], n_gt[WARPS + 1], n_eq[WARPS + 1], few[FEW];

    uint32_t len = a.kv_lens[s];
    if (len > a.max_kv_len) {
        len = a.max_kv_len;
        if (tid == 0) report_bad(a.status);
    }
    const uint32_t protect = a.protect ? min(a.protect[s], len) : 0u;
    const uint32_t target = kept_of(len, protect, a.recent, a.budget);
    const bool fits = target <= a.kept_stride || target == len;
    const uint32_t n_new = fits ? target : len;                 // a row that kept cannot hold is not cut
    if (tid == 0 && rank == 0 && row < a.n_seqs * a.n_kv_heads && row % a.n_kv_heads == 0) a.new_lens[s] = n_new;
    uint32_t* out = a.kept + (size_t)row * a.kept_stride;
    if (n_new == len) {
        if (!fits && tid == 0) report_bad(a.status);
        for (uint32_t i = rank * THREADS + tid; i < min(len, a.kept_stride); i += parts * THREADS) out[i] = i;
        return;
    }
    const uint32_t lo = protect, n_mid = len - a.recent - protect, need = n_new - protect - a.recent;   // need < n_mid
    for (uint32_t i = rank * THREADS + tid; i < protect + a.recent; i += parts * THREADS)
        out[i < protect ? i : need + i] = i < protect ? i : len - a.recent + (i - protect);
    if (need == 0) return;

    // ---- this CTA's slice of the tokens to choose from ----
    const uint32_t per = (n_mid + parts - 1) / parts, begin = min(n_mid, rank * per), n = min(per, n_mid - begin);
    const float* src = a.scores + (size_t)row * a.score_stride + lo + begin;
    auto key_at = [&](uint32_t i) { return a.staged ? keys[i] : key_of(src[i]); };

    // ---- the key of the last token that stays ----
    uint32_t prefix = 0, mask = 0, left = need;
    for (int pass = 0; pass < 3; pass++) {
        const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
        const uint32_t digit_mask = pass == 2 ? 1023u : 2047u;
#pragma unroll
        for (int i = 0; i < BINS / 4; i += THREADS) reinterpret_cast<uint4*>(hist)[i + tid] = make_uint4(0, 0, 0, 0);
        if (tid == 0) chosen[2] = 0;
        __syncthreads();
        if (pass == 0) {                                        // the scores are read here
            constexpr int AHEAD = 8;                            // asked for together
            for (uint32_t i0 = tid; i0 < n; i0 += AHEAD * THREADS) {
                float x[AHEAD];
#pragma unroll
                for (int q = 0; q < AHEAD; q++) x[q] = i0 + q * THREADS < n ? src[i0 + q * THREADS] : 0.0f;
#pragma unroll
                for (int q = 0; q < AHEAD; q++) {
                    const uint32_t i = i0 + q * THREADS, k = key_of(x[q]);
                    if (i < n) {
                        if (a.staged) keys[i] = k;
                        atomicAdd(&hist[k >> 21], 1u);
                    }
                }
            }
        } else {
            for (uint32_t i = tid; i < n; i += THREADS) {
                const uint32_t k = key_at(i);
                if ((k & mask) == prefix) atomicAdd(&hist[(k >> shift) & digit_mask], 1u);
            }
        }
        if (parts > 1) cluster.sync();
        else __syncthreads();
        // thread t has the bins from BINS - 1 - PER_THREAD * t downwards, of all CTAs
        uint32_t c[PER_THREAD], sum = 0;
        const uint32_t bin0 = BINS - PER_THREAD * (tid + 1);
#pragma unroll
        for (int i = 0; i < PER_THREAD; i++) c[i] = hist[bin0 + PER_THREAD - 1 - i];
        if (parts > 1) {
            for (uint32_t r = 1; r < parts; r++) {
                const uint32_t* other = cluster.map_shared_rank(hist, (rank + r) % parts);
#pragma unroll
                for (int i = 0; i < PER_THREAD; i++) c[i] += other[bin0 + PER_THREAD - 1 - i];
            }
        }
#pragma unroll
        for (int i = 0; i < PER_THREAD; i++) sum += c[i];
        uint32_t incl = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t v = __shfl_up_sync(0xFFFFFFFFu, incl, o);
            if (lane >= (uint32_t)o) incl += v;
        }
        if (lane == 31) warp_sum[warp] = incl;
        __syncthreads();
        uint32_t above = incl - sum;
#pragma unroll
        for (int w = 0; w < WARPS; w++) above += w < (int)warp ? warp_sum[w] : 0u;
        if (above < left && left <= above + sum) {              // one thread
#pragma unroll
            for (int i = 0; i < PER_THREAD; i++) {
                if (above < left && left <= above + c[i]) {
                    chosen[0] = bin0 + PER_THREAD - 1 - i;
                    chosen[1] = above;
                    chosen[3] = c[i];
                }
                above += c[i];
            }
        }
        if (parts > 1) cluster.sync();                          // nobody reads this histogram any more
        else __syncthreads();
        prefix |= chosen[0] << shift;
        mask |= digit_mask << shift;
        left -= chosen[1];
        const uint32_t in_bin = chosen[3];
        if (pass == 2) break;
        if (parts == 1 && in_bin <= (uint32_t)FEW) {
            // few tokens share the known bits: they are gathered
            for (uint32_t i0 = warp * 32; i0 < n; i0 += THREADS) {
                const uint32_t i = i0 + lane, k = i < n ? key_at(i) : 0u;
                const bool hit = i < n && (k & mask) == prefix;
                const uint32_t m = __ballot_sync(0xFFFFFFFFu, hit);
                if (m) {
                    uint32_t at = 0;
                    if (lane == 0) at = atomicAdd(&chosen[2], (uint32_t)__popc(m));
                    at = __shfl_sync(0xFFFFFFFFu, at, 0);
                    if (hit) few[at + __popc(m & below)] = k;
                }
            }
            __syncthreads();
            // The key that `left` of them reach: every thread ranks one of them against all, threads of equal keys alike.
            if (tid < in_bin) {
                const uint32_t mine = few[tid];
                uint32_t gt = 0, ge = 0;
#pragma unroll 4
                for (uint32_t i = 0; i < in_bin; i++) {
                    gt += few[i] > mine;
                    ge += few[i] >= mine;
                }
                if (gt < left && left <= ge) {
                    chosen[0] = mine;
                    chosen[1] = left - gt;
                }
            }
            __syncthreads();
            prefix = chosen[0];
            left = chosen[1];
            break;
        }
        __syncthreads();
    }

    // ---- indices in ascending order: keys above `prefix`, and the first `left` that equal it ----
    const uint32_t seg = ((n + WARPS - 1) / WARPS + 31) / 32 * 32, w0 = min(n, warp * seg), w1 = min(n, w0 + seg);
    uint32_t gt = 0, eq = 0;
    for (uint32_t i = w0 + lane; i < w1; i += 32) {
        const uint32_t k = key_at(i);
        gt += k > prefix;
        eq += k == prefix;
    }
    gt = __reduce_add_sync(0xFFFFFFFFu, gt);
    eq = __reduce_add_sync(0xFFFFFFFFu, eq);
    if (lane == 0) {
        n_gt[warp] = gt;
        n_eq[warp] = eq;
    }
    __syncthreads();
    uint32_t gt_before = 0, eq_before = 0;
    if (parts > 1) {
        if (tid == 0) {
            uint32_t g = 0, e = 0;
            for (int w = 0; w < WARPS; w++) {
                g += n_gt[w];
                e += n_eq[w];
            }
            n_gt[WARPS] = g;
            n_eq[WARPS] = e;
        }
        cluster.sync();
        for (uint32_t r = 0; r < rank; r++) {
            gt_before += *cluster.map_shared_rank(&n_gt[WARPS], r);
            eq_before += *cluster.map_shared_rank(&n_eq[WARPS], r);
        }
    }
#pragma unroll
    for (int w = 0; w < WARPS; w++) {
        gt_before += w < (int)warp ? n_gt[w] : 0u;
        eq_before += w < (int)warp ? n_eq[w] : 0u;
    }
    uint32_t* at = out + lo + gt_before + min(eq_before, left);
    uint32_t eq_left = left - min(eq_before, left);             // of the keys that equal `prefix`, those still to come stay
    const uint32_t first = lo + begin;
    for (uint32_t i0 = w0; i0 < w1; i0 += 32) {
        const uint32_t i = i0 + lane, k = i < w1 ? key_at(i) : 0u;
        bool keep = i < w1 && k > prefix;
        const uint32_t m_eq = __ballot_sync(0xFFFFFFFFu, i < w1 && k == prefix);
        if (m_eq) {
            if ((m_eq >> lane & 1u) && (uint32_t)__popc(m_eq & below) < eq_left) keep = true;
            eq_left -= min((uint32_t)__popc(m_eq), eq_left);
        }
        const uint32_t m_keep = __ballot_sync(0xFFFFFFFFu, keep);
        if (keep) at[__popc(m_keep & below)] = first + i;
        at += __popc(m_keep);
    }
    if (parts > 1) cluster.sync();                              // a CTA's counts may still be read by its neighbours
}

// ---------------------------------------------------------------------------------------------------------------------------------
constexpr uint32_t MAX_LAYERS = 128;         // of one launch: their addresses are kernel parameters
struct CompactArgs {
    uint64_t k_layers[MAX_LAYERS], v_layers[MAX_LAYERS];
    float *k_scales, *v_scales;              // of the first layer, or null
    float* scores;                           // [layers][n_seqs][n_kv_heads][score_stride], or null
    const uint32_t *tables, *kv_lens, *kept, *new_lens;
    uint32_t* status;
    uint64_t block_stride, scale_layer;      // bytes; floats
    uint32_t row_stride, n_seqs, n_kv_heads, table_stride, max_kv_len, total_blocks, kept_stride, score_stride;
};
constexpr int CMP_THREADS = 256;

// Two E4M3 bytes of products that are at most 448: to nearest even, below 2^-6 to a signed zero like every writer of the pool (the
// conversion alone would leave subnormals there); NaN stays NaN.
__device__ __forceinline__ uint32_t encode_pair(float lo, float hi) {
    if (fabsf(lo) < 0x1p-6f) lo = __uint_as_float(__float_as_uint(lo) & 0x80000000u);
    if (fabsf(hi) < 0x1p-6f) hi = __uint_as_float(__float_as_uint(hi) & 0x80000000u);
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}

// ROW: bytes of one kv head's row.  blockIdx: x = (sequence, kv head), y = layer, z = K, V, scores.
template <int ROW, bool SCALED> __global__ void __launch_bounds__(CMP_THREADS) evict_compact(const __grid_constant__ CompactArgs a) {
    constexpr int CPR = ROW / 16, TILE = ROW == 256 ? 128 : 256, UNROLL = TILE * CPR / CMP_THREADS;
    const uint32_t tid = threadIdx.x, kvh = blockIdx.x % a.n_kv_heads, s = blockIdx.x / a.n_kv_heads, layer = blockIdx.y;
    const uint32_t len = min(a.kv_lens[s], a.max_kv_len), n_new = min(a.new_lens[s], len);
    if (tid == 0 && blockIdx.z == 0 && (a.kv_lens[s] > a.max_kv_len || a.new_lens[s] > len || (n_new < len && n_new > a.kept_stride))) report_bad(a.status);
    if (n_new == len || n_new > a.kept_stride) return;          // nothing moves
    const size_t row = ((size_t)layer * a.n_seqs + s) * a.n_kv_heads + kvh;
    const uint32_t* kept = a.kept + row * a.kept_stride;
    auto source_of = [&](uint32_t j) -> uint32_t {              // rows only move down; anything else is reported and stays
        const uint32_t k = kept[j];
        if (k >= j && k < len) return k;
        report_bad(a.status);
        return j;
    };

    if (blockIdx.z == 2) {                                      // ---- the accumulated weights move along, those behind the new end become 0 ----
        if (!a.scores) return;
        float* sc = a.scores + row * a.score_stride;
        for (uint32_t j0 = 0; j0 < n_new; j0 += 4 * CMP_THREADS) {
            float v[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const uint32_t j = j0 + i * CMP_THREADS + tid;
                v[i] = j < n_new ? sc[source_of(j)] : 0.0f;
            }
            __syncthreads();
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const uint32_t j = j0 + i * CMP_THREADS + tid;
                if (j < n_new) sc[j] = v[i];
            }
        }
        __syncthreads();
        for (uint32_t j = n_new + tid; j < len; j += CMP_THREADS) sc[j] = 0.0f;
        return;
    }

    const bool is_v = blockIdx.z == 1;
    char* base = reinterpret_cast<char*>(is_v ? a.v_layers[layer] : a.k_layers[layer]) + (size_t)kvh * ROW;
    float* scales = SCALED ? (is_v ? a.v_scales : a.k_scales) + layer * a.scale_layer + kvh : nullptr;
    const uint32_t* table = a.tables + (size_t)s * a.table_stride;
    __shared__ uint64_t from[2][TILE], to[2][TILE];
    __shared__ float ratio[2][TILE];
    constexpr uint64_t STAYS = ~0ull;
    uint32_t buf = 0;
    for (uint32_t j0 = 0; j0 < n_new; j0 += TILE, buf ^= 1u) {
        // ---- where the tile's rows come from; thread t has row t ----
        float block_scale = 0.0f;
        uint32_t scale_block = 0;
        bool new_scale = false;
        if (tid < (uint32_t)TILE) {
            const uint32_t j = j0 + tid;
            const bool live = j < n_new;
            uint64_t f = STAYS, t = 0;
            float r = 1.0f, sr = 0.0f;
            uint32_t bj = 0;
            bool moves = false;
            if (live) {
                const uint32_t k = source_of(j);
                const uint32_t bk = table[k / BS];
                bj = table[j / BS];
                if (bk < a.total_blocks && bj < a.total_blocks) {
                    moves = k != j;
                    f = (uint64_t)bk * a.block_stride + (uint64_t)(k % BS) * a.row_stride;
                    t = (uint64_t)bj * a.block_stride + (uint64_t)(j % BS) * a.row_stride;
                    if (SCALED) sr = scales[(size_t)bk * a.n_kv_heads];
                } else {
                    report_bad(a.status);
                }
            }
            if (SCALED) {                                       // the sixteen rows of a block are half a warp
                float top = sr;
#pragma unroll
                for (int o = 8; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
                if (top > 0.0f && sr != top) r = __fdiv_rn(sr, top);
                const uint32_t any = __ballot_sync(0xFFFFFFFFu, moves) >> (tid & 16u);
                block_scale = top;
                scale_block = bj;
                new_scale = (tid % BS) == 0 && (any & 0xFFFFu) != 0 && bj < a.total_blocks && live;
            }
            from[buf][tid] = moves || r != 1.0f ? f : STAYS;
            to[buf][tid] = t;
            ratio[buf][tid] = r;
        }
        __syncthreads();
        uint4 v[UNROLL];
#pragma unroll
        for (int u = 0; u < UNROLL; u++) {
            const uint32_t c = tid + u * CMP_THREADS, r = c / CPR;
            const uint64_t f = from[buf][r];
            if (f != STAYS) v[u] = *reinterpret_cast<const uint4*>(base + f + (c % CPR) * 16);
        }
        __syncthreads();                                        // the whole tile has been read
#pragma unroll
        for (int u = 0; u < UNROLL; u++) {
            const uint32_t c = tid + u * CMP_THREADS, r = c / CPR;
            if (from[buf][r] == STAYS) continue;
            if (SCALED) {
                const float f = ratio[buf][r];
                if (f != 1.0f) {
                    uint32_t w[4] = {v[u].x, v[u].y, v[u].z, v[u].w};
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        uint32_t h0, h1;
                        asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h0) : "h"((unsigned short)(w[i] & 0xFFFFu)));
                        asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h1) : "h"((unsigned short)(w[i] >> 16)));
                        const float2 x0 = __half22float2(*reinterpret_cast<__half2*>(&h0)), x1 = __half22float2(*reinterpret_cast<__half2*>(&h1));
                        w[i] = encode_pair(__fmul_rn(x0.x, f), __fmul_rn(x0.y, f)) | (encode_pair(__fmul_rn(x1.x, f), __fmul_rn(x1.y, f)) << 16);
                    }
                    v[u] = make_uint4(w[0], w[1], w[2], w[3]);
                }
            }
            *reinterpret_cast<uint4*>(base + to[buf][r] + (c % CPR) * 16) = v[u];
        }
        if (SCALED && new_scale) scales[(size_t)scale_block * a.n_kv_heads] = block_scale;
    }
}

int32_t fail(int32_t code, const char* fmt, unsigned long long x = 0, unsigned long long y = 0) {
    char buf[256];
    snprintf(buf, sizeof buf, fmt, x, y);
    return tkv_internal::set_error(code, 0, buf);
}
int32_t launch_error(const char* what, cudaError_t e) {
    cudaGetLastError();                                         // reported here, not by whoever asks next
    char buf[256];
    snprintf(buf, sizeof buf, "%s launch: %s (cuda error %d)", what, cudaGetErrorString(e), (int)e);
    return tkv_internal::set_error(TKV_ERR_CUDA, (int32_t)e, buf);
}

template <int ROW, bool SCALED> cudaError_t launch_compact(const CompactArgs& a, dim3 grid, cudaStream_t st) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(CMP_THREADS);
    cfg.stream = st;
    return cudaLaunchKernelEx(&cfg, evict_compact<ROW, SCALED>, a);
}

}  // namespace

extern "C" {

int32_t tkv_evict_select_enqueue(const TkvEvictSelect* p, void* stream) {
    if (!p) return fail(TKV_ERR_INVALID_CONFIG, "NULL argument");
    const uint64_t rows = (uint64_t)p->n_layers * p->n_seqs * p->n_kv_heads;
    if (rows == 0) return TKV_OK;
    if (!p->scores || !p->kv_lens || !p->kept || !p->new_lens) return fail(TKV_ERR_INVALID_CONFIG, "NULL buffer");
    if ((p->scores | p->kv_lens | p->protect | p->kept | p->new_lens | p->status) % 4) return fail(TKV_ERR_INVALID_CONFIG, "buffers must be 4-byte aligned");
    if (p->max_kv_len > p->score_stride)
        return fail(TKV_ERR_DIMENSION_MISMATCH, "dimension mismatch: expected %llu, got %llu (score_stride below max_kv_len)", p->max_kv_len, p->score_stride);
    // a bound that no sequence can exceed cuts none and needs no room
    const uint32_t widest = std::max(p->budget < p->max_kv_len ? p->budget : 0u, p->recent < p->max_kv_len ? p->recent : 0u);
    if (widest > p->kept_stride)
        return fail(TKV_ERR_DIMENSION_MISMATCH, "dimension mismatch: expected %llu, got %llu (kept_stride below the budget)", widest, p->kept_stride);
    // One CTA per row up to 32 768 tokens, then the smallest cluster whose CTAs have no more (64 rows of 16 384 tokens: 17 us by one CTA each, 72 by
    // clusters of four, whose barriers cost more than its CTAs save; 64 of 40 000: 33 by one CTA each, 27 by two, 47 by four).
    uint32_t cluster = 1;
    while (cluster < MAX_CLUSTER && p->max_kv_len / cluster > 32768) cluster *= 2;
    if (rows * cluster > 0x7FFFFFFFull) return fail(TKV_ERR_INVALID_CONFIG, "%llu rows: batch too large", rows);
    // every row reads its sequence's length and protection; the first one of a layer writes the new length
    const uint64_t lens_bytes = 4ull * p->n_seqs;
    auto meets = [&](uint64_t other) { return other && p->new_lens < other + lens_bytes && other < p->new_lens + lens_bytes; };
    if (meets(p->kv_lens) || meets(p->protect)) return fail(TKV_ERR_INVALID_CONFIG, "new_lens must not share memory with kv_lens or protect: every row reads those");
    const uint32_t slice = (uint32_t)(((uint64_t)p->max_kv_len + cluster - 1) / cluster);   // (a bound near 2^32 must not wrap to a small slice)
    SelectArgs a{};
    a.scores = reinterpret_cast<const float*>(p->scores);
    a.kv_lens = reinterpret_cast<const uint32_t*>(p->kv_lens);
    a.protect = reinterpret_cast<const uint32_t*>(p->protect);
    a.kept = reinterpret_cast<uint32_t*>(p->kept);
    a.new_lens = reinterpret_cast<uint32_t*>(p->new_lens);
    a.status = reinterpret_cast<uint32_t*>(p->status);
    a.n_seqs = p->n_seqs;
    a.n_kv_heads = p->n_kv_heads;
    a.max_kv_len = p->max_kv_len;
    a.score_stride = p->score_stride;
    a.kept_stride = p->kept_stride;
    a.budget = p->budget;
    a.recent = p->recent;
    a.staged = slice <= STAGE_TOKENS;
    int prev = -1;
    cudaError_t e = cudaGetDevice(&prev);
    if (e == cudaSuccess && prev != p->device) e = cudaSetDevice(p->device);
    if (e == cudaSuccess) {
        const size_t smem = a.staged ? (size_t)slice * 4 : 0;
        // 256 threads take rows six to an SM (40 registers, one value spilled), 512 a row faster: 512 x 6 000 tokens 23 us and 27, but 64 x 8 192 20 us and 14, 512 x 16 384 92 and 46
        const bool large = slice > 8192 || (rows <= 296 && slice > 1024);
        auto kernel = large ? evict_select<512> : evict_select<256>;
        if (smem > 32 * 1024) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(STAGE_TOKENS * 4));
        if (e == cudaSuccess) {
            cudaLaunchConfig_t cfg{};
            cfg.gridDim = dim3((unsigned)(rows * cluster));
            cfg.blockDim = dim3(large ? 512 : 256);
            cfg.dynamicSmemBytes = smem;
            cfg.stream = static_cast<cudaStream_t>(stream);
            cudaLaunchAttribute at[1];
            at[0].id = cudaLaunchAttributeClusterDimension;
            at[0].val.clusterDim.x = cluster;
            at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
            cfg.attrs = at;
            cfg.numAttrs = 1;
            e = cudaLaunchKernelEx(&cfg, kernel, a);
        }
    }
    if (prev >= 0 && prev != p->device) cudaSetDevice(prev);
    return e == cudaSuccess ? TKV_OK : launch_error("evict select", e);
}

int32_t tkv_evict_compact_enqueue(const TkvPool* pool, const TkvEvictCompact* p, void* stream) {
    if (!pool || !p) return fail(TKV_ERR_INVALID_CONFIG, "NULL argument");
    if (pool->dtype != TKV_DTYPE_F16 && pool->dtype != TKV_DTYPE_E4M3)
        return fail(TKV_ERR_INVALID_CONFIG, "eviction moves rows of F16 or E4M3 pools (dtype %llu)", (unsigned long long)pool->dtype);
    if (pool->head_dim != 64 && pool->head_dim != 128)
        return fail(TKV_ERR_DIMENSION_MISMATCH, "dimension mismatch: expected %llu, got %llu (eviction is built for head_dim 64 and 128)", 128, pool->head_dim);
    if (pool->block_size != BS)
        return fail(TKV_ERR_DIMENSION_MISMATCH, "dimension mismatch: expected %llu, got %llu (tokens per block)", BS, pool->block_size);
    if ((uint64_t)p->layer_begin + p->n_layers > pool->n_layers)
        return fail(TKV_ERR_INVALID_CONFIG, "layers up to %llu outside the pool (%llu layers)", (uint64_t)p->layer_begin + p->n_layers, pool->n_layers);
    if ((pool->k_scales == 0) != (pool->v_scales == 0)) return fail(TKV_ERR_INVALID_CONFIG, "k_scales and v_scales must both be set or both be 0");
    if (pool->k_scales && pool->dtype != TKV_DTYPE_E4M3) return fail(TKV_ERR_INVALID_CONFIG, "only an E4M3 pool carries scales");
    if (!p->n_seqs || !p->n_layers || !pool->n_kv_heads) return TKV_OK;
    if (!p->tables || !p->kv_lens || !p->kept || !p->new_lens || !pool->k_layer_ptrs || !pool->v_layer_ptrs) return fail(TKV_ERR_INVALID_CONFIG, "NULL buffer");
    if ((p->tables | p->kv_lens | p->kept | p->new_lens | p->scores | p->status | pool->k_scales | pool->v_scales) % 4)
        return fail(TKV_ERR_INVALID_CONFIG, "buffers must be 4-byte aligned");
    if ((p->max_kv_len + 15ull) / 16 > p->table_stride)
        return fail(TKV_ERR_DIMENSION_MISMATCH, "dimension mismatch: expected %llu, got %llu (table_stride below the blocks of max_kv_len)",
                    (p->max_kv_len + 15ull) / 16, p->table_stride);
    if (p->scores && p->max_kv_len > p->score_stride)
        return fail(TKV_ERR_DIMENSION_MISMATCH, "dimension mismatch: expected %llu, got %llu (score_stride below max_kv_len)", p->max_kv_len, p->score_stride);
    const uint64_t per_layer = (uint64_t)p->n_seqs * pool->n_kv_heads;
    if (per_layer > 0x7FFFFFFFull) return fail(TKV_ERR_INVALID_CONFIG, "%llu rows per layer: batch too large", per_layer);
    for (uint32_t l = 0; l < p->n_layers; l++) {
        const uint64_t kp = pool->k_layer_ptrs[p->layer_begin + l], vp = pool->v_layer_ptrs[p->layer_begin + l];
        if (!kp || !vp || (kp | vp) % 16) return fail(TKV_ERR_INVALID_CONFIG, "layer tensors must be set and 16-byte aligned (layer %llu)", p->layer_begin + l);
    }
    const uint32_t es = pool->dtype == TKV_DTYPE_E4M3 ? 1u : 2u, row = pool->head_dim * es;
    int prev = -1;
    cudaError_t e = cudaGetDevice(&prev);
    if (e == cudaSuccess && prev != pool->device) e = cudaSetDevice(pool->device);
    for (uint32_t l0 = 0; e == cudaSuccess && l0 < p->n_layers; l0 += MAX_LAYERS) {
        const uint32_t n = std::min(MAX_LAYERS, p->n_layers - l0);
        CompactArgs a{};
        for (uint32_t l = 0; l < n; l++) {
            a.k_layers[l] = pool->k_layer_ptrs[p->layer_begin + l0 + l];
            a.v_layers[l] = pool->v_layer_ptrs[p->layer_begin + l0 + l];
        }
        a.scale_layer = (uint64_t)pool->total_blocks * pool->n_kv_heads;
        if (pool->k_scales) {
            a.k_scales = reinterpret_cast<float*>(pool->k_scales) + (p->layer_begin + l0) * a.scale_layer;
            a.v_scales = reinterpret_cast<float*>(pool->v_scales) + (p->layer_begin + l0) * a.scale_layer;
        }
        a.scores = p->scores ? reinterpret_cast<float*>(p->scores) + l0 * per_layer * p->score_stride : nullptr;
        a.tables = reinterpret_cast<const uint32_t*>(p->tables);
        a.kv_lens = reinterpret_cast<const uint32_t*>(p->kv_lens);
        a.kept = reinterpret_cast<const uint32_t*>(p->kept) + l0 * per_layer * p->kept_stride;
        a.new_lens = reinterpret_cast<const uint32_t*>(p->new_lens);
        a.status = reinterpret_cast<uint32_t*>(p->status);
        a.row_stride = pool->n_kv_heads * row;
        a.block_stride = (uint64_t)BS * a.row_stride;
        a.n_seqs = p->n_seqs;
        a.n_kv_heads = pool->n_kv_heads;
        a.table_stride = p->table_stride;
        a.max_kv_len = p->max_kv_len;
        a.total_blocks = pool->total_blocks;
        a.kept_stride = p->kept_stride;
        a.score_stride = p->score_stride;
        const dim3 grid((unsigned)per_layer, n, a.scores ? 3 : 2);
        cudaStream_t st = static_cast<cudaStream_t>(stream);
        const bool scaled = a.k_scales != nullptr;
        if (row == 256) e = launch_compact<256, false>(a, grid, st);                    // 128 F16 dims
        else if (row == 128) e = scaled ? launch_compact<128, true>(a, grid, st) : launch_compact<128, false>(a, grid, st);
        else e = scaled ? launch_compact<64, true>(a, grid, st) : launch_compact<64, false>(a, grid, st);
    }
    if (prev >= 0 && prev != pool->device) cudaSetDevice(prev);
    return e == cudaSuccess ? TKV_OK : launch_error("evict compact", e);
}

}  // extern "C"
