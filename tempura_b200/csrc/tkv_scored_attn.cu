// Decode attention that also accumulates, per cached token and kv head, how much softmax weight it received: the measure by which
// tkv_evict_* decides what a full cache gives up.
//
//   w[g][t] = 2^(x[g][t] - M[g]) / L[g],   out = sum_t w[g][t] v[t],   scores[t] = decay * scores[t] + sum_g w[g][t]
//
// with x the scaled scores in the log2 domain.  A weight needs the row's final maximum and sum, which exist only when the last
// token has been seen.  Reading K a second time for it would cost half the traffic again; instead the first kernel (rows_attn)
// leaves x in F32 (4 bytes per query head and token against 4 x head_dim of an F16 cache row shared by the group) and the second
// one joins the partial results and turns x into weights.  Sums, maxima, x and scores are F32 throughout.
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cmath>
#include <cstdio>
#include <stdint.h>

#include "../../include/tkv.h"
#include "tkv_rows_attn.cuh"

namespace tkv_internal {
int32_t set_error(int32_t code, int32_t cuda_code, const char* text);
}

namespace {

using tkv_rows::exp2_fast;

constexpr uint32_t CTAS = 148;               // one per SM of the part this is built for; partial results are sized by it
constexpr int CHUNK = 1024;                  // tokens per CTA of the second kernel

struct FinishArgs {
    const float *part_o, *part_ml, *logits;
    const uint32_t *plan, *kv_lens;
    float* scores;
    void* out;
    uint32_t n_seqs, n_q_heads, n_kv_heads, group, logit_stride, score_stride, max_kv_len, tasks, subs;
    float decay;
};

// One CTA per (sequence, kv head, task): the first `group` tasks join the partial results of one query head, the others turn the
// scores of CHUNK tokens into weights.  Bound by L2 and launch: everything it reads was written just before.
template <int D, bool F32> __global__ void __launch_bounds__(256) scored_finish(const FinishArgs a) {
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u;
    const uint32_t task = blockIdx.x % a.tasks, row = blockIdx.x / a.tasks, kvh = row % a.n_kv_heads, s = row / a.n_kv_heads;
    const uint32_t len = min(a.kv_lens[s], a.max_kv_len);
    const bool join = task < a.group;
    const uint32_t t0 = join ? 0u : (task - a.group) * CHUNK;
    if (!join && t0 >= len) return;
    const float* x = a.logits + ((size_t)s * a.n_q_heads + kvh * a.group) * a.logit_stride;
    float xs[CHUNK / 256][8];                // asked for before the partial results are joined: one latency instead of two
    if (!join) {
#pragma unroll
        for (int i = 0; i < CHUNK / 256; i++) {
            const uint32_t t = t0 + i * 256 + tid;
#pragma unroll
            for (uint32_t g = 0; g < 8; g++) xs[i][g] = g < a.group && t < len ? x[(size_t)g * a.logit_stride + t] : -INFINITY;
        }
    }
    const uint32_t share = a.plan[0], lo = a.plan[1 + s], hi = a.plan[2 + s];
    const uint32_t p0 = hi > lo ? lo / share : 0u, n = hi > lo ? ((hi - 1) / share - p0 + 1) * a.subs : 0u;
    const size_t first = (size_t)(p0 + s) * a.subs;     // partial results first .. first + n - 1
    __shared__ float top[8], inv[8];
    if (warp < a.group && (!join || warp == task)) {            // warp g: maximum and sum of query head g
        float m = -INFINITY, l = 0.0f;
        const float2* ml = reinterpret_cast<const float2*>(a.part_ml) + first * a.n_q_heads + kvh * a.group + warp;
        for (uint32_t i = lane; i < n; i += 32) {
            const float2 v = ml[(size_t)i * a.n_q_heads];
            const float mm = fmaxf(m, v.x);
            if (mm != -INFINITY) l = l * exp2_fast(m - mm) + v.y * exp2_fast(v.x - mm);
            else l += v.y;                                      // a part whose scores are all -inf or NaN says so in its sum
            m = mm;
        }
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) {
            const float m_o = __shfl_xor_sync(0xFFFFFFFFu, m, off), l_o = __shfl_xor_sync(0xFFFFFFFFu, l, off);
            const float mm = fmaxf(m, m_o);
            l = mm == -INFINITY ? l + l_o : l * exp2_fast(m - mm) + l_o * exp2_fast(m_o - mm);
            m = mm;
        }
        if (lane == 0) {
            top[warp] = m == -INFINITY ? 0.0f : m;
            inv[warp] = l == 0.0f ? 0.0f : 1.0f / l;            // an empty row: weights and output 0
        }
    }
    __syncthreads();
    if (join) {
        constexpr int PER = D / 32;
        float acc[PER];
#pragma unroll
        for (int i = 0; i < PER; i++) acc[i] = 0.0f;
        const float m = top[task];
        for (uint32_t i = warp; i < n; i += 8) {
            const size_t r = (first + i) * a.n_q_heads + kvh * a.group + task;
            const float2 ml = *reinterpret_cast<const float2*>(a.part_ml + r * 2);
            float v[PER];
#pragma unroll
            for (int k = 0; k < PER; k++) v[k] = a.part_o[r * D + k * 32 + lane];
            const float f = exp2_fast(ml.x - m);
            if (ml.x != -INFINITY || ml.y != 0.0f) {            // an empty part's O was never written
#pragma unroll
                for (int k = 0; k < PER; k++) acc[k] += f * v[k];
            }
        }
        __shared__ float part[8][D];
#pragma unroll
        for (int k = 0; k < PER; k++) part[warp][k * 32 + lane] = acc[k];
        __syncthreads();
        if (tid < D) {
            float v = 0.0f;
#pragma unroll
            for (int w = 0; w < 8; w++) v += part[w][tid];
            v *= inv[task];
            const size_t at = ((size_t)s * a.n_q_heads + kvh * a.group + task) * D + tid;
            if (F32) reinterpret_cast<float*>(a.out)[at] = v;
            else reinterpret_cast<__half*>(a.out)[at] = __float2half_rn(v);
        }
    } else {
        float* sc = a.scores + ((size_t)s * a.n_kv_heads + kvh) * a.score_stride;
#pragma unroll
        for (int i = 0; i < CHUNK / 256; i++) {
            const uint32_t t = t0 + i * 256 + tid;
            if (t < len) {
                float w = 0.0f;
#pragma unroll
                for (uint32_t g = 0; g < 8; g++)
                    if (g < a.group) w += exp2_fast(xs[i][g] - top[g]) * inv[g];
                sc[t] = a.decay == 0.0f ? w : a.decay * sc[t] + w;
            }
        }
    }
}

int32_t fail(int32_t code, const char* fmt, unsigned long long x = 0, unsigned long long y = 0) {
    char buf[256];
    snprintf(buf, sizeof buf, fmt, x, y);
    return tkv_internal::set_error(code, 0, buf);
}
uint64_t up(uint64_t x, uint64_t to) { return (x + to - 1) / to * to; }

struct Layout {
    tkv_rows::Split split;
    uint64_t ml, o, logits, bytes;           // offsets; the plan is at 0
    uint32_t logit_stride;
};
Layout layout_of(uint32_t n_seqs, uint32_t n_q_heads, uint32_t n_kv_heads, uint32_t head_dim, uint32_t max_kv_len) {
    Layout l;
    l.split = tkv_rows::split_for((uint64_t)n_seqs * ((max_kv_len + 15ull) / 16), n_kv_heads, CTAS);
    const uint64_t slots = ((uint64_t)l.split.parts + n_seqs) * 2;          // an E4M3 pool's slots hold two partial results
    l.logit_stride = (uint32_t)up(max_kv_len, 16);
    l.ml = up(4ull * (n_seqs + 2ull), 256);
    l.o = l.ml + up(slots * n_q_heads * 8ull, 256);
    l.logits = l.o + up(slots * n_q_heads * head_dim * 4ull, 256);
    l.bytes = l.logits + (uint64_t)n_seqs * n_q_heads * l.logit_stride * 4ull;
    return l;
}

}  // namespace

extern "C" {

uint64_t tkv_scored_attn_scratch_bytes(uint32_t n_seqs, uint32_t n_q_heads, uint32_t n_kv_heads, uint32_t head_dim, uint32_t max_kv_len) {
    if (!n_seqs || !n_kv_heads || max_kv_len > 0xFFFFFFF0u) return 0;
    return layout_of(n_seqs, n_q_heads, n_kv_heads, head_dim, max_kv_len).bytes;
}

int32_t tkv_scored_attn_enqueue(const TkvPool* pool, const TkvScoredAttn* p, void* stream) {
    if (!pool || !p) return fail(TKV_ERR_INVALID_CONFIG, "NULL argument");
    if (pool->dtype != TKV_DTYPE_F16 && pool->dtype != TKV_DTYPE_E4M3)
        return fail(TKV_ERR_INVALID_CONFIG, "scored attention reads F16 or E4M3 pools (dtype %llu)", (unsigned long long)pool->dtype);
    if (p->q_dtype != TKV_DTYPE_F16 && p->q_dtype != TKV_DTYPE_F32)
        return fail(TKV_ERR_INVALID_CONFIG, "q and out are F16 or F32 (dtype %llu)", (unsigned long long)p->q_dtype);
    if (pool->head_dim != 64 && pool->head_dim != 128)
        return fail(TKV_ERR_DIMENSION_MISMATCH, "dimension mismatch: expected %llu, got %llu (scored attention is built for head_dim 64 and 128)", 128,
                    pool->head_dim);
    if (pool->block_size != tkv_rows::BS)
        return fail(TKV_ERR_DIMENSION_MISMATCH, "dimension mismatch: expected %llu, got %llu (tokens per block)", tkv_rows::BS, pool->block_size);
    if (p->layer >= pool->n_layers) return fail(TKV_ERR_INVALID_CONFIG, "layer %llu outside the pool (%llu layers)", p->layer, pool->n_layers);
    if (!pool->n_kv_heads || !p->n_q_heads || p->n_q_heads % pool->n_kv_heads || p->n_q_heads / pool->n_kv_heads > 8)
        return fail(TKV_ERR_DIMENSION_MISMATCH, "dimension mismatch: expected %llu, got %llu (query heads must be 1..8 times the kv heads)",
                    pool->n_kv_heads, p->n_q_heads);
    if (pool->n_kv_heads > CTAS * tkv_rows::WARPS) return fail(TKV_ERR_INVALID_CONFIG, "at most %llu kv heads (%llu)", CTAS * tkv_rows::WARPS, pool->n_kv_heads);
    if ((pool->k_scales == 0) != (pool->v_scales == 0)) return fail(TKV_ERR_INVALID_CONFIG, "k_scales and v_scales must both be set or both be 0");
    if (pool->k_scales && pool->dtype != TKV_DTYPE_E4M3) return fail(TKV_ERR_INVALID_CONFIG, "only an E4M3 pool carries scales");
    if (!std::isfinite(p->sm_scale)) return fail(TKV_ERR_INVALID_CONFIG, "sm_scale is not finite");
    if (!(p->decay >= 0.0f && p->decay <= 1.0f)) return fail(TKV_ERR_INVALID_CONFIG, "decay must lie in [0, 1]");
    if (p->n_seqs == 0) return TKV_OK;
    if (!p->q || !p->out || !p->tables || !p->kv_lens || !p->scores || !pool->k_layer_ptrs || !pool->v_layer_ptrs || !pool->total_blocks)
        return fail(TKV_ERR_INVALID_CONFIG, "NULL buffer");
    if (p->max_kv_len > 0xFFFFFFF0u || (uint64_t)p->n_seqs * ((p->max_kv_len + 15ull) / 16) >= 0x7FFFFFFFull)
        return fail(TKV_ERR_INVALID_CONFIG, "%llu sequences of %llu tokens: more than 2^31 blocks", p->n_seqs, p->max_kv_len);
    if ((p->max_kv_len + 15ull) / 16 > p->table_stride)
        return fail(TKV_ERR_DIMENSION_MISMATCH, "dimension mismatch: expected %llu, got %llu (table_stride below the blocks of max_kv_len)",
                    (p->max_kv_len + 15ull) / 16, p->table_stride);
    if (p->max_kv_len > p->score_stride)
        return fail(TKV_ERR_DIMENSION_MISMATCH, "dimension mismatch: expected %llu, got %llu (score_stride below max_kv_len)", p->max_kv_len, p->score_stride);
    const uint64_t kp = pool->k_layer_ptrs[p->layer], vp = pool->v_layer_ptrs[p->layer];
    if (!kp || !vp) return fail(TKV_ERR_INVALID_CONFIG, "NULL buffer");
    if ((kp | vp | p->q | p->out) % 16 || p->scratch % 256) return fail(TKV_ERR_INVALID_CONFIG, "layer tensors, q and out must be 16-byte aligned, scratch 256-byte");
    if ((p->tables | p->kv_lens | p->scores | p->status | pool->k_scales | pool->v_scales) % 4)
        return fail(TKV_ERR_INVALID_CONFIG, "tables, lengths, scores, scales and status must be 4-byte aligned");
    const Layout l = layout_of(p->n_seqs, p->n_q_heads, pool->n_kv_heads, pool->head_dim, p->max_kv_len);
    if (!p->scratch || p->scratch_bytes < l.bytes)
        return fail(TKV_ERR_DIMENSION_MISMATCH, "dimension mismatch: expected %llu, got %llu (scratch bytes)", l.bytes, p->scratch ? p->scratch_bytes : 0);
    const uint32_t group = p->n_q_heads / pool->n_kv_heads, tasks = group + (p->max_kv_len + CHUNK - 1) / CHUNK;
    const uint64_t finish_grid = (uint64_t)p->n_seqs * pool->n_kv_heads * tasks;
    if (finish_grid > 0x7FFFFFFFull) return fail(TKV_ERR_INVALID_CONFIG, "%llu sequences of %llu tokens: batch too large", p->n_seqs, p->max_kv_len);

    tkv_rows::Args a{};
    const uint32_t es = pool->dtype == TKV_DTYPE_E4M3 ? 1u : 2u;
    const size_t layer_scales = (size_t)p->layer * pool->total_blocks * pool->n_kv_heads;
    a.k_base = reinterpret_cast<const char*>(kp);
    a.v_base = reinterpret_cast<const char*>(vp);
    a.k_scales = pool->k_scales ? reinterpret_cast<const float*>(pool->k_scales) + layer_scales : nullptr;
    a.v_scales = pool->v_scales ? reinterpret_cast<const float*>(pool->v_scales) + layer_scales : nullptr;
    a.q = reinterpret_cast<const void*>(p->q);
    a.tables = reinterpret_cast<const uint32_t*>(p->tables);
    a.kv_lens = reinterpret_cast<const uint32_t*>(p->kv_lens);
    a.plan = reinterpret_cast<uint32_t*>(p->scratch);
    a.part_ml = reinterpret_cast<float*>(p->scratch + l.ml);
    a.part_o = reinterpret_cast<float*>(p->scratch + l.o);
    a.logits = reinterpret_cast<float*>(p->scratch + l.logits);
    a.status = reinterpret_cast<uint32_t*>(p->status);
    a.row_stride = pool->n_kv_heads * pool->head_dim * es;
    a.block_stride = (uint64_t)tkv_rows::BS * a.row_stride;
    a.n_seqs = p->n_seqs;
    a.n_q_heads = p->n_q_heads;
    a.n_kv_heads = pool->n_kv_heads;
    a.group = group;
    a.table_stride = p->table_stride;
    a.max_kv_len = p->max_kv_len;
    a.total_blocks = pool->total_blocks;
    a.logit_stride = l.logit_stride;
    a.scale_log2 = p->sm_scale * 1.4426950408889634f;
    FinishArgs f{};
    f.part_o = a.part_o;
    f.part_ml = a.part_ml;
    f.logits = a.logits;
    f.plan = a.plan;
    f.kv_lens = a.kv_lens;
    f.scores = reinterpret_cast<float*>(p->scores);
    f.out = reinterpret_cast<void*>(p->out);
    f.n_seqs = p->n_seqs;
    f.n_q_heads = p->n_q_heads;
    f.n_kv_heads = pool->n_kv_heads;
    f.group = group;
    f.logit_stride = l.logit_stride;
    f.score_stride = p->score_stride;
    f.max_kv_len = p->max_kv_len;
    f.tasks = tasks;
    f.subs = tkv_rows::subs_of(es == 1, p->q_dtype == TKV_DTYPE_F32);
    f.decay = p->decay;

    int prev = -1;
    cudaError_t e = cudaGetDevice(&prev);
    if (e == cudaSuccess && prev != pool->device) e = cudaSetDevice(pool->device);
    if (e == cudaSuccess) {
        cudaStream_t st = static_cast<cudaStream_t>(stream);
        const bool f32 = p->q_dtype == TKV_DTYPE_F32;
        e = tkv_rows::launch_rows(pool->head_dim, es == 1, f32, a, l.split, st);
        if (e == cudaSuccess) {
            const unsigned grid = (unsigned)finish_grid;
            if (pool->head_dim == 128) {
                if (f32) scored_finish<128, true><<<grid, 256, 0, st>>>(f);
                else scored_finish<128, false><<<grid, 256, 0, st>>>(f);
            } else {
                if (f32) scored_finish<64, true><<<grid, 256, 0, st>>>(f);
                else scored_finish<64, false><<<grid, 256, 0, st>>>(f);
            }
            e = cudaGetLastError();
        }
    }
    if (prev >= 0 && prev != pool->device) cudaSetDevice(prev);
    if (e != cudaSuccess) {
        char buf[256];
        snprintf(buf, sizeof buf, "scored attention launch: %s (cuda error %d)", cudaGetErrorString(e), (int)e);
        return tkv_internal::set_error(TKV_ERR_CUDA, (int32_t)e, buf);
    }
    return TKV_OK;
}

}  // extern "C"
