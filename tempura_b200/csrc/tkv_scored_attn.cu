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

#include <algorithm>
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

struct FinishArgs {
    const float *part_o, *part_ml, *logits;
    const uint32_t *plan, *kv_lens;
    float* scores;
    void* out;
    uint32_t n_seqs, n_q_heads, n_kv_heads, group, logit_stride, score_stride, max_kv_len, tasks, v4;
    float decay;
};

// Tokens per thread of the second kernel: their scores of all G query heads wait in registers (16 sequences of up to 4 096 tokens: 2 with
// eight query heads 47 us for the whole call, 4 49 us; with four query heads 42.6 and 42.3).
__host__ __device__ constexpr int tokens_of(int g) { return g > 4 ? 2 : 4; }

// One CTA per (sequence, kv head, task): the first G tasks join the partial results of one query head each, the others turn the scores of 256 x TOK tokens into weights.  Bound by latency and L2:
// everything it reads was written just before, so a thread asks for its scores before it joins the maxima and sums, and asks
// for all of those at once.  v4: rows of accumulated weights are aligned to 16 bytes, so that a thread stores its tokens together.
template <int D, bool F32, int G> __global__ void __launch_bounds__(256) scored_finish(const FinishArgs a) {
    constexpr int TOK = tokens_of(G);
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u;
    const uint32_t task = blockIdx.x % a.tasks, row = blockIdx.x / a.tasks, kvh = row % a.n_kv_heads, s = row / a.n_kv_heads;
    const bool join = task < (uint32_t)G;
    constexpr uint32_t RUN = 256 * TOK;
    const uint32_t skip = (a.tasks - G) * RUN;
    uint32_t t0 = join ? 0u : (task - G) * RUN;
    asm volatile("griddepcontrol.wait;" ::: "memory");          // launched ahead of the first kernel's end
    const uint32_t len = min(a.kv_lens[s], a.max_kv_len);
    const uint32_t share = a.plan[0], lo = a.plan[1 + s], hi = a.plan[2 + s];
    const float* src = a.logits + ((size_t)s * a.n_q_heads + kvh * G) * a.logit_stride + TOK * tid;
    auto read = [&](float (&x)[G][TOK], uint32_t at) {          // rows of x are padded to 16 tokens: a vector stays inside; what lies behind len is not used
        if (at + TOK * tid < a.logit_stride) {
#pragma unroll
            for (int g = 0; g < G; g++) {
                if (TOK == 4) {
                    const float4 v = *reinterpret_cast<const float4*>(src + (size_t)g * a.logit_stride + at);
                    x[g][0] = v.x;
                    x[g][1] = v.y;
                    x[g][TOK - 2] = v.z;
                    x[g][TOK - 1] = v.w;
                } else {
                    const float2 v = *reinterpret_cast<const float2*>(src + (size_t)g * a.logit_stride + at);
                    x[g][0] = v.x;
                    x[g][1] = v.y;
                }
            }
        }
    };
    float x[G][TOK];
    if (!join) read(x, t0);
    if (!join && t0 >= len) return;
    const uint32_t p0 = hi > lo ? lo / share : 0u, n = hi > lo ? ((hi - 1) / share - p0 + 1) : 0u;
    const size_t first = p0 + s;                               // partial results first .. first + n - 1
    __shared__ float top[8], inv[8];
    if (warp < (uint32_t)G && (!join || warp == task)) { // warp g: maximum and sum of query head g
        float m = -INFINITY, l = 0.0f;
        const float2* ml = reinterpret_cast<const float2*>(a.part_ml) + first * a.n_q_heads + kvh * G + warp;
        for (uint32_t i0 = 0; i0 < n; i0 += 256) {
            float2 v[8];
#pragma unroll
            for (int k = 0; k < 8; k++) {
                const uint32_t i = i0 + 32 * k + lane;
                v[k] = i < n ? ml[(size_t)i * a.n_q_heads] : make_float2(-INFINITY, 0.0f);
            }
#pragma unroll
            for (int k = 0; k < 8; k++) {
                const float mm = fmaxf(m, v[k].x);
                l = mm == -INFINITY ? l + v[k].y : l * exp2_fast(m - mm) + v[k].y * exp2_fast(v[k].x - mm);   // scores all NaN: the sum says so
                m = mm;
            }
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
        const uint32_t head = task;
        const float m = top[head];
#pragma unroll 8
        for (uint32_t i = warp; i < n; i += 8) {
            const size_t r = (first + i) * a.n_q_heads + kvh * G + head;
            const float2 ml = *reinterpret_cast<const float2*>(a.part_ml + r * 2);
            float v[PER];
#pragma unroll
            for (int k = 0; k < PER; k++) v[k] = a.part_o[r * D + k * 32 + lane];
            const float f = exp2_fast(ml.x - m);
#pragma unroll
            for (int k = 0; k < PER; k++) acc[k] = ml.x != -INFINITY || ml.y != 0.0f ? __fmaf_rn(f, v[k], acc[k]) : acc[k];   // an empty part's O counts for nothing
        }
        const size_t at = ((size_t)s * a.n_q_heads + kvh * G + head) * D;
        __shared__ float part[8][D];
#pragma unroll
        for (int k = 0; k < PER; k++) part[warp][k * 32 + lane] = acc[k];
        __syncthreads();
        if (tid < D) {
            float v = 0.0f;
#pragma unroll
            for (int w8 = 0; w8 < 8; w8++) v += part[w8][tid];
            v *= inv[head];
            if (F32) reinterpret_cast<float*>(a.out)[at + tid] = v;
            else reinterpret_cast<__half*>(a.out)[at + tid] = __float2half_rn(v);
        }
    } else {
        float* sc = a.scores + ((size_t)s * a.n_kv_heads + kvh) * a.score_stride + TOK * tid;
        for (;; t0 += skip) {
            const uint32_t t = t0 + TOK * tid;
            float w[TOK], y[G][TOK];
#pragma unroll
            for (int i = 0; i < TOK; i++) w[i] = a.decay != 0.0f && t + i < len ? a.decay * sc[t0 + i] : 0.0f;
#pragma unroll
            for (int g = 0; g < G; g++)
#pragma unroll
                for (int i = 0; i < TOK; i++) y[g][i] = x[g][i];
            const bool more = t0 + skip < len;
            if (more) read(x, t0 + skip);                       // the next run's, under this run's arithmetic
#pragma unroll
            for (int g = 0; g < G; g++) {
                const float m = top[g], f = inv[g];
#pragma unroll
                for (int i = 0; i < TOK; i++) w[i] = __fmaf_rn(exp2_fast(y[g][i] - m), f, w[i]);
            }
            if (a.v4 && t + TOK <= len) {
                if (TOK == 4) *reinterpret_cast<float4*>(sc + t0) = make_float4(w[0], w[1], w[TOK - 2], w[TOK - 1]);
                else *reinterpret_cast<float2*>(sc + t0) = make_float2(w[0], w[1]);
            } else {
#pragma unroll
                for (int i = 0; i < TOK; i++)
                    if (t + i < len) sc[t0 + i] = w[i];
            }
            if (!more) break;
        }
    }
}

template <int D, bool F32, int G> cudaError_t launch_finish_g(const FinishArgs& a, unsigned grid, cudaStream_t st) {
    // The launch does not wait for the first kernel's end (the kernel itself does): its CTAs are in place when the last partial result is written.
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(256);
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, scored_finish<D, F32, G>, a);
}
template <int D, bool F32> cudaError_t launch_finish(const FinishArgs& a, unsigned grid, cudaStream_t st) {
    switch (a.group) {
        case 1: return launch_finish_g<D, F32, 1>(a, grid, st);
        case 2: return launch_finish_g<D, F32, 2>(a, grid, st);
        case 3: return launch_finish_g<D, F32, 3>(a, grid, st);
        case 4: return launch_finish_g<D, F32, 4>(a, grid, st);
        case 5: return launch_finish_g<D, F32, 5>(a, grid, st);
        case 6: return launch_finish_g<D, F32, 6>(a, grid, st);
        case 7: return launch_finish_g<D, F32, 7>(a, grid, st);
        default: return launch_finish_g<D, F32, 8>(a, grid, st);
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
    const uint64_t slots = (uint64_t)l.split.parts + n_seqs;                // part p and sequence s meet in slot p + s
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
    const float scale_log2 = p->sm_scale * 1.4426950408889634f;
    if (!std::isfinite(scale_log2)) return fail(TKV_ERR_INVALID_CONFIG, "sm_scale x log2(e) is not finite");
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
    const uint32_t group = p->n_q_heads / pool->n_kv_heads, run = 256 * tokens_of((int)group), runs = (p->max_kv_len + run - 1) / run;
    // four CTAs per SM turn scores into weights where there are rows and runs for them
    const uint64_t rows = (uint64_t)p->n_seqs * pool->n_kv_heads;
    const uint32_t per_row = (uint32_t)std::min<uint64_t>(runs, std::max<uint64_t>(4ull * CTAS / rows, 1ull)), tasks = group + per_row;
    const uint64_t finish_grid = rows * tasks;
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
    a.scale_log2 = scale_log2;
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
    f.v4 = p->scores % 16 == 0 && p->score_stride % 4 == 0;
    f.decay = p->decay;

    int prev = -1;
    cudaError_t e = cudaGetDevice(&prev);
    if (e == cudaSuccess && prev != pool->device) e = cudaSetDevice(pool->device);
    if (e == cudaSuccess) {
        cudaStream_t st = static_cast<cudaStream_t>(stream);
        const bool f32 = p->q_dtype == TKV_DTYPE_F32;
        e = tkv_rows::launch_rows(pool->head_dim, es == 1, f32, a, l.split, false, st);
        if (e == cudaSuccess) {
            const unsigned grid = (unsigned)finish_grid;
            if (pool->head_dim == 128) e = f32 ? launch_finish<128, true>(f, grid, st) : launch_finish<128, false>(f, grid, st);
            else e = f32 ? launch_finish<64, true>(f, grid, st) : launch_finish<64, false>(f, grid, st);
        }
    }
    if (prev >= 0 && prev != pool->device) cudaSetDevice(prev);
    if (e != cudaSuccess) {
        cudaGetLastError();                                     // reported here, not by whoever asks next
        char buf[256];
        snprintf(buf, sizeof buf, "scored attention launch: %s (cuda error %d)", cudaGetErrorString(e), (int)e);
        return tkv_internal::set_error(TKV_ERR_CUDA, (int32_t)e, buf);
    }
    return TKV_OK;
}

}  // extern "C"
