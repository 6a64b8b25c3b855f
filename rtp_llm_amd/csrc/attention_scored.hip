// Paged attention with score forms, gfx950: scores capped by a tanh and biased by distance, rows that see an interval of the cache (causal, windows, prefixes,
// documents), log-sum-exps, and the attention weight that each cached token draws (what kv_evict.hip ranks them by).
//
//   u = scale q.k        s = cap tanh(u / cap)  (cap > 0, else u)        s += slope[h] (key position - row position)
//   row r, head h:  p_j = exp(s_j - lse),  lse = log sum_j exp(s_j),  out = sum_j p_j V_j   over the slots j in [begin[r], end[r]); an empty interval: out 0, lse -inf
//   weights[j, kv head] <- decay weights[j, kv head] + sum over the call's rows of the sequence and the heads of the group of p_j
#include "common.h"
#include "internal.h"
#include "scored.h"

namespace {

// ---- simple forms: a wave per (row, head)
template <int HD, bool BF, bool INT8>
__global__ __launch_bounds__(256) void scored_rows_kernel(const ScoredParams p) {
    __shared__ float qs[4][HD], ps[4][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int b = blockIdx.y, col = blockIdx.x * 4 + wave;
    int base, len;
    scored_rows_of(p, b, base, len);
    if (col >= len * p.nh) return;
    const int row = base + col / p.nh, h = col % p.nh, kh = h / p.G;
    int lo, hi;
    scored_interval(p, row, lo, hi);
    const int32_t* bt = p.block_table + (size_t)b * p.max_blocks;
    for (int d = lane; d < HD; d += 64) qs[wave][d] = act_from_bits<BF>(reinterpret_cast<const uint16_t*>(p.q)[(size_t)row * p.ldq + h * HD + d]);
    __builtin_amdgcn_wave_barrier();
    const float slope = p.slopes ? p.slopes[h] : 0.f;
    const int qp = p.slopes ? p.positions[row] : 0;
    float m = NEG_BIG, l = 0.f, o[HD / 64];
#pragma unroll
    for (int c = 0; c < HD / 64; ++c) o[c] = 0.f;
    for (int t0 = lo; t0 < hi; t0 += 64) {
        const int t = t0 + lane;
        const bool ok = t < hi;
        const int tc = ok ? t : hi - 1;
        const int blk = scored_block(p, bt, tc), ti = tc % p.page;
        const size_t hk = ((size_t)blk * 2) * p.nkv + kh, hv = hk + p.nkv;
        float s = 0.f;
        for (int d = 0; d < HD; ++d) {
            const size_t at = (hk * p.page + ti) * HD + d;
            const float k = INT8 ? (float)((int)reinterpret_cast<const uint8_t*>(p.kv_base)[at] - 128) : act_from_bits<BF>(reinterpret_cast<const uint16_t*>(p.kv_base)[at]);
            s = __builtin_fmaf(qs[wave][d], k, s);
        }
        if (INT8) s *= p.scale_base[hk * p.page + ti];
        s *= p.scale_log2;
        if (p.inv_cap > 0.f) s = p.cap_log2 * tanh_of(s * p.inv_cap);
        if (p.slopes) {
            const int kp = p.key_pos ? p.key_pos[((size_t)blk * p.nkv + kh) * p.page + ti] : tc;
            s = __builtin_fmaf(slope * kLog2e, (float)(kp - qp), s);
        }
        s = ok ? s : NEG_BIG;
        const float mn = fmaxf(m, wave_max(s)), alpha = __builtin_amdgcn_exp2f(m - mn);
        const float pe = ok ? __builtin_amdgcn_exp2f(s - mn) : 0.f;
        l = l * alpha + wave_sum(pe);
        m = mn;
        ps[wave][lane] = INT8 ? (ok ? pe * p.scale_base[hv * p.page + ti] : 0.f) : pe;
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int c = 0; c < HD / 64; ++c) o[c] *= alpha;
        const int n = min(64, hi - t0);
        for (int j = 0; j < n; ++j) {
            const int bj = __shfl(blk, j), tj = (t0 + j) % p.page;
            const size_t vb = ((size_t)bj * 2 + 1) * p.nkv + kh;
#pragma unroll
            for (int c = 0; c < HD / 64; ++c) {
                const size_t at = (vb * HD + lane + 64 * c) * p.page + tj;
                const float v = INT8 ? (float)((int)reinterpret_cast<const uint8_t*>(p.kv_base)[at] - 128) : act_from_bits<BF>(reinterpret_cast<const uint16_t*>(p.kv_base)[at]);
                o[c] = __builtin_fmaf(ps[wave][j], v, o[c]);
            }
        }
        __builtin_amdgcn_wave_barrier();
    }
    const float inv = l > 0.f ? 1.f / l : hi > lo ? __builtin_nanf("") : 0.f;
#pragma unroll
    for (int c = 0; c < HD / 64; ++c) reinterpret_cast<uint16_t*>(p.out)[((size_t)row * p.nh + h) * HD + lane + 64 * c] = act_to_bits<BF>(o[c] * inv);
    if (lane == 0 && p.lse) p.lse[(size_t)row * p.nh + h] = hi > lo ? (m + __builtin_amdgcn_logf(l)) * kLn2 : -__builtin_inff();
}

// A thread per (slot, kv head): the probabilities of all rows and heads that see it.
template <int HD, bool BF, bool INT8>
__global__ __launch_bounds__(256) void scored_weights_kernel(const ScoredParams p) {
    const int b = blockIdx.z, kh = blockIdx.y, t = blockIdx.x * 256 + threadIdx.x;
    int base, len;
    scored_rows_of(p, b, base, len);
    int reach = 0;
    for (int i = 0; i < len; ++i) { int lo, hi; scored_interval(p, base + i, lo, hi); reach = max(reach, hi); }
    if (t >= reach) return;
    const int32_t* bt = p.block_table + (size_t)b * p.max_blocks;
    const int raw = bt[t / p.page];
    if (raw < 0 || raw >= p.num_blocks) return;
    const int ti = t % p.page;
    const size_t hk = ((size_t)raw * 2) * p.nkv + kh, wat = ((size_t)raw * p.nkv + kh) * p.page + ti;
    float sum = 0.f;
    for (int i = 0; i < len; ++i) {
        int lo, hi;
        scored_interval(p, base + i, lo, hi);
        if (t < lo || t >= hi) continue;
        for (int h = kh * p.G; h < kh * p.G + p.G; ++h) {
            float s = 0.f;
            for (int d = 0; d < HD; ++d) {
                const size_t at = (hk * p.page + ti) * HD + d;
                const float k = INT8 ? (float)((int)reinterpret_cast<const uint8_t*>(p.kv_base)[at] - 128) : act_from_bits<BF>(reinterpret_cast<const uint16_t*>(p.kv_base)[at]);
                s = __builtin_fmaf(act_from_bits<BF>(reinterpret_cast<const uint16_t*>(p.q)[(size_t)(base + i) * p.ldq + h * HD + d]), k, s);
            }
            if (INT8) s *= p.scale_base[hk * p.page + ti];
            s *= p.scale_log2;
            if (p.inv_cap > 0.f) s = p.cap_log2 * tanh_of(s * p.inv_cap);
            if (p.slopes) s = __builtin_fmaf(p.slopes[h] * kLog2e, (float)((p.key_pos ? p.key_pos[wat] : t) - p.positions[base + i]), s);
            sum += __builtin_amdgcn_exp2f(s - p.lse[(size_t)(base + i) * p.nh + h] * kLog2e);
        }
    }
    p.weights[wat] = scored_decayed(p, p.weights[wat], sum);
}

} // namespace

extern "C" size_t mi355_paged_attn_scored_workspace_bytes(int32_t B, int32_t q_len, int32_t rows, int32_t nh, int32_t nkv, int32_t hd, int32_t max_seq_len, int32_t track) {
    if (B <= 0 || q_len <= 0 || rows <= 0 || nh <= 0 || nkv <= 0 || hd <= 0 || max_seq_len <= 0) return 0;
    return track ? (size_t)rows * nh * sizeof(float) : 0;
}

extern "C" int mi355_paged_attn_scored(const void* q, int32_t ldq, const mi355_kv_layer_t* kv, const int32_t* block_table, int32_t max_blocks_per_seq,
                                       const int32_t* row_start, int32_t B, int32_t q_len, int32_t rows, int32_t nh, const mi355_attn_score_t* score,
                                       int32_t max_seq_len, void* out, float* lse, float* weights, float decay, void* workspace, size_t workspace_bytes,
                                       mi355_stream_t stream) {
    ScoredParams p;
    const int rc = scored_params(p, q, ldq, kv, block_table, max_blocks_per_seq, row_start, B, q_len, rows, nh, score, max_seq_len, out, lse, weights, decay);
    if (rc != MI355_OK) return rc;
    const size_t need = mi355_paged_attn_scored_workspace_bytes(B, q_len, rows, nh, kv->nkv, kv->hd, max_seq_len, weights != nullptr);
    if (need && (need > workspace_bytes || !workspace)) {
        mi355_set_error("paged_attn_scored: workspace %zu < %zu", workspace_bytes, need);
        return MI355_ERR_WORKSPACE;
    }
    if (weights && !lse) p.lse = (float*)workspace;
    const bool bf = kv->act_dtype == MI355_ACT_BF16, int8 = kv->kv_dtype == MI355_KV_INT8;
    hipStream_t st = (hipStream_t)stream;
    const dim3 grid(cdiv(q_len * nh, 4), B), wgrid(cdiv(max_seq_len, 256), kv->nkv, B);
#define L_(HD_, BF_, I8_) do { hipLaunchKernelGGL((scored_rows_kernel<HD_, BF_, I8_>), grid, dim3(256), 0, st, p); \
                               if (weights) hipLaunchKernelGGL((scored_weights_kernel<HD_, BF_, I8_>), wgrid, dim3(256), 0, st, p); } while (0)
#define LB_(HD_) do { if (bf) { if (int8) L_(HD_, true, true); else L_(HD_, true, false); } else { if (int8) L_(HD_, false, true); else L_(HD_, false, false); } } while (0)
    if (kv->hd == 128) LB_(128); else LB_(64);
#undef LB_
#undef L_
    MI355_CHECK_LAUNCH("paged_attn_scored");
    return MI355_OK;
}
