// What the launches of paged attention with score forms share: arguments, their checks, intervals of rows, the score's form.
#pragma once
#include "common.h"

namespace {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f, NEG_BIG = -1e30f;

struct ScoredParams {
    const void*    q;
    const void*    kv_base;
    const float*   scale_base;
    const int32_t* block_table;
    const int32_t* row_start;      // null: sequence b has the rows b q_len ..
    const int32_t *begin, *end;    // slots that a row sees (begin null: 0)
    const float*   slopes;
    const int32_t *positions, *key_pos;
    void*          out;
    float*         lse;
    float*         weights;
    float          scale1;         // of a product of q and k: scale log2(e); capped: scale / cap
    float          cap_log2;       // capped: cap log2(e), of the tanh
    float          decay;
    int            capped;
    int            ldq, max_blocks, B, q_len, rows, nh, nkv, G, page, num_blocks, max_seq;
    uint32_t       page_magic;     // 2^32 / page + 1: floor(t / page) = (t magic) >> 32 for t page < 2^32
};

// Rows of a sequence.  row_start is device data: whatever it holds, the rows are at most q_len and lie inside q.
__device__ __forceinline__ void scored_rows_of(const ScoredParams& p, int b, int& base, int& len) {
    base = b * p.q_len; len = p.q_len;
    if (p.row_start) {
        base = min(max(p.row_start[b], 0), p.rows);
        len = min(min(max(p.row_start[b + 1] - base, 0), p.q_len), p.rows - base);
    }
}
// [lo, hi) of a row, inside the cache; nothing seen: lo = hi = 0
__device__ __forceinline__ void scored_interval(const ScoredParams& p, int row, int& lo, int& hi) {
    hi = min(max(p.end[row], 0), p.max_seq);
    lo = p.begin ? max(p.begin[row], 0) : 0;
    if (lo >= hi) lo = hi = 0;
}
// Block of slot t, clamped into the pool.
__device__ __forceinline__ int scored_block(const ScoredParams& p, const int32_t* bt, int t) {
    return min(max(bt[(int)(((unsigned long long)(unsigned)t * p.page_magic) >> 32)], 0), p.num_blocks - 1);
}

// The position that a row's biases are taken from: that of its last seen slot, the newest token's as a rule.  Scores so stay small next to the keys that matter, however far the row's
// position is; the log-sum-exp gets the rest, slope (reference - row position), at the end.  A row's own: with one for all rows of a sequence or tile, those that see slots far from it lose what
// the bias between rounds away (slope 0.5, 60000 slots: 2e-3 of a weight).
__device__ __forceinline__ int scored_ref(const ScoredParams& p, int b, int kh, int hi) {
    if (!p.key_pos) return hi - 1;
    const int blk = scored_block(p, p.block_table + (size_t)b * p.max_blocks, hi - 1);
    return p.key_pos[((size_t)blk * p.nkv + kh) * p.page + (hi - 1) % p.page];
}
__device__ __forceinline__ float scored_shift(const ScoredParams& p, int row, int h, int ref) { return p.slopes ? p.slopes[h] * (float)(ref - p.positions[row]) : 0.f; }

// A slot's weight after the call.  decay 0 takes nothing of what was there, NaN included.
__device__ __forceinline__ float scored_decayed(const ScoredParams& p, float old, float sum) {
    return p.decay == 0.f ? sum : __builtin_fmaf(old, p.decay, sum);
}

// tanh.  Up to 0.625 a polynomial (u + u z P(z), z = u^2, P of degree 4 fitted to (tanh(u) / u - 1) / z: with its coefficients in fp32 8.6e-9 relative at worst), beyond (1 - t) / (1 + t) with
// t = exp(-2 |u|).  The quotient alone loses, next to 0, what a cap of 50 multiplies: 3e-6 of a score of 5, and of its weight.  Scores far below their cap are the common ones,
// and the polynomial is 7 full-rate instructions where the quotient takes two quarter-rate ones more: a wave forms the quotient only if one of its scores needs it.
constexpr float kTanhNear = 0.625f;
__device__ __forceinline__ float tanh_near(float u) {
    const float z = u * u;
    float r = -0.005704986397f;
    r = __builtin_fmaf(r, z, 0.02063908614f);
    r = __builtin_fmaf(r, z, -0.05373971537f);
    r = __builtin_fmaf(r, z, 0.13331441581f);
    r = __builtin_fmaf(r, z, -0.33333280683f);
    return __builtin_fmaf(u * z, r, u);
}
__device__ __forceinline__ float tanh_far(float u) {
    const float t = __builtin_amdgcn_exp2f(fabsf(u) * (-2.f * kLog2e));
    return __builtin_copysignf((1.f - t) * __builtin_amdgcn_rcpf(1.f + t), u);
}
// tanh of N scores, the quotient formed only where one of the wave's needs it.
template <int N> __device__ __forceinline__ void tanh_all(float (&u)[N]) {
    float r[N];
    bool far = false;
#pragma unroll
    for (int i = 0; i < N; ++i) { r[i] = tanh_near(u[i]); far |= !(fabsf(u[i]) <= kTanhNear); }
    if (__builtin_amdgcn_ballot_w64(far)) {
#pragma unroll
        for (int i = 0; i < N; ++i) r[i] = fabsf(u[i]) <= kTanhNear ? r[i] : tanh_far(u[i]);
    }
#pragma unroll
    for (int i = 0; i < N; ++i) u[i] = r[i];
}

// What a column's sum becomes: nothing seen: zeros and -inf; seen, but every score -inf: not a number, as a softmax of those is.
__device__ __forceinline__ float scored_inv(float l, bool seen) { return !seen ? 0.f : l > 0.f ? 1.f / l : __builtin_nanf(""); }
__device__ __forceinline__ float scored_lse(float m, float l, bool seen, float shift) { return seen ? __builtin_fmaf(m + __builtin_amdgcn_logf(l), kLn2, shift) : -__builtin_inff(); }
template <bool BF> __device__ __forceinline__ void scored_store(const ScoredParams& p, int row, int h, int HD, int d0, const f32x4& acc, float m, float l, bool seen, int ref) {
    const float inv = scored_inv(l, seen);
    u32x2 v = {0u, 0u};
    if (seen) { v[0] = act_pack<BF>(acc[0] * inv, acc[1] * inv); v[1] = act_pack<BF>(acc[2] * inv, acc[3] * inv); }
    const size_t at = (size_t)row * p.nh + h;
    *reinterpret_cast<u32x2*>(reinterpret_cast<uint16_t*>(p.out) + at * HD + d0) = v;
    if (d0 == 0 && p.lse) p.lse[at] = scored_lse(m, l, seen, scored_shift(p, row, h, ref));
}

inline int scored_params(ScoredParams& p, const void* q, int ldq, const mi355_kv_layer_t* kv, const int32_t* block_table, int max_blocks, const int32_t* row_start, int B, int q_len,
                         int rows, int nh, const mi355_attn_score_t* sc, int max_seq, void* out, float* lse, float* weights, float decay) {
    MI355_CHECK_ARG(q && kv && kv->kv_base && block_table && sc && sc->end && out, "paged_attn_scored: null pointer");
    MI355_CHECK_ARG(kv->hd == 64 || kv->hd == 128, "paged_attn_scored: hd=%d (64 or 128)", kv->hd);
    // offsets inside a page's keys or values of one head are 32 bits
    MI355_CHECK_ARG(kv->page >= 16 && kv->page % 16 == 0 && (long)kv->page * kv->hd * (kv->kv_dtype == MI355_KV_INT8 ? 1 : 2) < (1l << 31),
                    "paged_attn_scored: page=%d (a multiple of 16, heads of %d below 2^31 bytes)", kv->page, kv->hd);
    MI355_CHECK_ARG(B > 0 && q_len > 0 && rows > 0 && nh > 0 && kv->nkv > 0 && nh % kv->nkv == 0, "paged_attn_scored: B=%d q_len=%d rows=%d nh=%d nkv=%d", B, q_len, rows, nh, kv->nkv);
    MI355_CHECK_ARG(row_start ? (long)rows <= (long)B * q_len : (long)rows == (long)B * q_len, "paged_attn_scored: %d rows, %d sequences of %s%d", rows, B, row_start ? "at most " : "", q_len);
    MI355_CHECK_ARG(B <= 65535 && kv->nkv <= 65535 && (long)rows * nh < (1l << 31) && (long)q_len * nh < (1l << 30), "paged_attn_scored: B=%d nkv=%d rows=%d nh=%d exceed the grid", B, kv->nkv, rows, nh);
    MI355_CHECK_ARG(ldq >= nh * kv->hd && ldq % 8 == 0, "paged_attn_scored: ldq=%d for %d heads of %d (whole 16-byte pieces)", ldq, nh, kv->hd);
    MI355_CHECK_ARG(kv->num_blocks > 0 && max_seq > 0 && max_blocks > 0 && (long)max_blocks * kv->page >= max_seq, "paged_attn_scored: max_seq_len=%d exceeds the block table", max_seq);
    MI355_CHECK_ARG((long)max_seq * kv->page < (1l << 32) && max_seq < (1 << 30) && (long)kv->num_blocks * 2 * kv->nkv * kv->page < (1l << 31),
                    "paged_attn_scored: max_seq_len * page >= 2^32, max_seq_len >= 2^30 or 2^31 (token, head) pairs in the pool");
    const bool int8 = kv->kv_dtype == MI355_KV_INT8, bf = kv->act_dtype == MI355_ACT_BF16;
    MI355_CHECK_ARG(bf || kv->act_dtype == MI355_ACT_F16, "paged_attn_scored: act_dtype=%d", kv->act_dtype);
    MI355_CHECK_ARG(int8 ? kv->scale_base != nullptr : kv->kv_dtype == (bf ? MI355_KV_BF16 : MI355_KV_FP16), "paged_attn_scored: kv_dtype=%d with act_dtype=%d (8 bits need scales, 16 bits the activations' type)",
                    kv->kv_dtype, kv->act_dtype);
    MI355_CHECK_ARG((((uintptr_t)q | (uintptr_t)kv->kv_base | (uintptr_t)out) & 15) == 0 && (((uintptr_t)kv->scale_base | (uintptr_t)sc->key_pos) & 15) == 0,
                    "paged_attn_scored: q, cache, scales, key_pos and out lie on 16 bytes");
    MI355_CHECK_ARG(sc->softcap == 0.f || (sc->softcap >= 1e-6f && sc->softcap <= 1e6f), "paged_attn_scored: softcap=%g (0: none, or 1e-6 to 1e6)", (double)sc->softcap);
    MI355_CHECK_ARG(sc->scale > 0.f && sc->scale < 1e6f, "paged_attn_scored: scale=%g (> 0)", (double)sc->scale);
    MI355_CHECK_ARG(!sc->slopes || sc->positions, "paged_attn_scored: slopes need the rows' positions");
    MI355_CHECK_ARG(!weights || (decay >= 0.f && decay <= 1.f), "paged_attn_scored: decay=%g (0 to 1)", (double)decay);
    p.q = q; p.ldq = ldq; p.kv_base = kv->kv_base; p.scale_base = kv->scale_base; p.block_table = block_table; p.row_start = row_start;
    p.begin = sc->begin; p.end = sc->end; p.slopes = sc->slopes; p.positions = sc->positions; p.key_pos = sc->slopes ? sc->key_pos : nullptr;
    p.out = out; p.lse = lse; p.weights = weights; p.decay = decay;
    p.capped = sc->softcap > 0.f;
    p.scale1 = p.capped ? sc->scale / sc->softcap : sc->scale * kLog2e;
    p.cap_log2 = sc->softcap * kLog2e;
    p.max_blocks = max_blocks; p.B = B; p.q_len = q_len; p.rows = rows; p.nh = nh; p.nkv = kv->nkv; p.G = nh / kv->nkv;
    p.page = kv->page; p.num_blocks = kv->num_blocks; p.max_seq = max_seq;
    p.page_magic = (uint32_t)((1ull << 32) / (unsigned)kv->page + 1);
    return MI355_OK;
}

} // namespace
