// Paged attention with score forms, gfx950: scores capped by a tanh and biased by distance, rows that see an interval of the cache (causal, windows, prefixes,
// documents), log-sum-exps, and the attention weight that each cached token draws (what kv_evict.hip ranks them by).
//
//   u = scale q.k        s = cap tanh(u / cap)  (cap > 0, else u)        s += slope[h] (key position - row position)
//   row r, head h:  p_j = exp(s_j - lse),  lse = log sum_j exp(s_j),  out = sum_j p_j V_j   over the slots j in [begin[r], end[r]); an empty interval: out 0, lse -inf
//   weights[j, kv head] <- decay weights[j, kv head] + sum over the call's rows of the sequence and the heads of the group of p_j
//
// Everything is kept in the log2 domain: s2 = s log2(e), p = exp2(s2 - m) / l with m a column's running maximum and l its sum.  The weights are formed from m and l, not from their
// logarithm: under distance biases of thousands that alone would be off by 5e-4 of a weight.
#include <algorithm>
#include <type_traits>

#include "common.h"
#include "internal.h"
#include "scored.h"

namespace {

// ================================================================================================ few rows
// A (row, head) pair of a sequence's key/value head is one of 16 columns of v_mfma_f32_16x16x32: S^T = K q^T with 16 tokens and O^T = V^T P with 16 channels as rows, so keys and values are
// read once for up to 32 pairs (two tiles of columns).  The two 16-token halves of a 32-token group take the tokens {8 w + r} and {8 w + 4 + r}, w = lane / 16, so that the lane that holds
// eight scores of a column holds the same eight as the second product's operand: nothing crosses lanes between the products.
// A wave walks its groups on its own.  They come by DMA into a ring of its own in LDS: what is in flight takes no registers, and a page's 16 tokens are one scalar base for loads
// whose lanes' offsets never change.  A key's 16-byte pieces are swizzled by the token, a channel's 16 values stay side by side.
//
// Work: the tokens that any row of a sequence sees, in units of 128 (a group for each of a block's four waves), times key/value heads, laid end to end over all sequences and dealt to the
// blocks in equal runs.  A pair of a sequence and a head that lies inside one run is finished there, others leave a part in each run and scored_join_kernel merges them.  Sequences
// of unequal length so take the time of their mean: a run may end one pair and begin the next.
struct DecodeParams : ScoredParams {
    float*   tmp_out;    // [2 nblocks][ncol][hd]: parts; a run's first segment in slot 2 run, a later one that goes on in the next run in 2 run + 1
    float*   tmp_ml;     // [2 nblocks][ncol][2]
    float*   ml_all;     // [pairs][ncol][2] of pairs that were finished in one run (with weights)
    float*   spill;      // [pairs][ncol][ctx_pad] scores in the log2 domain (with weights), from the sequence's first unit on
    int4*    meta;       // [pairs]: first slot, parts, the sequence's first seen slot rounded down to 32, its reach
    int      nblocks, ncol, ctx_pad, runs;   // runs: 0 = a block per pair
};
constexpr int UNIT = 128;

// The slots that a sequence's rows see, [seen, hi), and lo = seen down to 32; nothing: zeros.
__device__ __forceinline__ void scored_span(const ScoredParams& p, int b, int& lo, int& hi, int& seen) {
    int base, len;
    scored_rows_of(p, b, base, len);
    seen = 0x7fffffff; hi = 0;
    for (int i = 0; i < len; ++i) {
        int a, e;
        scored_interval(p, base + i, a, e);
        if (e > a) { seen = min(seen, a); hi = max(hi, e); }
    }
    if (hi == 0) seen = 0;
    lo = seen & ~31;
}
__device__ __forceinline__ int units_of(int lo, int hi) { return (hi - lo + UNIT - 1) / UNIT; }

typedef int i32x4 __attribute__((ext_vector_type(4)));

// 8 cache bytes (code + 128) -> the codes, exact in both types.  With the offset left inside (1152 under fp16's exponent of 1024, 128 in bf16) and taken out of the sums behind the products,
// a score would be the small difference of sums some 30 times its terms: 5e-5 of it, and so of a weight.
template <bool BF> __device__ __forceinline__ u32x4 widen_codes(uint32_t lo, uint32_t hi) {
    if constexpr (BF) {
        auto pk = [](uint32_t a, uint32_t b) {
            return __builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, (float)b - 128.f), __builtin_bit_cast(uint32_t, (float)a - 128.f), 0x07060302u);
        };
        return u32x4{pk(lo & 0xFFu, lo >> 8 & 0xFFu), pk(lo >> 16 & 0xFFu, lo >> 24), pk(hi & 0xFFu, hi >> 8 & 0xFFu), pk(hi >> 16 & 0xFFu, hi >> 24)};
    }
    const uint32_t C = 0x64646464u;
    u32x4 v = {__builtin_amdgcn_perm(C, lo, 0x04010400u), __builtin_amdgcn_perm(C, lo, 0x04030402u), __builtin_amdgcn_perm(C, hi, 0x04010400u), __builtin_amdgcn_perm(C, hi, 0x04030402u)};
    const f16x2 off = {(f16)-1152.f, (f16)-1152.f};
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = as_u32(as_h2(v[i]) + off);
    return v;
}

// LDS of a wave's stage: keys, values, and (EXTRA) 1 KB of scales and positions; stages that 160 KB hold, as many as pay.
template <int HD, bool INT8, bool EXTRA> struct Ring {
    static constexpr int ES = INT8 ? 1 : 2, KB = 32 * HD * ES, LOADS = 2 * KB / 1024 + (EXTRA ? 1 : 0), STAGE = LOADS * 1024, N = HD == 128 && !INT8 ? 2 : INT8 && HD == 128 ? 4 : 4;
    static constexpr int MERGE = 4 * 16 * (HD + 4) * 4 + 2 * 4 * 16 * 4, BYTES = 4 * N * STAGE > MERGE ? 4 * N * STAGE : MERGE;
};

template <int HD, bool INT8, int NT, bool BF, bool KP>
__global__ __launch_bounds__(256) void scored_decode_kernel(const DecodeParams p) {
    constexpr bool EXTRA = INT8 || KP;
    // 8 bits under fp16: probabilities take the value's scale, an amax / 127, before they are rounded.  64 of it keep the small ones out of fp16's subnormals (amax <= 65504: 64 scales fit) if
    // no probability exceeds 1.
    constexpr float VS = INT8 && !BF ? 64.f : 1.f, DEFER = INT8 && !BF ? 0.f : 6.f;
    using R = Ring<HD, INT8, EXTRA>;
    constexpr int NSTEP = HD / 32, NDB = HD / 16, ES = R::ES, CK = HD * ES / 16, RS = R::N;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int j = lane & 15, w = lane >> 4;
    extern __shared__ __attribute__((aligned(16))) char dec_sm[];
    auto s_o = reinterpret_cast<float(*)[16][HD + 4]>(dec_sm);                        // the merge's, over the ring
    auto s_m = reinterpret_cast<float(*)[16]>(dec_sm + 4 * 16 * (HD + 4) * 4);
    float(*s_l)[16] = s_m + 4;
    char* ring = dec_sm + wave * RS * R::STAGE;
    const uint32_t ring0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)ring;
    // lanes' offsets in loads of keys (R::KB / 1024 of them, 1024 / (HD ES) rows each) and values
    constexpr int KL = R::KB / 1024, KR = 1024 / (HD * ES), KU = KL / 2;             // KU: loads of a 16-token unit
    uint32_t koff[KL];
#pragma unroll
    for (int d = 0; d < KL; ++d) {
        const int tok = d * KR + lane / CK, f = ((tok & 3) | (tok >> 3 & 3) << 2) & (CK - 1);
        koff[d] = (uint32_t)((tok & 15) * HD * ES + (((lane % CK) ^ f) << 4));
    }
    const uint32_t voff = INT8 ? (uint32_t)(lane * p.page) : (uint32_t)((lane >> 1) * p.page + (lane & 1) * 8) * 2u;
    constexpr int VC = INT8 ? 64 : 32, VU = HD / VC;                                 // channels of a load, loads of a unit
    // where the lane's fragments lie in a stage
    const int ktok = (j & 3) + 8 * (j >> 2), kf = ((j & 3) | (j >> 2) << 2) & (CK - 1);

    // ---- this block's run of units
    int b, kh, lo, hi, seen0, units, u, u1;                // the pair at hand, its span, the run's next unit inside it, the run's end (counted from the pair's first unit)
    if (p.runs) {
        int total = 0;
        for (int b0 = 0; b0 < p.B; b0 += 64) {
            int l = 0, h = 0, seen;
            if (b0 + lane < p.B) scored_span(p, b0 + lane, l, h, seen);
            int n = units_of(l, h) * p.nkv;
#pragma unroll
            for (int o = 32; o > 0; o >>= 1) n += __shfl_xor(n, o);
            total += n;
        }
        total = __builtin_amdgcn_readfirstlane(total);
        const int W = max(1, (total + p.nblocks - 1) / p.nblocks), start = blockIdx.x * W, stop = min(total, start + W);
        if (start >= stop && blockIdx.x != 0) return;
        int before = 0, at = -1, at_s = 0;          // units before this group of 64 sequences; the sequence in which the run begins
        for (int b0 = 0; b0 < p.B; b0 += 64) {
            int l = 0, h = 0, seen;
            if (b0 + lane < p.B) scored_span(p, b0 + lane, l, h, seen);
            const int per = units_of(l, h), n = per * p.nkv;
            int incl = n;
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) { const int up = __shfl_up(incl, o); if (lane >= o) incl += up; }
            const int s = before + incl - n;
            if (blockIdx.x == 0 && wave == 0 && b0 + lane < p.B)
                for (int k = 0; k < p.nkv; ++k) {
                    const int a = s + k * per, e = a + per, r0 = a / W, r1 = per ? (e - 1) / W : r0 - 1;
                    p.meta[(size_t)(b0 + lane) * p.nkv + k] = make_int4(2 * r0 + (a == r0 * W ? 0 : 1), r1 - r0 + 1, l, h);
                }
            const uint64_t in = __builtin_amdgcn_ballot_w64(start >= s && start < s + n);
            if (in && at < 0) { const int who = __builtin_ctzll(in); at = b0 + who; at_s = __builtin_amdgcn_readlane(s, who); }
            before += __builtin_amdgcn_readlane(incl, 63);
            if (at >= 0 && blockIdx.x != 0) break;
        }
        if (start >= stop) return;
        b = at;
        scored_span(p, b, lo, hi, seen0);
        lo = __builtin_amdgcn_readfirstlane(lo); hi = __builtin_amdgcn_readfirstlane(hi); seen0 = __builtin_amdgcn_readfirstlane(seen0);
        units = units_of(lo, hi);
        kh = (start - at_s) / units;
        u = start - at_s - kh * units;
        u1 = u + stop - start;
    } else {
        b = blockIdx.x / p.nkv; kh = blockIdx.x - b * p.nkv;
        scored_span(p, b, lo, hi, seen0);
        lo = __builtin_amdgcn_readfirstlane(lo); hi = __builtin_amdgcn_readfirstlane(hi); seen0 = __builtin_amdgcn_readfirstlane(seen0);
        units = units_of(lo, hi); u = 0; u1 = units;
        if (tid == 0) p.meta[blockIdx.x] = make_int4(0, units ? 1 : 0, lo, hi);
    }

    bool first = true;
    while (u1 > 0) {                                // segments: units [u, min(u1, units)) of pair (b, kh)
        const int stop_u = min(u1, units);
        const bool whole = u == 0 && stop_u == units;
        int base, len;
        scored_rows_of(p, b, base, len);
        base = __builtin_amdgcn_readfirstlane(base); len = __builtin_amdgcn_readfirstlane(len);
        const int ncol = len * p.G;
        const int pstart = lo + u * UNIT, pend = min(hi, lo + stop_u * UNIT);
        const int32_t* bt = p.block_table + (size_t)b * p.max_blocks;
        const size_t pair = (size_t)b * p.nkv + kh;
        const int ref = p.slopes ? __builtin_amdgcn_readfirstlane(scored_ref(p, b, kh, hi)) : 0;

        u32x4 qf[NT][NSTEP];
        int c_lo[NT], c_hi[NT];
        float slope2[NT];
        int in_lo = 0, in_hi = 0x7fffffff;          // every column of this lane sees [in_lo, in_hi)
#pragma unroll
        for (int c = 0; c < NT; ++c) {
            const int col = c * 16 + j, rl = col / p.G, g = col - rl * p.G;
            const bool ok = col < ncol;
            const int row = base + (ok ? rl : 0), h = kh * p.G + (ok ? g : 0);
            scored_interval(p, row, c_lo[c], c_hi[c]);
            if (!ok) c_lo[c] = c_hi[c] = 0;
            if (c_hi[c] > c_lo[c]) { in_lo = max(in_lo, c_lo[c]); in_hi = min(in_hi, c_hi[c]); }
            slope2[c] = p.slopes ? p.slopes[h] * kLog2e : 0.f;
            const uint16_t* qrow = reinterpret_cast<const uint16_t*>(p.q) + (size_t)row * p.ldq + h * HD;
#pragma unroll
            for (int s = 0; s < NSTEP; ++s) {
                const int d = INT8 ? (s >> 1) * 64 + w * 16 + (s & 1) * 8 : s * 32 + w * 8;
                u32x4 v = *reinterpret_cast<const u32x4*>(qrow + d);
                if (!ok) v = (u32x4){0u, 0u, 0u, 0u};
                qf[c][s] = v;
            }
        }
#pragma unroll
        for (int o = 1; o < 16; o <<= 1) { in_lo = max(in_lo, __shfl_xor(in_lo, o)); in_hi = min(in_hi, __shfl_xor(in_hi, o)); }
        in_lo = __builtin_amdgcn_readfirstlane(in_lo); in_hi = __builtin_amdgcn_readfirstlane(in_hi);
        f32x4 o[NT][NDB];
        float m_run[NT], l_run[NT];
#pragma unroll
        for (int c = 0; c < NT; ++c) {
            m_run[c] = NEG_BIG; l_run[c] = 0.f;
#pragma unroll
            for (int db = 0; db < NDB; ++db) o[c][db] = (f32x4){0.f, 0.f, 0.f, 0.f};
        }
        // A stage: 32 tokens as two units of 16, each inside one page; units behind the last seen slot read that one's again (masked).
        const int last16 = (hi - 1) & ~15;
        auto page_of = [&](int t) { return (int)__builtin_amdgcn_readfirstlane((int)(((unsigned long long)(unsigned)t * p.page_magic) >> 32)); };
        const uint32_t head_bytes = (uint32_t)(p.page * HD * ES);
        int idv = 0;                                // block ids of 32 groups' units, a lane each: one load (which waits for the ring once) in 32
        auto issue = [&](int i, int buf) {
            const int tb = pstart + wave * 32 + i * UNIT;
            if ((i & 31) == 0) {
                const int t = min(tb + (lane >> 1) * UNIT + (lane & 1) * 16, last16);
                idv = bt[(int)(((unsigned long long)(unsigned)t * p.page_magic) >> 32)];
            }
            const int ids[2] = {__builtin_amdgcn_readlane(idv, (i & 31) * 2), __builtin_amdgcn_readlane(idv, (i & 31) * 2 + 1)};
            const uint32_t to = __builtin_amdgcn_readfirstlane(ring0 + buf * R::STAGE);
            int64_t extra[2];
#pragma unroll
            for (int a = 0; a < 2; ++a) {
                const int t = min(tb + 16 * a, last16), ti = t - page_of(t) * p.page, blk = min(max(ids[a], 0), p.num_blocks - 1);
                const uint32_t hk = (uint32_t)blk * (uint32_t)(2 * p.nkv) + (uint32_t)kh;
                const char* kb = (const char*)p.kv_base + (uint64_t)hk * head_bytes;
                const char* vb = kb + (uint64_t)(uint32_t)p.nkv * head_bytes + (uint32_t)(ti * ES);
                kb += (uint32_t)(ti * HD * ES);
#pragma unroll
                for (int d = 0; d < KU; ++d) dma16(to + (a * KU + d) * 1024, koff[a * KU + d], kb);
#pragma unroll
                for (int d = 0; d < VU; ++d) dma16(to + R::KB + (a * VU + d) * 1024, voff, vb + (uint32_t)(d * VC * ES) * (uint32_t)p.page);
                extra[a] = (int64_t)hk * p.page + ti;
            }
            if constexpr (EXTRA) {                  // 16-byte pieces: 8 of the keys' scales, 8 of the values', 8 of positions
                const int64_t at = (lane & 4 ? extra[1] : extra[0]) + (lane & 3) * 4;
                const char* from = (const char*)(p.scale_base + at + (lane & 8 ? (int64_t)p.nkv * p.page : 0));
                if constexpr (KP) {
                    const int64_t back = (int64_t)p.nkv * p.page;             // [blocks][nkv][page] against the scales' [blocks][2][nkv][page]
                    const int64_t b0 = min(max(ids[0], 0), p.num_blocks - 1), b1 = min(max(ids[1], 0), p.num_blocks - 1);
                    if (!INT8 || lane & 16) from = (const char*)(p.key_pos + at - (lane & 4 ? b1 : b0) * back);
                }
                dma16(to + 2 * R::KB, from);
            }
        };
        auto compute_group = [&](const char* st, int tb, auto masked_c) {
            constexpr bool MASKED = decltype(masked_c)::value;
            const int vwin = tb + w * 8;            // the lane's first token
            u32x4 pf[NT];
            float alpha[NT];
            bool rescale = false;
            u32x4 ka[2][NSTEP];
#pragma unroll
            for (int tau = 0; tau < 2; ++tau)
#pragma unroll
                for (int s = 0; s < NSTEP; ++s) {
                    const char* krow = st + (ktok + tau * 4) * HD * ES;
                    if constexpr (INT8) {
                        const u32x4 kk = *reinterpret_cast<const u32x4*>(krow + ((((s >> 1) * 4 + w) ^ kf) << 4));
                        ka[tau][s] = widen_codes<BF>(kk[(s & 1) * 2], kk[(s & 1) * 2 + 1]);
                    } else ka[tau][s] = *reinterpret_cast<const u32x4*>(krow + (((s * 4 + w) ^ kf) << 4));
                }
            f32x4 ksc[INT8 ? 2 : 1], vsc[INT8 ? 2 : 1];
            i32x4 kpos[KP ? 2 : 1];
            if constexpr (INT8) {
                const f32x4* sc = reinterpret_cast<const f32x4*>(st + 2 * R::KB) + w * 2;
                ksc[0] = sc[0]; ksc[1] = sc[1]; vsc[0] = sc[8]; vsc[1] = sc[9];
            }
            if constexpr (KP) {
                const i32x4* kp = reinterpret_cast<const i32x4*>(st + 2 * R::KB) + (INT8 ? 16 : 0) + w * 2;
                kpos[0] = kp[0]; kpos[1] = kp[1];
            }
#pragma unroll
            for (int c = 0; c < NT; ++c) {
                f32x4 sacc[2];
#pragma unroll
                for (int tau = 0; tau < 2; ++tau) {
                    sacc[tau] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int s = 0; s < NSTEP; ++s) sacc[tau] = mfma_act<BF>(ka[tau][s], qf[c][s], sacc[tau]);
                }
                float sv[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    float v = sacc[e >> 2][e & 3];
                    if constexpr (INT8) v *= ksc[e >> 2][e & 3];
                    sv[e] = v * p.scale1;
                }
                if (p.capped) {
                    tanh_all(sv);
#pragma unroll
                    for (int e = 0; e < 8; ++e) sv[e] *= p.cap_log2;
                }
                if (p.slopes) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const int kp = KP ? kpos[KP ? e >> 2 : 0][e & 3] : vwin + e;
                        sv[e] = __builtin_fmaf(slope2[c], (float)(kp - ref), sv[e]);
                    }
                }
                float mx = NEG_BIG;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    if (MASKED) sv[e] = vwin + e >= c_lo[c] && vwin + e < c_hi[c] ? sv[e] : NEG_BIG;
                    mx = fmaxf(mx, sv[e]);
                }
                if (p.spill && c * 16 + j < ncol) {
                    float* to = p.spill + (pair * p.ncol + c * 16 + j) * (size_t)p.ctx_pad + (vwin - lo);
                    *reinterpret_cast<f32x4*>(to) = f32x4{sv[0], sv[1], sv[2], sv[3]};
                    *reinterpret_cast<f32x4*>(to + 4) = f32x4{sv[4], sv[5], sv[6], sv[7]};
                }
                mx = xor32_max(xor16_max(mx));      // the column's 32 tokens lie in the lanes j, j + 16, j + 32, j + 48
                // The running maximum moves, and sums and outputs are scaled, only where some column's grew by more than DEFER: until then exp2(s2 - m) may exceed 1 by 2^DEFER.
                const bool grow = __builtin_amdgcn_ballot_w64(mx > m_run[c] + DEFER) != 0;
                const float m_new = grow ? fmaxf(m_run[c], mx) : m_run[c];
                alpha[c] = grow ? __builtin_amdgcn_exp2f(m_run[c] - m_new) : 1.f;
                rescale |= grow;
                m_run[c] = m_new;
                float psum = 0.f, pes[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const bool seen = !MASKED || (vwin + e >= c_lo[c] && vwin + e < c_hi[c]);
                    float pe = seen ? __builtin_amdgcn_exp2f(sv[e] - m_new) : 0.f;
                    psum += pe;
                    if constexpr (INT8) pe = seen ? pe * (vsc[e >> 2][e & 3] * VS) : 0.f;
                    pes[e] = pe;
                }
                pf[c] = act_pack8<BF>(pes);
                l_run[c] = l_run[c] * alpha[c] + psum;
            }
            if (rescale) {
#pragma unroll
                for (int c = 0; c < NT; ++c)
#pragma unroll
                    for (int db = 0; db < NDB; ++db) o[c][db] *= alpha[c];
            }
#pragma unroll
            for (int db = 0; db < NDB; ++db) {
                u32x4 a;
                const char* vch = st + R::KB + (w >> 1) * (HD * 16 * ES) + (db * 16 + j) * (16 * ES) + (w & 1) * (8 * ES);
                if constexpr (INT8) {
                    const u32x2 v8 = *reinterpret_cast<const u32x2*>(vch);
                    a = widen_codes<BF>(v8[0], v8[1]);
                } else {
                    a = *reinterpret_cast<const u32x4*>(vch);
                    if (MASKED) {                   // slots that no row sees may hold anything, NaN too: their weights are zero, their values are made so
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            if (vwin + e >= hi || vwin + e < seen0) a[e >> 1] &= (e & 1) ? 0x0000FFFFu : 0xFFFF0000u;
                    }
                }
#pragma unroll
                for (int c = 0; c < NT; ++c) o[c][db] = mfma_act<BF>(a, pf[c], o[c][db]);
            }
        };
        const int n = (pend - pstart - wave * 32 + UNIT - 1) / UNIT;                  // this wave's groups (none: 0 or less)
        wait_vm<0>();                               // the queries are here: no wait for them inside the loop
        for (int i = 0; i < min(RS - 1, n); ++i) issue(i, i);
        int buf = 0;
        for (int i = 0; i < n; ++i) {
            const int tb = pstart + wave * 32 + i * UNIT;
            if (i + RS - 1 < n) {
                issue(i + RS - 1, buf == 0 ? RS - 1 : buf - 1);
                wait_vm<R::LOADS * (RS - 1)>();
            } else
                wait_vm<0>();
            const char* st = ring + buf * R::STAGE;
            buf = buf == RS - 1 ? 0 : buf + 1;
            if (tb >= in_lo && tb + 32 <= in_hi) compute_group(st, tb, std::false_type{});
            else compute_group(st, tb, std::true_type{});
            wait_vm<63>();                          // the stage has been read before a later load may land in it
        }
        __syncthreads();                            // every wave is done with its ring
        // ---- the four waves meet in LDS, a tile of columns at a time
        const size_t slot = (size_t)blockIdx.x * 2 + (first ? 0 : 1);
#pragma unroll
        for (int c = 0; c < NT; ++c) {
            const float lr = xor32_sum(xor16_sum(l_run[c]));
            if (c) __syncthreads();                 // the tile before has been read
#pragma unroll
            for (int db = 0; db < NDB; ++db) *reinterpret_cast<f32x4*>(&s_o[wave][j][db * 16 + w * 4]) = o[c][db];
            if (w == 0) { s_m[wave][j] = m_run[c]; s_l[wave][j] = lr; }
            __syncthreads();
            const int here = min(16, ncol - c * 16);
            for (int idx = tid; idx < here * (HD / 4); idx += 256) {
                const int jj = idx / (HD / 4), d0 = (idx - jj * (HD / 4)) * 4, col = c * 16 + jj;
                const float mstar = fmaxf(fmaxf(s_m[0][jj], s_m[1][jj]), fmaxf(s_m[2][jj], s_m[3][jj]));
                f32x4 acc = {0.f, 0.f, 0.f, 0.f};
                float l = 0.f;
#pragma unroll
                for (int ww = 0; ww < 4; ++ww) {
                    const float f = __builtin_amdgcn_exp2f(s_m[ww][jj] - mstar);
                    const f32x4 ow = *reinterpret_cast<const f32x4*>(&s_o[ww][jj][d0]);
                    acc += ow * f;
                    l += s_l[ww][jj] * f;
                }
                if constexpr (VS != 1.f) acc *= 1.f / VS;
                if (whole) {
                    const int rl = col / p.G, row = base + rl, h = kh * p.G + (col - rl * p.G);
                    int a, e;
                    scored_interval(p, row, a, e);
                    scored_store<BF>(p, row, h, HD, d0, acc, mstar, l, e > a, ref);
                    if (p.ml_all && d0 == 0) *reinterpret_cast<float2*>(p.ml_all + (pair * p.ncol + col) * 2) = make_float2(mstar, l);
                } else {
                    *reinterpret_cast<f32x4*>(p.tmp_out + (slot * p.ncol + col) * HD + d0) = acc;
                    if (d0 == 0) *reinterpret_cast<float2*>(p.tmp_ml + (slot * p.ncol + col) * 2) = make_float2(mstar, l);
                }
            }
        }
        __syncthreads();                            // the merge is over: the ring may be filled again
        // ---- on to the next pair
        first = false;
        u1 -= units; u = 0;
        if (u1 <= 0) break;
        if (++kh == p.nkv) {
            kh = 0;
            do {
                if (++b >= p.B) return;             // cannot be: the run ends inside the last sequence
                scored_span(p, b, lo, hi, seen0);
                lo = __builtin_amdgcn_readfirstlane(lo); hi = __builtin_amdgcn_readfirstlane(hi); seen0 = __builtin_amdgcn_readfirstlane(seen0);
                units = units_of(lo, hi);
            } while (units == 0);
        }
    }
}

// What the runs left: a wave per (pair, column) merges its parts (nothing to do where there is one; zeros where there is none), and, behind those blocks, a thread per slot adds the
// probabilities of all columns to the slot's weight.
constexpr int JOIN_COLS = 32;
template <int HD, bool BF>
__global__ __launch_bounds__(256) void scored_join_kernel(const DecodeParams p, int join_blocks, int chunks) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    auto slot_of = [](const int4& mt, int i) { return i == 0 ? mt.x : (mt.x / 2 + i) * 2; };
    if ((int)blockIdx.x < join_blocks) {
        const int gid = blockIdx.x * 4 + wave, pair = gid / p.ncol, col = gid - pair * p.ncol;
        if (pair >= p.B * p.nkv) return;
        const int4 mt = p.meta[pair];
        if (mt.y == 1) return;
        const int b = pair / p.nkv, kh = pair - b * p.nkv;
        int base, len;
        scored_rows_of(p, b, base, len);
        if (col >= len * p.G) return;
        const int rl = col / p.G, row = base + rl, h = kh * p.G + (col - rl * p.G);
        float m = NEG_BIG;
        for (int i = lane; i < mt.y; i += 64) m = fmaxf(m, p.tmp_ml[((size_t)slot_of(mt, i) * p.ncol + col) * 2]);
        m = wave_max(m);
        constexpr int CPL = HD / 64;
        float l = 0.f, acc[CPL];
#pragma unroll
        for (int c = 0; c < CPL; ++c) acc[c] = 0.f;
        for (int i0 = 0; i0 < mt.y; i0 += 8) {      // eight parts in flight, added in their order
            float2 ml[8];
            float v[8][CPL];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const size_t at = (size_t)slot_of(mt, min(i0 + i, mt.y - 1)) * p.ncol + col;
                ml[i] = *reinterpret_cast<const float2*>(p.tmp_ml + at * 2);
#pragma unroll
                for (int c = 0; c < CPL; ++c) v[i][c] = p.tmp_out[at * HD + lane * CPL + c];
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if (i0 + i >= mt.y) continue;
                const float f = __builtin_amdgcn_exp2f(ml[i].x - m);
                l += ml[i].y * f;
#pragma unroll
                for (int c = 0; c < CPL; ++c) acc[c] += v[i][c] * f;
            }
        }
        int a, e;
        scored_interval(p, row, a, e);
        const float inv = scored_inv(l, e > a);
        uint16_t* dst = reinterpret_cast<uint16_t*>(p.out) + ((size_t)row * p.nh + h) * HD + lane * CPL;
#pragma unroll
        for (int c = 0; c < CPL; ++c) dst[c] = act_to_bits<BF>(acc[c] * inv);
        if (lane == 0 && p.lse) p.lse[(size_t)row * p.nh + h] = scored_lse(m, l, e > a, p.slopes && e > a ? scored_shift(p, row, h, scored_ref(p, b, kh, mt.w)) : 0.f);
        return;
    }
    // ---- weights
    __shared__ float s_m[JOIN_COLS], s_i[JOIN_COLS];
    const int id = blockIdx.x - join_blocks, pair = id / chunks, chunk = id - pair * chunks;
    const int4 mt = p.meta[pair];
    if (chunk * 1024 >= mt.w) return;
    const int b = pair / p.nkv, kh = pair - b * p.nkv;
    int base, len;
    scored_rows_of(p, b, base, len);
    const int ncol = len * p.G;
    for (int col = wave; col < ncol; col += 4) {
        float m = NEG_BIG, l = 0.f;
        if (mt.y == 1) {
            const float2 v = *reinterpret_cast<const float2*>(p.ml_all + ((size_t)pair * p.ncol + col) * 2);
            m = v.x; l = v.y;
        } else {
            for (int i = lane; i < mt.y; i += 64) {
                const float2 v = *reinterpret_cast<const float2*>(p.tmp_ml + ((size_t)slot_of(mt, i) * p.ncol + col) * 2);
                const float mn = fmaxf(m, v.x);
                l = l * __builtin_amdgcn_exp2f(m - mn) + v.y * __builtin_amdgcn_exp2f(v.x - mn);
                m = mn;
            }
            const float mine = m;
            m = wave_max(m);
            l = wave_sum(l * __builtin_amdgcn_exp2f(mine - m));
        }
        int a, e;
        scored_interval(p, base + col / p.G, a, e);
        if (lane == 0) { s_m[col] = m; s_i[col] = scored_inv(l, e > a); }
    }
    __syncthreads();
    const int t = chunk * 1024 + tid * 4;           // four slots: inside a page (a multiple of 8 tokens)
    if (t >= mt.w) return;
    const int32_t* bt = p.block_table + (size_t)b * p.max_blocks;
    const int blk = bt[(int)(((unsigned long long)(unsigned)t * p.page_magic) >> 32)];
    if (blk < 0 || blk >= p.num_blocks) return;
    float* to = p.weights + ((size_t)blk * p.nkv + kh) * p.page + t % p.page;
    float sum[4] = {0.f, 0.f, 0.f, 0.f};
    if (t >= mt.z) {
        const float* sp = p.spill + (size_t)pair * p.ncol * p.ctx_pad + (t - mt.z);
        for (int c0 = 0; c0 < ncol; c0 += 8) {
            f32x4 v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = *reinterpret_cast<const f32x4*>(sp + (size_t)min(c0 + i, ncol - 1) * p.ctx_pad);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if (c0 + i >= ncol) continue;
                const float m = s_m[c0 + i], inv = s_i[c0 + i];
#pragma unroll
                for (int e = 0; e < 4; ++e) sum[e] += v[i][e] <= NEG_BIG || inv == 0.f ? 0.f : __builtin_amdgcn_exp2f(v[i][e] - m) * inv;
            }
        }
    }
    if (t + 4 <= mt.w) {
        const f32x4 old = *reinterpret_cast<const f32x4*>(to);
        *reinterpret_cast<f32x4*>(to) = f32x4{scored_decayed(p, old[0], sum[0]), scored_decayed(p, old[1], sum[1]), scored_decayed(p, old[2], sum[2]), scored_decayed(p, old[3], sum[3])};
    } else
        for (int e = 0; t + e < mt.w; ++e) to[e] = scored_decayed(p, to[e], sum[e]);
}

// ================================================================================================ simple forms: a wave per (row, head)
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
        s *= p.scale1;
        if (p.capped) s = p.cap_log2 * (fabsf(s) <= kTanhNear ? tanh_near(s) : tanh_far(s));
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
    const float inv = scored_inv(l, hi > lo);
#pragma unroll
    for (int c = 0; c < HD / 64; ++c) reinterpret_cast<uint16_t*>(p.out)[((size_t)row * p.nh + h) * HD + lane + 64 * c] = act_to_bits<BF>(o[c] * inv);
    if (lane == 0 && p.lse) p.lse[(size_t)row * p.nh + h] = scored_lse(m, l, hi > lo, 0.f);
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
            s *= p.scale1;
            if (p.capped) s = p.cap_log2 * (fabsf(s) <= kTanhNear ? tanh_near(s) : tanh_far(s));
            if (p.slopes) s = __builtin_fmaf(p.slopes[h] * kLog2e, (float)((p.key_pos ? p.key_pos[wat] : t) - p.positions[base + i]), s);
            sum += __builtin_amdgcn_exp2f(s - p.lse[(size_t)(base + i) * p.nh + h] * kLog2e);
        }
    }
    p.weights[wat] = scored_decayed(p, p.weights[wat], sum);
}

// ================================================================================================ plans
// How a call runs: sizes of its workspace's regions, each on 256 bytes.
struct Plan {
    bool   few;                // the few-row kernel: at most 32 (row, head) pairs of a key/value head a sequence
    int    nblocks, ncol, ctx_pad, runs;
    size_t tmp_out, tmp_ml, ml_all, spill, meta, lse, bytes;     // offsets; bytes: all
};
constexpr int RUNS = 256;      // one block of the few-row kernel a compute unit
Plan plan_of(int B, int q_len, int rows, int nh, int nkv, int hd, int max_seq, bool track) {
    Plan pl{};
    const int G = nh / nkv;
    size_t at = 0;
    auto region = [&](size_t bytes) { const size_t r = at; at += (bytes + 255) & ~(size_t)255; return r; };
    pl.few = (long)q_len * G <= JOIN_COLS;
    if (pl.few) {
        const long pairs = (long)B * nkv;
        pl.runs = pairs < 4 * RUNS;                              // beyond, pairs are many enough to even out by themselves, and nothing has to be merged
        pl.nblocks = pl.runs ? RUNS : (int)pairs;
        pl.ncol = q_len * G; pl.ctx_pad = (max_seq + 31 + UNIT) / 32 * 32;
        pl.meta = region(pairs * sizeof(int4));
        if (pl.runs) { pl.tmp_out = region((size_t)2 * RUNS * pl.ncol * hd * 4); pl.tmp_ml = region((size_t)2 * RUNS * pl.ncol * 8); }
        if (track) { pl.ml_all = region(pairs * pl.ncol * 8); pl.spill = region(pairs * pl.ncol * pl.ctx_pad * 4); }
    } else if (track) pl.lse = region((size_t)rows * nh * 4);
    pl.bytes = at;
    return pl;
}

template <int HD, bool INT8, int NT, bool BF>
int launch_decode(const DecodeParams& d, hipStream_t st) {
    auto run = [&](auto kernel, int lds) -> int {
        const int rc = raise_dynamic_lds((const void*)kernel, "paged_attn_scored");
        if (rc == MI355_OK) hipLaunchKernelGGL(kernel, dim3(d.nblocks), dim3(256), lds, st, d);
        return rc;
    };
    return d.key_pos ? run(scored_decode_kernel<HD, INT8, NT, BF, true>, Ring<HD, INT8, true>::BYTES) : run(scored_decode_kernel<HD, INT8, NT, BF, false>, Ring<HD, INT8, INT8>::BYTES);
}

} // namespace

extern "C" size_t mi355_paged_attn_scored_workspace_bytes(int32_t B, int32_t q_len, int32_t rows, int32_t nh, int32_t nkv, int32_t hd, int32_t max_seq_len, int32_t track) {
    if (B <= 0 || q_len <= 0 || rows <= 0 || nh <= 0 || nkv <= 0 || nh % nkv || hd <= 0 || max_seq_len <= 0) return 0;
    return plan_of(B, q_len, rows, nh, nkv, hd, max_seq_len, track != 0).bytes;
}

extern "C" int mi355_paged_attn_scored(const void* q, int32_t ldq, const mi355_kv_layer_t* kv, const int32_t* block_table, int32_t max_blocks_per_seq,
                                       const int32_t* row_start, int32_t B, int32_t q_len, int32_t rows, int32_t nh, const mi355_attn_score_t* score,
                                       int32_t max_seq_len, void* out, float* lse, float* weights, float decay, void* workspace, size_t workspace_bytes,
                                       mi355_stream_t stream) {
    DecodeParams p;
    const int rc = scored_params(p, q, ldq, kv, block_table, max_blocks_per_seq, row_start, B, q_len, rows, nh, score, max_seq_len, out, lse, weights, decay);
    if (rc != MI355_OK) return rc;
    const Plan pl = plan_of(B, q_len, rows, nh, kv->nkv, kv->hd, max_seq_len, weights != nullptr);
    if (pl.bytes && (pl.bytes > workspace_bytes || !workspace)) {
        mi355_set_error("paged_attn_scored: workspace %zu < %zu", workspace_bytes, pl.bytes);
        return MI355_ERR_WORKSPACE;
    }
    MI355_CHECK_ARG(((uintptr_t)workspace & 15) == 0, "paged_attn_scored: the workspace lies on 16 bytes");
    const bool bf = kv->act_dtype == MI355_ACT_BF16, int8 = kv->kv_dtype == MI355_KV_INT8;
    hipStream_t st = (hipStream_t)stream;
    char* ws = (char*)workspace;
    if (pl.few) {
        p.nblocks = pl.nblocks; p.ncol = pl.ncol; p.ctx_pad = pl.ctx_pad; p.runs = pl.runs;
        p.meta = (int4*)(ws + pl.meta);
        p.tmp_out = pl.runs ? (float*)(ws + pl.tmp_out) : nullptr; p.tmp_ml = pl.runs ? (float*)(ws + pl.tmp_ml) : nullptr;
        p.ml_all = weights ? (float*)(ws + pl.ml_all) : nullptr; p.spill = weights ? (float*)(ws + pl.spill) : nullptr;
        int lrc = MI355_OK;
#define LN_(HD_, I8_, BF_) do { lrc = pl.ncol <= 16 ? launch_decode<HD_, I8_, 1, BF_>(p, st) : launch_decode<HD_, I8_, 2, BF_>(p, st); } while (0)
#define LB_(HD_) do { if (bf) { if (int8) LN_(HD_, true, true); else LN_(HD_, false, true); } else { if (int8) LN_(HD_, true, false); else LN_(HD_, false, false); } } while (0)
        if (kv->hd == 128) LB_(128); else LB_(64);
#undef LB_
#undef LN_
        if (lrc != MI355_OK) return lrc;
        MI355_CHECK_LAUNCH("scored_decode_kernel");
        const int pairs = B * kv->nkv, chunks = weights ? cdiv(max_seq_len, 1024) : 0, joins = cdiv(pairs * pl.ncol, 4);
        const dim3 grid(joins + pairs * chunks);
        if (kv->hd == 128) { if (bf) hipLaunchKernelGGL((scored_join_kernel<128, true>), grid, dim3(256), 0, st, p, joins, chunks); else hipLaunchKernelGGL((scored_join_kernel<128, false>), grid, dim3(256), 0, st, p, joins, chunks); }
        else               { if (bf) hipLaunchKernelGGL((scored_join_kernel<64, true>), grid, dim3(256), 0, st, p, joins, chunks); else hipLaunchKernelGGL((scored_join_kernel<64, false>), grid, dim3(256), 0, st, p, joins, chunks); }
        MI355_CHECK_LAUNCH("scored_join_kernel");
        return MI355_OK;
    }
    if (weights && !lse) p.lse = (float*)(ws + pl.lse);
    const ScoredParams& sp = p;
    const dim3 grid(cdiv(q_len * nh, 4), B), wgrid(cdiv(max_seq_len, 256), kv->nkv, B);
#define L_(HD_, BF_, I8_) do { hipLaunchKernelGGL((scored_rows_kernel<HD_, BF_, I8_>), grid, dim3(256), 0, st, sp); \
                               if (weights) hipLaunchKernelGGL((scored_weights_kernel<HD_, BF_, I8_>), wgrid, dim3(256), 0, st, sp); } while (0)
#define LB_(HD_) do { if (bf) { if (int8) L_(HD_, true, true); else L_(HD_, true, false); } else { if (int8) L_(HD_, false, true); else L_(HD_, false, false); } } while (0)
    if (kv->hd == 128) LB_(128); else LB_(64);
#undef LB_
#undef L_
    MI355_CHECK_LAUNCH("paged_attn_scored");
    return MI355_OK;
}
