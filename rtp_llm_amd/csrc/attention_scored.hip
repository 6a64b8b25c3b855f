// Paged attention with score forms, gfx950: scores capped by a tanh and biased by distance, rows that see an interval of the cache (causal, windows, prefixes,
// documents), log-sum-exps, and the attention weight that each cached token draws (what kv_evict.hip ranks them by).
//
//   u = scale q.k        s = cap tanh(u / cap)  (cap > 0, else u)        s += slope[h] (key position - row position)
//   row r, head h:  p_j = exp(s_j - lse),  lse = log sum_j exp(s_j),  out = sum_j p_j V_j   over the slots j in [begin[r], end[r]); an empty interval: out 0, lse -inf
//   weights[j, kv head] <- decay weights[j, kv head] + sum over the call's rows of the sequence and the heads of the group of p_j
//
// Everything is kept in the log2 domain: s2 = s log2(e), p = exp2(s2 - m) / l with m a column's running maximum and l its sum.  The weights are formed from m and l, not from their
// logarithm: under distance biases of thousands that alone would be off by 5e-4 of a weight.
//
// Roundings to 16 bits, by choice: a probability (8-bit caches: times its value's scale, an fp32 number) to the activations' type before the second product, since matrix instructions that take
// fp32 run at a sixteenth of the rate, and results.  Scores, maxima, sums, weights, parts and log-sum-exps stay fp32.  Relative errors of outputs against 64 bits, as computed in fp32 and rounded
// once / here: 8 x 512 rows in fp16 2.07e-4 / 2.33e-4, 333 rows over 8 bits 2.07e-4 / 2.6e-4, documents in bf16 1.65e-3 / 1.81e-3.
#include <algorithm>
#include <type_traits>

#include "common.h"
#include "internal.h"
#include "scored.h"

namespace {

// Values that are not finite, in slots that some rows see and others do not: the second product would make zero times one, not a number, of them in the rows that do not.  Where a tile is
// masked its fragments (8 values of 16 bits) are looked at, and from one that has some they go into two of their own, as 2^127 where a row that sees the slot gets +inf (+inf, NaN) and as
// -2^127 where it gets -inf (-inf, NaN); times 2^127 for a slot that a column sees and 0 for others, in bf16, they become just that, and both together NaN.
template <bool BF> __device__ __forceinline__ uint32_t odd_bits(u32x4 a) {          // not 0: an exponent of ones
    constexpr uint32_t E = BF ? 0x7F807F80u : 0x7C007C00u, ONE = BF ? 0x00800080u : 0x04000400u;
    return (((a[0] & E) + ONE) | ((a[1] & E) + ONE) | ((a[2] & E) + ONE) | ((a[3] & E) + ONE)) & 0x80008000u;
}
template <bool BF> __device__ __forceinline__ void take_odd(u32x4& a, u32x4& up, u32x4& down) {
    constexpr uint32_t E = BF ? 0x7F80u : 0x7C00u, BIG = 0x7F00u;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        uint32_t keep = 0, u = 0, d = 0;
#pragma unroll
        for (int x = 0; x < 32; x += 16) {
            const uint32_t v = a[w] >> x & 0xFFFFu, mag = v & 0x7FFFu;
            keep |= mag < E ? v << x : 0u;
            u |= mag > E || v == E ? BIG << x : 0u;
            d |= mag > E || (mag == E && v != E) ? (BIG | 0x8000u) << x : 0u;
        }
        a[w] = keep; up[w] = u; down[w] = d;
    }
}
// 2^127 in bf16 for those of the 8 slots t .. t + 7 in [lo, hi)
__device__ __forceinline__ u32x4 seen_big(int t, int lo, int hi) {
    u32x4 r;
#pragma unroll
    for (int w = 0; w < 4; ++w) r[w] = (t + 2 * w >= lo && t + 2 * w < hi ? 0x7F00u : 0u) | (t + 2 * w + 1 >= lo && t + 2 * w + 1 < hi ? 0x7F000000u : 0u);
    return r;
}

// ================================================================================================ few rows
// A (row, head) pair of a sequence's key/value head is one of 16 columns of v_mfma_f32_16x16x32: S^T = K q^T with 16 tokens and O^T = V^T P with 16 channels as rows, so keys and values are
// read once for up to 32 pairs (two tiles of columns).  The two 16-token halves of a 32-token group take the tokens {8 w + r} and {8 w + 4 + r}, w = lane / 16, so that the lane that holds
// eight scores of a column holds the same eight as the second product's operand: nothing crosses lanes between the products.
// A wave walks its groups on its own.  They come by DMA into a ring of its own in LDS: what is in flight takes no registers, and a page's 16 tokens are one scalar base for loads
// whose lanes' offsets never change.  A key's 16-byte pieces are swizzled by the token, a channel's 16 values stay side by side.
//
// Work: the tokens that any row of a sequence sees, in units of a group of 32 for each of a block's waves, times key/value heads, laid end to end over all sequences and dealt to the
// blocks in equal runs.  A pair of a sequence and a head that lies inside one run is finished there, others leave a part in each run and scored_join_kernel merges them.  Sequences
// of unequal length so take the time of their mean: a run may end one pair and begin the next.
// Bound by memory: 64 sequences of up to 1024 tokens (28 over 4 heads of 128, 80 MB) 22 us, 3.6 TB/s, where a sum over a large array reads 4.0; one row over one short sequence is latency, 7 us.
// Two to four rows a sequence, 64 sequences of 1000 (131 MB), with the join: 32 and 38 us, 4 tracked ones 54, over 8 bits 33.
struct DecodeParams : ScoredParams {
    float*   tmp_out;    // [2 nblocks][ncol][hd]: parts; a run's first segment in slot 2 run, a later one that goes on in the next run in 2 run + 1
    float*   tmp_ml;     // [2 nblocks][ncol][2]
    float*   ml_all;     // [pairs][ncol][2] of pairs that were finished in one run (with weights)
    float*   spill;      // [pairs][ncol][ctx_pad] scores in the log2 domain (with weights), from the sequence's first unit on
    int4*    meta;       // [pairs]: first slot, parts, the sequence's first seen slot rounded down to 32, its reach
    int      nblocks, ncol, ctx_pad, runs;   // runs: 0 = a block per pair
};

// The slots that a sequence's rows see lie in [lo, hi), lo a multiple of 32; nothing: zeros.
__device__ __forceinline__ void scored_span(const ScoredParams& p, int base, int len, int& lo, int& hi) {
    int seen = 0x7fffffff;
    hi = 0;
    for (int i = 0; i < len; ++i) {
        int a, e;
        scored_interval(p, base + i, a, e);
        if (e > a) { seen = min(seen, a); hi = max(hi, e); }
    }
    lo = hi == 0 ? 0 : seen & ~31;
}

// a row's reference of biases where the thread writes its log-sum-exp
__device__ __forceinline__ int lse_ref(const ScoredParams& p, int b, int kh, int d0, int hi) { return p.slopes && p.lse && d0 == 0 && hi > 0 ? scored_ref(p, b, kh, hi) : 0; }

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

// Waves of a block, LDS of a wave's stage (keys, values, and, EXTRA, 1 KB of scales and positions), stages.  What is in flight fills LDS either way; eight waves, two a SIMD, hide what a group's chain
// of product, softmax and product leaves idle, where a stage is 8 KB or less and the registers of two tiles of columns are not in the way.  us with the join by four / by eight, one row a sequence:
// 8 bits, 28 over 4 heads of 128: 1 x 1000 slots 9.8 / 10.3, 13 x 4000 23.7 / 19.5, 64 x 1000 22.4 / 20.3, 4 x 30000 38.7 / 33.5; 16 bits, 14 over 2 of 64: 9.1 / 9.7, 14.1 / 13.4, 14.8 / 14.1,
// 20.6 / 18.7.
template <int HD, bool INT8, int NT, bool EXTRA> struct Ring {
    static constexpr int ES = INT8 ? 1 : 2, KB = 32 * HD * ES, LOADS = 2 * KB / 1024 + (EXTRA ? 1 : 0), STAGE = LOADS * 1024, NW = NT == 1 && (INT8 || HD == 64) ? 8 : 4;
    static constexpr int N = HD == 128 && !INT8 ? 2 : NW == 4 ? 4 : HD == 64 && INT8 ? 3 : 2, UNIT = 32 * NW;
    static constexpr int MERGE = NW * 16 * (HD + 4) * 4 + 2 * NW * 16 * 4, BYTES = NW * N * STAGE > MERGE ? NW * N * STAGE : MERGE;
    static_assert(BYTES <= 160 * 1024 && LOADS * (N - 1) < 63, "");
};

template <int HD, bool INT8, int NT, bool BF, bool KP>
__global__ __launch_bounds__((NT == 1 && (INT8 || HD == 64) ? 512 : 256)) void scored_decode_kernel(const DecodeParams p) {
    constexpr bool EXTRA = INT8 || KP;
    // 8 bits under fp16: probabilities take the value's scale, an amax / 127, before they are rounded.  64 of it keep the small ones out of fp16's subnormals (amax <= 65504: 64 scales fit) if
    // no probability exceeds 1.
    constexpr float VS = INT8 && !BF ? 64.f : 1.f, DEFER = INT8 && !BF ? 0.f : 6.f;
    using R = Ring<HD, INT8, NT, EXTRA>;
    constexpr int NW = R::NW, UNIT = R::UNIT, NTHR = 64 * NW;
    auto units_of = [](int from, int to) { return (to - from + UNIT - 1) / UNIT; };
    constexpr int NSTEP = HD / 32, NDB = HD / 16, ES = R::ES, CK = HD * ES / 16, RS = R::N;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int j = lane & 15, w = lane >> 4;
    extern __shared__ __attribute__((aligned(16))) char dec_sm[];
    auto s_o = reinterpret_cast<float(*)[16][HD + 4]>(dec_sm);                        // the merge's, over the ring
    auto s_m = reinterpret_cast<float(*)[16]>(dec_sm + NW * 16 * (HD + 4) * 4);
    float(*s_l)[16] = s_m + NW;
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

    // ---- this block's run of units.  Lane i looks at sequence i of each 64; up to 64 sequences its answers are all that the block needs of them.
    int b, kh, lo, hi, base, len, units, u, u1;  // the pair at hand, its span and rows, the run's next unit inside it, the run's end (counted from the pair's first unit)
    int my_lo = 0, my_hi = 0, my_base = 0, my_len = 0;
    auto look = [&](int b0) {
        my_lo = my_hi = my_base = my_len = 0;
        if (b0 + lane < p.B) { scored_rows_of(p, b0 + lane, my_base, my_len); scored_span(p, my_base, my_len, my_lo, my_hi); }
    };
    auto take = [&](int who) {
        if (p.B > 64) { look(who & ~63); who &= 63; }
        lo = __builtin_amdgcn_readlane(my_lo, who); hi = __builtin_amdgcn_readlane(my_hi, who);
        base = __builtin_amdgcn_readlane(my_base, who); len = __builtin_amdgcn_readlane(my_len, who);
        units = units_of(lo, hi);
    };
    if (p.runs) {
        int total = 0, incl = 0;
        for (int b0 = 0; b0 < p.B; b0 += 64) {
            look(b0);
            incl = units_of(my_lo, my_hi) * p.nkv;
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) { const int up = __shfl_up(incl, o); if (lane >= o) incl += up; }
            total += __builtin_amdgcn_readlane(incl, 63);
        }
        const int W = max(1, (total + p.nblocks - 1) / p.nblocks), start = blockIdx.x * W, stop = min(total, start + W);
        if (start >= stop && blockIdx.x != 0) return;
        int before = 0, at = -1, at_s = 0;          // units before this group of 64 sequences; the sequence in which the run begins
        for (int b0 = 0; b0 < p.B; b0 += 64) {
            if (p.B > 64) {
                look(b0);
                incl = units_of(my_lo, my_hi) * p.nkv;
#pragma unroll
                for (int o = 1; o < 64; o <<= 1) { const int up = __shfl_up(incl, o); if (lane >= o) incl += up; }
            }
            const int per = units_of(my_lo, my_hi), n = per * p.nkv, s = before + incl - n;
            if (blockIdx.x == 0 && wave == 0 && b0 + lane < p.B)
                for (int k = 0; k < p.nkv; ++k) {
                    const int a = s + k * per, e = a + per, r0 = a / W, r1 = per ? (e - 1) / W : r0 - 1;
                    p.meta[(size_t)(b0 + lane) * p.nkv + k] = make_int4(2 * r0 + (a == r0 * W ? 0 : 1), r1 - r0 + 1, my_lo, my_hi);
                }
            const uint64_t in = __builtin_amdgcn_ballot_w64(start >= s && start < s + n);
            if (in && at < 0) { const int who = __builtin_ctzll(in); at = b0 + who; at_s = __builtin_amdgcn_readlane(s, who); }
            before += __builtin_amdgcn_readlane(incl, 63);
            if (at >= 0 && blockIdx.x != 0) break;
        }
        if (start >= stop) return;
        b = at;
        take(b);
        kh = (start - at_s) / units;
        u = start - at_s - kh * units;
        u1 = u + stop - start;
    } else {
        b = blockIdx.x / p.nkv; kh = blockIdx.x - b * p.nkv;
        scored_rows_of(p, b, base, len);
        scored_span(p, base, len, lo, hi);
        lo = __builtin_amdgcn_readfirstlane(lo); hi = __builtin_amdgcn_readfirstlane(hi);
        base = __builtin_amdgcn_readfirstlane(base); len = __builtin_amdgcn_readfirstlane(len);
        units = units_of(lo, hi); u = 0; u1 = units;
        if (tid == 0) p.meta[blockIdx.x] = make_int4(0, units ? 1 : 0, lo, hi);
    }

    bool first = true;
    while (u1 > 0) {                                // segments: units [u, min(u1, units)) of pair (b, kh)
        const int stop_u = min(u1, units);
        const bool whole = u == 0 && stop_u == units;
        const int ncol = len * p.G;
        const int pstart = lo + u * UNIT, pend = min(hi, lo + stop_u * UNIT);
        const int32_t* bt = p.block_table + (size_t)b * p.max_blocks;
        const size_t pair = (size_t)b * p.nkv + kh;

        // the first groups' block ids are asked for together with the queries
        const int last16 = (hi - 1) & ~15;
        int idv = 0;                                // block ids of 32 groups' units, a lane each
        auto ids_of = [&](int i) {
            const int t = min(pstart + wave * 32 + (i + (lane >> 1)) * UNIT + (lane & 1) * 16, last16);
            idv = bt[(int)(((unsigned long long)(unsigned)t * p.page_magic) >> 32)];
        };
        ids_of(0);
        u32x4 qf[NT][NSTEP];
        int c_lo[NT], c_hi[NT], ref[NT];
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
            ref[c] = p.slopes && c_hi[c] > 0 ? scored_ref(p, b, kh, c_hi[c]) : 0;
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
        auto page_of = [&](int t) { return (int)__builtin_amdgcn_readfirstlane((int)(((unsigned long long)(unsigned)t * p.page_magic) >> 32)); };
        const uint32_t head_bytes = (uint32_t)(p.page * HD * ES);
        auto issue = [&](int i, int buf) {
            const int tb = pstart + wave * 32 + i * UNIT;
            if ((i & 31) == 0 && i > 0) {
                ids_of(i);
                wait_vm<0>();                       // here, where it is rare: left to the compiler the wait, for everything in flight, stands in every round
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
                        sv[e] = __builtin_fmaf(slope2[c], (float)(kp - ref[c]), sv[e]);
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
                    if (MASKED && __builtin_amdgcn_ballot_w64(odd_bits<BF>(a) != 0)) {
                        u32x4 up, down;
                        take_odd<BF>(a, up, down);
#pragma unroll
                        for (int c = 0; c < NT; ++c) {
                            const u32x4 big = seen_big(vwin, c_lo[c], c_hi[c]);
                            o[c][db] = mfma_act<true>(up, big, o[c][db]);
                            o[c][db] = mfma_act<true>(down, big, o[c][db]);
                        }
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
        // ---- the waves meet in LDS, a tile of columns at a time
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
            for (int idx = tid; idx < here * (HD / 4); idx += NTHR) {
                const int jj = idx / (HD / 4), d0 = (idx - jj * (HD / 4)) * 4, col = c * 16 + jj;
                float mstar = s_m[0][jj];
#pragma unroll
                for (int ww = 1; ww < NW; ++ww) mstar = fmaxf(mstar, s_m[ww][jj]);
                f32x4 acc = {0.f, 0.f, 0.f, 0.f};
                float l = 0.f;
#pragma unroll
                for (int ww = 0; ww < NW; ++ww) {
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
                    scored_store<BF>(p, row, h, HD, d0, acc, mstar, l, e > a, lse_ref(p, b, kh, d0, e));
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
                take(b);
            } while (units == 0);
        }
    }
}

// What the runs left: columns whose pair has several parts are merged (zeros where there is none), and, behind those blocks, a thread per slot adds the
// probabilities of all columns to the slot's weight.
template <int HD, bool BF, int SL, int CPB>
__global__ __launch_bounds__(256) void scored_join_kernel(const DecodeParams p, int join_blocks, int chunks) {
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    auto slot_of = [](const int4& mt, int i) { return i == 0 ? mt.x : (mt.x / 2 + i) * 2; };
    if ((int)blockIdx.x < join_blocks) {
        // CPB columns a block; groups of HD / 4 threads share a column's parts, eight in flight each: few columns, whose pairs have many parts, take a block each (heads of 128: 64 parts in one
        // round trip), many take a wave
        constexpr int TP = HD / 4, NG = 256 / TP, NGC = NG / CPB;
        __shared__ f32x4 s_acc[NG][TP];
        __shared__ float2 s_ml[NG];
        const int all_grp = tid / TP, grp = all_grp % NGC, d0 = tid % TP * 4, gid = blockIdx.x * CPB + all_grp / NGC;
        const int pair = min(gid / p.ncol, p.B * p.nkv - 1), col = gid % p.ncol, b = pair / p.nkv, kh = pair - b * p.nkv;
        const int4 mt = p.meta[pair];
        int base, len;
        scored_rows_of(p, b, base, len);
        const bool on = gid < p.B * p.nkv * p.ncol && mt.y != 1 && col < len * p.G;
        const int rl = on ? col / p.G : 0, row = on ? base + rl : 0, h = kh * p.G + (on ? col - rl * p.G : 0);
        float m = NEG_BIG, l = 0.f;
        f32x4 acc = {0.f, 0.f, 0.f, 0.f};
        for (int i0 = grp; on && i0 < mt.y; i0 += NGC * 8) {
            float2 ml[8];
            f32x4 v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const size_t at = (size_t)slot_of(mt, min(i0 + i * NGC, mt.y - 1)) * p.ncol + col;
                ml[i] = *reinterpret_cast<const float2*>(p.tmp_ml + at * 2);
                v[i] = *reinterpret_cast<const f32x4*>(p.tmp_out + at * HD + d0);
            }
            float mn = m;
#pragma unroll
            for (int i = 0; i < 8; ++i) mn = fmaxf(mn, ml[i].x);
            const float f0 = __builtin_amdgcn_exp2f(m - mn);
            l *= f0; acc *= f0; m = mn;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if (i0 + i * NGC >= mt.y) continue;
                const float f = __builtin_amdgcn_exp2f(ml[i].x - m);
                l += ml[i].y * f;
                acc += v[i] * f;
            }
        }
        s_acc[all_grp][tid % TP] = acc;
        if (d0 == 0) s_ml[all_grp] = make_float2(m, l);
        __syncthreads();
        if (grp != 0 || !on) return;
        float mn = m;
#pragma unroll
        for (int g = 1; g < NGC; ++g) mn = fmaxf(mn, s_ml[all_grp + g].x);
        const float f0 = __builtin_amdgcn_exp2f(m - mn);
        l *= f0; acc *= f0;
#pragma unroll
        for (int g = 1; g < NGC; ++g) {
            const float f = __builtin_amdgcn_exp2f(s_ml[all_grp + g].x - mn);
            l += s_ml[all_grp + g].y * f;
            acc += s_acc[all_grp + g][tid % TP] * f;
        }
        int a, e;
        scored_interval(p, row, a, e);
        scored_store<BF>(p, row, h, HD, d0, acc, mn, l, e > a, lse_ref(p, b, kh, d0, e));
        return;
    }
    // ---- weights: SL slots a thread, the first scores asked for before the columns' maxima and sums are merged
    __shared__ float s_m[32], s_i[32];
    __shared__ int2 s_seen[32];                                      // what a column sees: by the score alone a slot of -inf were one that it does not see, and a column that is not a number passed it over
    typedef float slots __attribute__((ext_vector_type(SL)));
    const int id = blockIdx.x - join_blocks, pair = id / chunks, chunk = id - pair * chunks;
    const int4 mt = p.meta[pair];
    if (chunk * 256 * SL >= mt.w) return;
    const int b = pair / p.nkv, kh = pair - b * p.nkv;
    int base, len;
    scored_rows_of(p, b, base, len);
    const int ncol = len * p.G;
    const int t = (chunk * 256 + tid) * SL;                          // four slots lie inside a page
    const bool in = t < mt.w;
    const int blk = in ? p.block_table[(size_t)b * p.max_blocks + (int)(((unsigned long long)(unsigned)t * p.page_magic) >> 32)] : -1;
    const float* sp = p.spill + (size_t)pair * p.ncol * p.ctx_pad + max(t - mt.z, 0);
    const bool some = in && t >= mt.z;
    slots v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (some) v[i] = *reinterpret_cast<const slots*>(sp + (size_t)min(i, ncol - 1) * p.ctx_pad);
    for (int col = wave; col < ncol; col += 4) {
        float m = NEG_BIG, l = 0.f;
        if (mt.y == 1) {
            const float2 x = *reinterpret_cast<const float2*>(p.ml_all + ((size_t)pair * p.ncol + col) * 2);
            m = x.x; l = x.y;
        } else {
            for (int i = lane; i < mt.y; i += 64) {
                const float2 x = *reinterpret_cast<const float2*>(p.tmp_ml + ((size_t)slot_of(mt, i) * p.ncol + col) * 2);
                const float mn = fmaxf(m, x.x);
                l = l * __builtin_amdgcn_exp2f(m - mn) + x.y * __builtin_amdgcn_exp2f(x.x - mn);
                m = mn;
            }
            const float mine = m;
            m = wave_max(m);
            l = wave_sum(l * __builtin_amdgcn_exp2f(mine - m));
        }
        int a, e;
        scored_interval(p, base + col / p.G, a, e);
        if (lane == 0) { s_m[col] = m; s_i[col] = scored_inv(l, e > a); s_seen[col] = make_int2(a, e); }
    }
    __syncthreads();
    if (!in || blk < 0 || blk >= p.num_blocks) return;
    float* to = p.weights + ((size_t)blk * p.nkv + kh) * p.page + t % p.page;
    slots old, sum;
#pragma unroll
    for (int e = 0; e < SL; ++e) { sum[e] = 0.f; old[e] = t + e < mt.w ? to[e] : 0.f; }
    if (some)
        for (int c0 = 0; c0 < ncol; c0 += 8) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if (c0 + i >= ncol) continue;
                const float m = s_m[c0 + i], inv = s_i[c0 + i];
                const int2 seen = s_seen[c0 + i];
#pragma unroll
                for (int e = 0; e < SL; ++e) sum[e] += t + e >= seen.x && t + e < seen.y ? __builtin_amdgcn_exp2f(v[i][e] - m) * inv : 0.f;
            }
            if (c0 + 8 < ncol) {
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = *reinterpret_cast<const slots*>(sp + (size_t)min(c0 + 8 + i, ncol - 1) * p.ctx_pad);
            }
        }
#pragma unroll
    for (int e = 0; e < SL; ++e)
        if (t + e < mt.w) to[e] = scored_decayed(p, old[e], sum[e]);
}

// ================================================================================================ many rows
// A wave owns 32 (row, head) pairs of a sequence's key/value head as the columns of v_mfma_f32_32x32x16, a block NW times as many: pairs lie row by row, the heads of a row side by side, so
// any number of heads per kv head fills the tiles, and a tile spans few rows (its keys end soon behind its rows).  S^T = K q^T takes 32 keys as rows in the order
// 16 (i / 2) + 8 half + 4 (i & 1) + r for row 8 i + 4 half + r: what a lane then holds of its column are two runs of eight keys, the second product's operand as it stands.
// Keys and values come 64 at a time through LDS for all waves: by DMA, two steps ahead of the products with one barrier a step (three stages), or, 8 bits, through registers, which widen them
// once for all waves.  A key's 16-byte pieces are swizzled by its low bits, a channel's 16 tokens lie side by side: no bank conflicts in either product's reads.
// 28 heads of 128, a launch among its like: 2 x 2048 rows behind 2048 slots 213 us (0.85 PFLOP/s; 239 in a trace of single passes), 4096 behind 12288 895 (0.94), 8 x 512 capped 42 (47), biased 45.
// Products take 43% of the busy time of a compute unit in the first of these, vector instructions 44%: what is left is waiting, of the two kinds for each other in a wave and at a step's barrier.  A
// wave reads 32 KB of fragments a step for 32 columns: at 128 bytes a clock LDS would be as busy as the products at their full rate.
// 8 bits: 2 x 2048 behind 2048 276 us, 8 x 512 44, 333 rows behind 3001 48 in 10 parts.  The codes that are held over the products cost heads of 128 registers: 2 to 12 are spilled with eight waves, 17
// to 25 with four.
// What the weights' pass needs of a column.
struct Col { float m, inv, slope2; int ref, lo, hi, pad0, pad1; };
static_assert(sizeof(Col) == 32, "two 16-byte loads");
struct ChunkParams : ScoredParams {
    float*  tmp_out;       // [parts][nkv][rows G][hd] (parts > 1)
    float4* tmp_ml;        // [parts][nkv][rows G]: maximum, sum, the reference of biases
    Col*    cols;          // [nkv][rows G] (with weights)
    float*  shares;        // [splits][B][nkv][max_seq] (splits > 1)
    int*    reach;         // [B], behind the shares
    int     tiles, parts;  // column tiles of the longest sequence, parts of the keys
    uint32_t g_magic;      // 2^32 / G + 1
};
// a key's swizzle: distinct over the keys that eight (rows of 128 bytes) or sixteen (256) neighbouring lanes read
template <int CK> __device__ __forceinline__ int swizzle_of(int t) { return CK == 16 ? t & 15 : (t & 3) | (t >> 3 & 1) << 2; }
typedef float f32x16 __attribute__((ext_vector_type(16)));
template <bool BF> __device__ __forceinline__ f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c) {
    if constexpr (BF) return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    else              return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
// a commutative combination, in which a value may count twice, over lanes 0 to 31 and 32 to 63 each, without LDS
template <class F> __device__ __forceinline__ int row32(int v, F&& f) {
    v = f(v, __builtin_amdgcn_update_dpp(v, v, 0xB1, 0xF, 0xF, false));      // lanes' neighbours in fours: 1 0 3 2
    v = f(v, __builtin_amdgcn_update_dpp(v, v, 0x4E, 0xF, 0xF, false));      // 2 3 0 1
    v = f(v, __builtin_amdgcn_update_dpp(v, v, 0x141, 0xF, 0xF, false));     // eights mirrored
    v = f(v, __builtin_amdgcn_update_dpp(v, v, 0x140, 0xF, 0xF, false));     // sixteens mirrored
    float a, c;
    swap16(__builtin_bit_cast(float, v), a, c);
    return f(__builtin_bit_cast(int, a), __builtin_bit_cast(int, c));
}
// a barrier for what lies in LDS: loads from memory and DMA stay in flight (__syncthreads waits for them)
__device__ __forceinline__ void lds_barrier() {
    wait_vm<63>();
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}
enum { FORM_PLAIN, FORM_CAP, FORM_BIAS };           // FORM_BIAS: capped or not

template <int HD, bool INT8, int NW> struct Stage {
    static constexpr int KEYS = 64, KB = KEYS * HD * 2, BYTES = 2 * KB + (INT8 ? 2 * KEYS * 4 : 0), N = INT8 || (HD == 128 && NW < 8) ? 2 : 3, LDS = N * BYTES + 64;
};

template <int HD, bool INT8, bool BF, int FORM, int NW>
__global__ __launch_bounds__(64 * NW, 2) void scored_chunk_kernel(const ChunkParams p) {
    using ST = Stage<HD, INT8, NW>;
    constexpr int KS = HD / 16, NDB = HD / 32, KB = ST::KB, ROW = HD * 2, CK = ROW / 16;
    constexpr float VS = INT8 && !BF ? 64.f : 1.f, DEFER = INT8 && !BF ? 0.f : 6.f;      // as in scored_decode_kernel
    extern __shared__ __attribute__((aligned(16))) char ch_sm[];
    int* lim = reinterpret_cast<int*>(ch_sm + ST::N * ST::BYTES);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), col = lane & 31, half = lane >> 5;
    // late tiles, which see most, first; a sequence's and head's blocks are B nkv parts apart, on one XCD where 8 divides that
    int id = blockIdx.x;
    const int part = id % p.parts; id /= p.parts;
    const int kh = id % p.nkv; id /= p.nkv;
    const int b = id % p.B, tile = p.tiles - 1 - id / p.B;
    int base, len;
    scored_rows_of(p, b, base, len);
    const int ncol = len * p.G, c0 = tile * 32 * NW + wave * 32;
    if (tile * 32 * NW >= ncol) return;
    const bool ok = c0 + col < ncol;
    const int cc = min(c0 + col, ncol - 1), rl = cc / p.G, row = base + rl, h = kh * p.G + cc - rl * p.G;
    int lo, hi;
    scored_interval(p, row, lo, hi);
    if (!ok) lo = hi = 0;
    const bool seen = hi > lo;
    u32x4 qf[KS];
#pragma unroll
    for (int s = 0; s < KS; ++s) qf[s] = *reinterpret_cast<const u32x4*>(reinterpret_cast<const uint16_t*>(p.q) + (size_t)row * p.ldq + h * HD + s * 16 + half * 8);
    const int ref = FORM == FORM_BIAS && seen ? scored_ref(p, b, kh, hi) : 0;
    const int32_t* bt = p.block_table + (size_t)b * p.max_blocks;
    int idv = 0;                                    // block ids of 16 steps' units of 16 keys, a lane each
    auto ids_of = [&](int t0, int last) {
        const int t = min(t0 + lane * 16, last);
        idv = bt[(int)(((unsigned long long)(unsigned)t * p.page_magic) >> 32)];
        wait_vm<0>();                               // here, where it is rare: left to the compiler the wait, for everything in flight, stands in every step
    };
    // Where the walk begins is known before what the rows see is where that starts at slot 0: the first stages are then on their way during the reductions below (what they read behind the
    // last seen slot, inside the pool, is masked).
    const bool early = !INT8 && !p.begin && p.parts == 1;
    if (early) ids_of(0, (p.max_seq - 1) & ~15);
    auto page_of = [&](int t) { return (int)__builtin_amdgcn_readfirstlane((int)(((unsigned long long)(unsigned)t * p.page_magic) >> 32)); };
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)ch_sm;
    int klo = 0, s0 = 0, last16 = (p.max_seq - 1) & ~15;
    auto ids_for = [&](int st) { if (((st - s0) & 15) == 0 && !(early && st == s0)) ids_of(klo + st * 64, last16); };
    // base of a unit's keys and values; a unit past the last seen slot is that one's again (masked)
    const uint32_t head_elems = (uint32_t)(p.page * HD);
    auto unit_at = [&](int st, int u, int& ti, uint32_t& hk) {
        const int t = min(klo + st * 64 + u * 16, last16);
        ti = t - page_of(t) * p.page;
        hk = (uint32_t)min(max(__builtin_amdgcn_readlane(idv, ((st - s0) & 15) * 4 + u), 0), p.num_blocks - 1) * (uint32_t)(2 * p.nkv) + (uint32_t)kh;
    };
    // ---- 16 bits: 1 KB loads, KL of keys (1024 / ROW keys each) and as many of values (32 channels of a unit each) a stage
    constexpr int KL = KB / 1024, JK = KL / NW, KU = KL / 4;                          // loads of keys a stage, a wave, a unit
    const int krow = (wave % KU) * (1024 / ROW) + lane / CK;
    const uint32_t koff = (uint32_t)(krow * ROW + (((lane % CK) ^ swizzle_of<CK>(krow)) << 4)), voff = (uint32_t)((lane >> 1) * p.page + (lane & 1) * 8) * 2u;
    auto issue = [&](int st, int buf) {
        ids_for(st);
#pragma unroll
        for (int j = 0; j < JK; ++j) {
            const int d = j * NW + wave;
            int ti; uint32_t hk;
            unit_at(st, d / KU, ti, hk);
            const uint16_t* kb = (const uint16_t*)p.kv_base + (uint64_t)hk * head_elems;
            const uint32_t to = __builtin_amdgcn_readfirstlane(lds0 + buf * ST::BYTES + d * 1024);
            dma16(to, koff, kb + (uint32_t)(ti * HD));
            dma16(to + KB, voff, kb + (uint64_t)(uint32_t)p.nkv * head_elems + (uint32_t)ti + (uint32_t)(d % KU * 32) * (uint32_t)p.page);
        }
    };
    if constexpr (!INT8) if (early) { issue(0, 0); if (ST::N > 2) issue(1, 1); }
    // [wlo, whi): what some column of the wave sees; [ilo, ihi): what all do (columns that see nothing do not count)
    if (tid == 0) { lim[0] = 0x7fffffff; lim[1] = 0; }
    lds_barrier();
    const int wlo = __builtin_amdgcn_readfirstlane(row32(seen ? lo : 0x7fffffff, [](int a, int c) { return min(a, c); })), whi = __builtin_amdgcn_readfirstlane(row32(hi, [](int a, int c) { return max(a, c); }));
    const int ilo = __builtin_amdgcn_readfirstlane(row32(lo, [](int a, int c) { return max(a, c); })), ihi = __builtin_amdgcn_readfirstlane(row32(seen ? hi : 0x7fffffff, [](int a, int c) { return min(a, c); }));
    if (lane == 0) { atomicMin(&lim[0], wlo); atomicMax(&lim[1], whi); }
    lds_barrier();
    const int seen0 = __builtin_amdgcn_readfirstlane(lim[0]), khi = __builtin_amdgcn_readfirstlane(lim[1]);
    klo = khi > 0 ? seen0 & ~63 : 0;
    const int all = (khi - klo + 63) / 64, s1 = (int)((long)all * (part + 1) / p.parts);           // this part's steps
    s0 = (int)((long)all * part / p.parts);
    last16 = khi > 0 ? (khi - 1) & ~15 : 0;
    const float slope2 = FORM == FORM_BIAS ? p.slopes[h] * kLog2e : 0.f;
    f32x16 o[NDB];
#pragma unroll
    for (int d = 0; d < NDB; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[d][i] = 0.f;
    float m = NEG_BIG, l = 0.f;
#pragma unroll
    for (int s = 0; s < KS; ++s)
        if (!ok) qf[s] = u32x4{0u, 0u, 0u, 0u};
    // ---- 8 bits: 16-byte pieces through registers, a thread takes the same piece numbers of every stage
    constexpr int PIECES = 64 * HD / 16, JP = INT8 ? (PIECES + 64 * NW - 1) / (64 * NW) : 1;
    u32x4 rk[JP], rv[JP];
    float rs = 0.f;
    auto fetch8 = [&](int st) {
        ids_for(st);
#pragma unroll
        for (int j = 0; j < JP; ++j) {
            const int i = j * 64 * NW + tid, u = __builtin_amdgcn_readfirstlane(i / HD);          // HD pieces a unit: whole waves (HD 64, 128)
            int ti; uint32_t hk;
            unit_at(st, min(u, 3), ti, hk);
            const char* kb = (const char*)p.kv_base + (uint64_t)hk * head_elems;
            const int q = i % HD;
            rk[j] = *reinterpret_cast<const u32x4*>(kb + ti * HD + q * 16);
            rv[j] = *reinterpret_cast<const u32x4*>(kb + (uint64_t)(uint32_t)p.nkv * head_elems + q * p.page + ti);
        }
        if (tid < 128) {                            // scales: 64 of keys, 64 of values
            const int t = min(klo + st * 64 + (tid & 63 & ~15), last16), blk = __shfl(idv, ((st - s0) & 15) * 4 + ((tid & 63) >> 4));
            const size_t hk = (size_t)min(max(blk, 0), p.num_blocks - 1) * 2 * p.nkv + kh + (tid >= 64 ? p.nkv : 0);
            rs = p.scale_base[hk * p.page + t % p.page + (tid & 15)];
            const int key = klo + st * 64 + (tid & 63);
            if (key >= khi || key < seen0) rs = 0.f;    // whatever the pool holds there
        }
    };
    auto store8 = [&](int buf) {
        char* st = ch_sm + buf * ST::BYTES;
#pragma unroll
        for (int j = 0; j < JP; ++j) {
            const int i = j * 64 * NW + tid;
            if (PIECES % (64 * NW) && i >= PIECES) break;
            const int t = i / (HD / 16), c = (i % (HD / 16)) * 2, f = swizzle_of<CK>(t & 15);
            *reinterpret_cast<u32x4*>(st + t * ROW + ((c ^ f) << 4)) = widen_codes<BF>(rk[j][0], rk[j][1]);
            *reinterpret_cast<u32x4*>(st + t * ROW + (((c + 1) ^ f) << 4)) = widen_codes<BF>(rk[j][2], rk[j][3]);
            *reinterpret_cast<u32x4*>(st + KB + i * 32) = widen_codes<BF>(rv[j][0], rv[j][1]);
            *reinterpret_cast<u32x4*>(st + KB + i * 32 + 16) = widen_codes<BF>(rv[j][2], rv[j][3]);
        }
        if (tid < 128) reinterpret_cast<float*>(st + 2 * KB)[tid] = rs;              // 0 for a slot that no row here sees (fetch8)
    };

    // where the lane's fragments lie: its key in a group of 32, that key's pieces
    const int kt = 16 * (col >> 4) + 8 * (col >> 2 & 1) + 4 * (col >> 3 & 1) + (col & 3), kf = swizzle_of<CK>(kt & 15);
    // A step's 64 keys as two groups of 32.  The fragments are asked for a phase ahead of their use (the second group's keys and the first one's values before the first softmax): read where
    // they are used, every product waited for its own.
    auto read_keys = [&](const char* st, int g, u32x4 (&f)[KS]) {
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) f[ks] = *reinterpret_cast<const u32x4*>(st + (g * 32 + kt) * ROW + (((ks * 2 + half) ^ kf) << 4));
    };
    auto read_values = [&](const char* st, int g, u32x4 (&f)[2][NDB]) {
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int d = 0; d < NDB; ++d) f[k][d] = *reinterpret_cast<const u32x4*>(st + KB + ((g * 2 + k) * HD + d * 32 + col) * 32 + half * 16);
    };
    auto scores = [&](const u32x4 (&f)[KS], f32x16& s) {
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] = 0.f;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) s = mfma32<BF>(f[ks], qf[ks], s);
    };
    // scores of a group -> probabilities as the second product's operand; sv[8 kk + e] is key t0 + 16 kk + 8 half + e
    auto weigh = [&](const f32x16& s, const char* st, int g, int t0, u32x4 (&pf)[2], bool masked) {
        float sv[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) sv[i] = s[i];
        if constexpr (INT8) {
            const f32x4* sc = reinterpret_cast<const f32x4*>(st + 2 * KB) + g * 8 + half * 2;
#pragma unroll
            for (int i = 0; i < 16; ++i) sv[i] *= sc[(i >> 3) * 4 + (i >> 2 & 1)][i & 3];
        }
        float mul = p.scale1;                       // scores are sv times mul from here on
        if constexpr (FORM != FORM_PLAIN) {
            if (FORM == FORM_CAP || p.capped) {
#pragma unroll
                for (int i = 0; i < 16; ++i) sv[i] *= p.scale1;
                tanh_all(sv);
                mul = p.cap_log2;
            }
        }
        if constexpr (FORM == FORM_BIAS) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int t = t0 + (k >> 1) * 16 + half * 8 + (k & 1) * 4;
                i32x4 kp = {t - ref, t + 1 - ref, t + 2 - ref, t + 3 - ref};
                if (p.key_pos) {                    // the planes' rows of four tokens lie inside a page
                    const int tc = min(t, last16 + 12), blk = scored_block(p, bt, tc);
                    kp = *reinterpret_cast<const i32x4*>(p.key_pos + ((size_t)blk * p.nkv + kh) * p.page + tc % p.page);
                    kp -= ref;
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) sv[k * 4 + e] = __builtin_fmaf(slope2, (float)kp[e], sv[k * 4 + e] * mul);
            }
            mul = 1.f;
        }
        if (masked) {
            const int a = lo - t0 - half * 8, e = hi - t0 - half * 8;
#pragma unroll
            for (int i = 0; i < 16; ++i) sv[i] = (i >> 3) * 16 + (i & 7) >= a && (i >> 3) * 16 + (i & 7) < e ? sv[i] : -__builtin_inff();
        }
        float mx = -__builtin_inff();
#pragma unroll
        for (int i = 0; i < 16; ++i) mx = fmaxf(mx, sv[i]);
        mx = fmaxf(xor32_max(mx) * mul, NEG_BIG);
        if (__builtin_amdgcn_ballot_w64(mx > m + DEFER)) {
            const float mn = fmaxf(m, mx);
            float alpha = __builtin_amdgcn_exp2f(m - mn);
            l *= alpha;
            // In place, by hand: as plain products the compiler keeps all outputs twice, before and after, copies one over the other and spills.  It does not see what the statements read, so
            // the wait states between a product's issue and a read of its result (11 for the 8 passes of these), and from there to the next product, stand here.
            asm volatile("s_nop 15\n\ts_nop 7" : "+v"(alpha));
#pragma unroll
            for (int d = 0; d < NDB; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i) asm volatile("v_mul_f32 %0, %1, %0" : "+v"(o[d][i]) : "v"(alpha));
            asm volatile("s_nop 7");
            m = mn;
        }
        float psum = 0.f;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            float pe[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                pe[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(sv[k * 8 + e], mul, -m));
                psum += pe[e];
            }
            if constexpr (INT8) {
                const f32x4* vs = reinterpret_cast<const f32x4*>(st + 2 * KB) + 16 + g * 8 + k * 4 + half * 2;
                if (masked) {                       // a scale that is not finite is that of the rows that see it
#pragma unroll
                    for (int e = 0; e < 8; ++e) pe[e] = pe[e] == 0.f ? 0.f : pe[e] * (vs[e >> 2][e & 3] * VS);
                } else {
#pragma unroll
                    for (int e = 0; e < 8; ++e) pe[e] *= vs[e >> 2][e & 3] * VS;
                }
            }
            pf[k] = act_pack8<BF>(pe);
        }
        l += psum;
    };
    auto add = [&](u32x4 (&f)[2][NDB], const u32x4 (&pf)[2], int t0, bool masked) {
        if (!INT8 && masked) {
            uint32_t odd = 0;
#pragma unroll
            for (int k = 0; k < 2; ++k)
#pragma unroll
                for (int d = 0; d < NDB; ++d) odd |= odd_bits<BF>(f[k][d]);
            if (__builtin_amdgcn_ballot_w64(odd != 0)) {
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const u32x4 big = seen_big(t0 + k * 16 + half * 8, lo, hi);
#pragma unroll
                    for (int d = 0; d < NDB; ++d) {
                        u32x4 a = f[k][d], up, down;
                        take_odd<BF>(a, up, down);
                        // in place, by hand, as the rescaling above, with the waits around both (18 states from a product's issue to a read of its result)
                        asm volatile("s_nop 15\n\ts_nop 7\n\tv_mfma_f32_32x32x16_bf16 %0, %1, %3, %0\n\ts_nop 15\n\ts_nop 7\n\tv_mfma_f32_32x32x16_bf16 %0, %2, %3, %0\n\ts_nop 15\n\ts_nop 7"
                                     : "+v"(o[d]) : "v"(up), "v"(down), "v"(big));
#pragma unroll
                        for (int w = 0; w < 4; ++w) asm volatile("v_mov_b32 %0, %1" : "+v"(f[k][d][w]) : "v"(a[w]));
                    }
                }
            }
        }
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int d = 0; d < NDB; ++d) o[d] = mfma32<BF>(f[k][d], pf[k], o[d]);
    };
    auto step = [&](const char* st, int t0) {
        if (t0 >= whi || t0 + 64 <= wlo) return;
        const bool masked = t0 < ilo || t0 + 64 > ihi;
        u32x4 kf0[KS], kf1[KS], vf[2][NDB], pf[2];
        f32x16 s;
        read_keys(st, 0, kf0);
        scores(kf0, s);
        read_keys(st, 1, kf1);
        read_values(st, 0, vf);
        asm volatile("" ::: "memory");
        weigh(s, st, 0, t0, pf, masked);
        scores(kf1, s);
        add(vf, pf, t0, masked);
        read_values(st, 1, vf);
        asm volatile("" ::: "memory");
        weigh(s, st, 1, t0 + 32, pf, masked);
        add(vf, pf, t0 + 32, masked);
    };
    if constexpr (!INT8) {
        constexpr int NS = ST::N;
        if (!early) for (int i = 0; i < min(NS - 1, s1 - s0); ++i) issue(s0 + i, i);
        int buf = 0;
        for (int st = s0; st < s1; ++st) {
            if (st + 1 < s1) wait_vm<2 * JK * (NS - 2)>(); else wait_vm<0>();        // this step's loads of this wave (the next step's may be left)
            __builtin_amdgcn_s_barrier();           // everyone's; and everyone is done with the stage before
            asm volatile("" ::: "memory");
            if (st + NS - 1 < s1) issue(st + NS - 1, buf == 0 ? NS - 1 : buf - 1);
            step(ch_sm + buf * ST::BYTES, klo + st * 64);
            buf = buf == NS - 1 ? 0 : buf + 1;
        }
        if (early && s0 == s1) wait_vm<0>();        // nothing is seen: what was asked for early must not land in LDS that is another block's by then
    } else if (s0 < s1) {
        fetch8(s0);
        store8(0);
        if (s0 + 1 < s1) fetch8(s0 + 1);
        int buf = 0;
        for (int st = s0; st < s1; ++st) {
            __syncthreads();                        // this stage is whole, and everyone is done with the other one
            if (st + 1 < s1) { store8(buf ^ 1); if (st + 2 < s1) fetch8(st + 2); }
            step(ch_sm + buf * ST::BYTES, klo + st * 64);
            buf ^= 1;
        }
    }
    l = xor32_sum(l);
    if (!ok) return;
    const size_t at = (size_t)kh * p.rows * p.G + (size_t)base * p.G + cc;           // the column among all of its kv head
    if (p.parts > 1) {
        const size_t slot = (size_t)part * p.nkv * p.rows * p.G + at;
#pragma unroll
        for (int d = 0; d < NDB; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                f32x4 v = {o[d][i * 4], o[d][i * 4 + 1], o[d][i * 4 + 2], o[d][i * 4 + 3]};
                if constexpr (VS != 1.f) v *= 1.f / VS;
                *reinterpret_cast<f32x4*>(p.tmp_out + slot * HD + d * 32 + i * 8 + half * 4) = v;
            }
        if (half == 0) p.tmp_ml[slot] = make_float4(m, l, __builtin_bit_cast(float, ref), 0.f);
        return;
    }
    const float inv = scored_inv(l, seen) * (1.f / VS);
    uint16_t* out = reinterpret_cast<uint16_t*>(p.out) + ((size_t)row * p.nh + h) * HD + half * 4;
#pragma unroll
    for (int d = 0; d < NDB; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            u32x2 v = {0u, 0u};
            if (seen) { v[0] = act_pack<BF>(o[d][i * 4] * inv, o[d][i * 4 + 1] * inv); v[1] = act_pack<BF>(o[d][i * 4 + 2] * inv, o[d][i * 4 + 3] * inv); }
            *reinterpret_cast<u32x2*>(out + d * 32 + i * 8) = v;
        }
    if (half == 0) {
        if (p.lse) p.lse[(size_t)row * p.nh + h] = scored_lse(m, l, seen, seen ? scored_shift(p, row, h, ref) : 0.f);
        if (p.cols) p.cols[at] = Col{m, scored_inv(l, seen), slope2, ref, seen ? lo : 0, seen ? hi : 0, 0, 0};
    }
}

// Parts of the keys into results: 16 bytes a thread, HD / 4 threads a column, eight parts in flight.
template <int HD, bool BF>
__global__ __launch_bounds__(256) void scored_parts_kernel(const ChunkParams p) {
    constexpr int TP = HD / 4;
    const int d0 = threadIdx.x % TP * 4;
    const size_t cols = (size_t)p.rows * p.G, all = cols * p.nkv, at = (size_t)blockIdx.x * (256 / TP) + threadIdx.x / TP;
    if (at >= all) return;
    float m = NEG_BIG, l = 0.f;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    int ref = 0;
    for (int i0 = 0; i0 < p.parts; i0 += 8) {
        float4 ml[8];
        f32x4 v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const size_t slot = min(i0 + i, p.parts - 1) * all + at;
            ml[i] = p.tmp_ml[slot];
            v[i] = *reinterpret_cast<const f32x4*>(p.tmp_out + slot * HD + d0);
        }
        ref = __builtin_bit_cast(int, ml[0].z);
        float mn = m;
#pragma unroll
        for (int i = 0; i < 8; ++i) mn = fmaxf(mn, ml[i].x);
        const float f0 = __builtin_amdgcn_exp2f(m - mn);
        l *= f0; acc *= f0; m = mn;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (i0 + i >= p.parts) continue;
            const float f = __builtin_amdgcn_exp2f(ml[i].x - m);
            l += ml[i].y * f;
            acc += v[i] * f;
        }
    }
    const int kh = (int)(at / cols), c = (int)(at - kh * cols), row = c / p.G, h = kh * p.G + c - row * p.G;
    if (p.row_start) {                              // the row's sequence; a row behind the last has no parts
        int lo = 0, hi = p.B;
        while (lo < hi) { const int mid = (lo + hi) >> 1; if (p.row_start[mid + 1] > row) hi = mid; else lo = mid + 1; }
        if (lo >= p.B) return;
        int base, len;
        scored_rows_of(p, lo, base, len);
        if (row < base || row >= base + len) return;
    }
    int a, e;
    scored_interval(p, row, a, e);
    const bool seen = e > a;
    scored_store<BF>(p, row, h, HD, d0, acc, m, l, seen, ref);
    if (p.cols && d0 == 0) p.cols[at] = Col{m, scored_inv(l, seen), p.slopes ? p.slopes[h] * kLog2e : 0.f, ref, a, e, 0, 0};
}

// The weights of many rows: S^T once more, a wave's 64 keys in registers, the columns streaming by, and every column's maximum and sum known.  A block takes 256 keys, its 8 waves the two halves of
// 128 columns at a time (three stages of DMA); a probability is added in the lane of its column, lanes and halves meet once at the end: no atomics, the same sums every time.  A block's
// columns are those of the rows between the first and the last that see some of its keys; tiles that most rows see come first; where blocks are few the columns are dealt to `splits` blocks
// and scored_decay_kernel adds their shares.  2 x 2048 rows of 28 heads behind 2048 slots: 163 us, 0.55 PFLOP/s of products; compute units are busy for 85% of it, vector
// instructions, the exponentials first, take 53% of that time and products 30%.  (Products of the next 32 columns laid among the exponentials of the last ones: 181 us against 170 then, the
// registers' copies took more.)
template <int HD, bool INT8, bool BF, int FORM>
__global__ __launch_bounds__(512, 2) void scored_sums_kernel(const ChunkParams p, int splits) {
    constexpr int KS = HD / 16, ROW = HD * 2, CK = ROW / 16, QB = 128 * ROW, SB = QB + 4096, LOADS = QB / 1024, JL = LOADS / 8, NS = 3;
    extern __shared__ __attribute__((aligned(16))) char su_sm[];
    float* meet = reinterpret_cast<float*>(su_sm);                   // [256], over the columns when they are done
    int* s_reach = reinterpret_cast<int*>(su_sm + NS * SB);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), col = lane & 31, half = lane >> 5, cg = wave >> 2;
    int id = blockIdx.x;
    const int kh = id % p.nkv; id /= p.nkv;
    const int b = id % p.B; id /= p.B;
    const int split = id % splits, tile = id / splits;               // early keys, which most rows see, first
    int base, len;
    scored_rows_of(p, b, base, len);
    const int ncol = len * p.G, tw = tile * 256 + (wave & 3) * 64;    // the wave's first slot
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)su_sm;
    const char* cols = reinterpret_cast<const char*>(p.cols + (size_t)kh * p.rows * p.G + (size_t)base * p.G);
    auto issue = [&](int st, int buf) {
#pragma unroll
        for (int j = 0; j < JL; ++j) {
            const int d = j * 8 + wave, cl = d * (1024 / ROW) + lane / CK, c = min(st * 128 + cl, ncol - 1);
            const int r = p.G == 1 ? c : (int)(((unsigned long long)(unsigned)c * p.g_magic) >> 32);
            dma16(__builtin_amdgcn_readfirstlane(lds0 + buf * SB + d * 1024), (const uint16_t*)p.q + (size_t)(base + r) * p.ldq + (kh * p.G + c - r * p.G) * HD + ((lane % CK) ^ (cl & (CK - 1))) * 8);
        }
        if (wave < 4)                                                // 32 columns' facts a load (the last, past the sequence's, are its last one's: not looked at)
            dma16(__builtin_amdgcn_readfirstlane(lds0 + buf * SB + QB + wave * 1024), cols + (size_t)min(st * 128 + wave * 32 + (lane >> 1), ncol - 1) * 32 + (lane & 1) * 16);
    };
    // the last slot that any row sees, and the rows [r0, r1) between which all lie that see some of the tile: their columns are the block's
    if (tid == 0) { s_reach[0] = 0; s_reach[1] = 0x7fffffff; s_reach[2] = 0; }
    int reach = 0, r0 = 0x7fffffff, r1 = 0;
    for (int i0 = tid; i0 < len; i0 += 4 * 512) {
        int a[4], e[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) scored_interval(p, base + min(i0 + j * 512, len - 1), a[j], e[j]);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int i = min(i0 + j * 512, len - 1);
            reach = max(reach, e[j]);
            if (e[j] > tile * 256 && a[j] < tile * 256 + 256) { r0 = min(r0, i); r1 = max(r1, i + 1); }
        }
    }
    // the wave's keys, on their way during the reductions
    const int32_t* bt = p.block_table + (size_t)b * p.max_blocks;
    u32x4 kfr[2][KS];
    float ksc[INT8 ? 2 : 1][INT8 ? 16 : 1];
    i32x4 kp[FORM == FORM_BIAS ? 2 : 1][FORM == FORM_BIAS ? 4 : 1];
#pragma unroll
    for (int g = 0; g < 2; ++g) {
        const int t = min(tw + g * 32 + col, p.max_seq - 1), blk = scored_block(p, bt, t);
        const size_t at = (((size_t)blk * 2) * p.nkv + kh) * p.page + t % p.page;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            if constexpr (INT8) {
                const u32x2 v = *reinterpret_cast<const u32x2*>((const char*)p.kv_base + at * HD + s * 16 + half * 8);
                kfr[g][s] = widen_codes<BF>(v[0], v[1]);
            } else kfr[g][s] = *reinterpret_cast<const u32x4*>((const uint16_t*)p.kv_base + at * HD + s * 16 + half * 8);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {                                // the lane's results are keys 8 i + 4 half + r
            const int tt = tw + g * 32 + i * 8 + half * 4, tc = min(tt, (p.max_seq - 1) & ~3), bl = scored_block(p, bt, tc);
            if constexpr (INT8) {
                const f32x4 v = *reinterpret_cast<const f32x4*>(p.scale_base + (((size_t)bl * 2) * p.nkv + kh) * p.page + tc % p.page);
#pragma unroll
                for (int e = 0; e < 4; ++e) ksc[INT8 ? g : 0][INT8 ? i * 4 + e : 0] = v[e];
            }
            if constexpr (FORM == FORM_BIAS) {
                kp[g][i] = i32x4{tt, tt + 1, tt + 2, tt + 3};
                if (p.key_pos) kp[g][i] = *reinterpret_cast<const i32x4*>(p.key_pos + ((size_t)bl * p.nkv + kh) * p.page + tc % p.page);
            }
        }
    }
    const auto larger = [](int a, int c) { return max(a, c); };
    reach = row32(reach, larger); r1 = row32(r1, larger); r0 = row32(r0, [](int a, int c) { return min(a, c); });
    lds_barrier();
    if ((lane & 31) == 0) { atomicMax(&s_reach[0], reach); atomicMin(&s_reach[1], r0); atomicMax(&s_reach[2], r1); }
    lds_barrier();
    reach = __builtin_amdgcn_readfirstlane(s_reach[0]); r0 = __builtin_amdgcn_readfirstlane(s_reach[1]); r1 = __builtin_amdgcn_readfirstlane(s_reach[2]);
    if (splits > 1 && tile == 0 && kh == 0 && split == 0 && tid == 0) p.reach[b] = reach;
    if (tile * 256 >= reach) return;
    const int first = r1 > 0 ? r0 * p.G / 128 : 0, all = r1 > 0 ? (r1 * p.G + 127) / 128 - first : 0;
    const int st0 = first + (int)((long)all * split / splits), st1 = first + (int)((long)all * (split + 1) / splits);
    if (st0 < st1) issue(st0, 0);
    if (st0 + 1 < st1) issue(st0 + 1, 1);
    float acc[2][16];
#pragma unroll
    for (int g = 0; g < 2; ++g)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[g][i] = 0.f;
    int buf = 0;
    const int f = col & (CK - 1);
    wait_vm<0>();                                                    // the keys are here: no wait for them inside the loop
    for (int st = st0; st < st1; ++st) {
        if (st + 1 < st1) { if (wave < 4) wait_vm<JL + 1>(); else wait_vm<JL>(); } else wait_vm<0>();      // all but the next step's loads of this wave
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        if (st + 2 < st1) issue(st + 2, buf == 0 ? 2 : buf - 1);
        const char* stage = su_sm + buf * SB;
        buf = buf == 2 ? 0 : buf + 1;
#pragma unroll
        for (int ct = 0; ct < 2; ++ct) {
            const int cl = cg * 64 + ct * 32 + col;
            Col c = reinterpret_cast<const Col*>(stage + QB)[cl];
            if (st * 128 + cl >= ncol) c.lo = c.hi = 0;
            if (!__builtin_amdgcn_ballot_w64(c.lo < tw + 64 && c.hi > tw)) continue;
            if (__builtin_amdgcn_ballot_w64(c.inv != c.inv)) {       // a column that is not a number: so are the slots it sees, and no others
                const bool odd = c.inv != c.inv;
                const int a = odd ? c.lo - tw - half * 4 : 0, e = odd ? c.hi - tw - half * 4 : 0;
#pragma unroll
                for (int i = 0; i < 32; ++i) {                       // in place, so that the sums are not kept twice
                    const int t = (i >> 4) * 32 + (i >> 2 & 3) * 8 + (i & 3);
                    asm volatile("v_add_f32 %0, %0, %1" : "+v"(acc[i >> 4][i & 15]) : "v"(t >= a && t < e ? c.inv : 0.f));
                }
                if (odd) { c.lo = c.hi = 0; c.inv = 0.f; }
            }
            const bool masked = __builtin_amdgcn_ballot_w64(c.lo > tw || c.hi < tw + 64) != 0;
            f32x16 s[2];
#pragma unroll
            for (int i = 0; i < 16; ++i) s[0][i] = s[1][i] = 0.f;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                const u32x4 q = *reinterpret_cast<const u32x4*>(stage + cl * ROW + (((ks * 2 + half) ^ f) << 4));
                s[0] = mfma32<BF>(kfr[0][ks], q, s[0]);
                s[1] = mfma32<BF>(kfr[1][ks], q, s[1]);
            }
            c.m = fmaxf(c.m, NEG_BIG);
#pragma unroll
            for (int g = 0; g < 2; ++g) {
                float sv[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) sv[i] = INT8 ? s[g][i] * ksc[INT8 ? g : 0][INT8 ? i : 0] : s[g][i];
                float mul = p.scale1;
                if constexpr (FORM != FORM_PLAIN) {
                    if (FORM == FORM_CAP || p.capped) {
#pragma unroll
                        for (int i = 0; i < 16; ++i) sv[i] *= p.scale1;
                        tanh_all(sv);
                        mul = p.cap_log2;
                    }
                }
                if constexpr (FORM == FORM_BIAS) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) sv[i] = __builtin_fmaf(c.slope2, (float)(kp[g][i >> 2][i & 3] - c.ref), sv[i] * mul);
                    mul = 1.f;
                }
                if (masked) {                                        // a column that sees nothing: exp(-inf) = 0 of each
                    const int a = c.lo - tw - g * 32 - half * 4, e = c.hi - tw - g * 32 - half * 4;
#pragma unroll
                    for (int i = 0; i < 16; ++i) sv[i] = (i >> 2) * 8 + (i & 3) >= a && (i >> 2) * 8 + (i & 3) < e ? sv[i] : -__builtin_inff();
                }
#pragma unroll
                for (int i = 0; i < 16; ++i) acc[g][i] = __builtin_fmaf(__builtin_amdgcn_exp2f(__builtin_fmaf(sv[i], mul, -c.m)), c.inv, acc[g][i]);
            }
        }
    }
    float sums[32];                                                  // over the 32 lanes: lane `col` ends up with result `col`, 16 of each group; at every step half the results go over
#pragma unroll
    for (int i = 0; i < 32; ++i) sums[i] = acc[i >> 4][i & 15];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
#pragma unroll
        for (int i = 0; i < o; ++i) {
            float a = sums[i], e = sums[i + o];
            asm("" : "+v"(a), "+v"(e));                              // two registers, not an index that a lane looks up
            const float keep = col & o ? e : a, give = col & o ? a : e;
            sums[i] = keep + __shfl_xor(give, o);
        }
    float sum = sums[0];
    __syncthreads();
    const int key = (wave & 3) * 64 + (col >> 4) * 32 + (col >> 2 & 3) * 8 + half * 4 + (col & 3);
    if (cg > 0) meet[key] = sum;
    __syncthreads();
    if (cg > 0) return;
    sum += meet[key];
    const int t = tile * 256 + key;
    if (t >= reach) return;
    if (splits > 1) {
        p.shares[(((size_t)split * p.B + b) * p.nkv + kh) * p.max_seq + t] = sum;
        return;
    }
    const int blk = bt[(int)(((unsigned long long)(unsigned)t * p.page_magic) >> 32)];
    if (blk < 0 || blk >= p.num_blocks) return;
    float* to = p.weights + ((size_t)blk * p.nkv + kh) * p.page + t % p.page;
    *to = scored_decayed(p, *to, sum);
}

__global__ __launch_bounds__(256) void scored_decay_kernel(const ChunkParams p, int splits) {
    const int b = blockIdx.z, kh = blockIdx.y, t = blockIdx.x * 256 + threadIdx.x;
    if (t >= p.reach[b]) return;
    float sum = 0.f;
    for (int i = 0; i < splits; ++i) sum += p.shares[(((size_t)i * p.B + b) * p.nkv + kh) * p.max_seq + t];
    const int blk = p.block_table[(size_t)b * p.max_blocks + (int)(((unsigned long long)(unsigned)t * p.page_magic) >> 32)];
    if (blk < 0 || blk >= p.num_blocks) return;
    float* to = p.weights + ((size_t)blk * p.nkv + kh) * p.page + t % p.page;
    *to = scored_decayed(p, *to, sum);
}

// ================================================================================================ plans
// How a call runs, and its workspace's regions, each on 256 bytes.
struct Plan {
    bool   few;                // the few-row kernel: at most 32 (row, head) pairs of a key/value head a sequence
    int    nblocks, ncol, ctx_pad, runs;
    int    waves, tiles, parts, splits;                          // the many-row kernels
    size_t tmp_out, tmp_ml, ml_all, spill, meta, bytes;          // offsets; bytes: all
};
constexpr long GRID_THREADS = 1l << 32;   // a launch's threads along x are 32 bits
constexpr int RUNS = 256;      // one block of the few-row kernel a compute unit
Plan plan_of(int B, int q_len, int rows, int nh, int nkv, int hd, int max_seq, bool track, bool int8) {
    Plan pl{};
    const int G = nh / nkv;
    size_t at = 0;
    auto region = [&](size_t bytes) { const size_t r = at; at += (bytes + 255) & ~(size_t)255; return r; };
    pl.few = (long)q_len * G <= 32;
    if (pl.few) {
        const long pairs = (long)B * nkv;
        // Runs take the time of the mean length where a block per pair takes that of the longest, and pay for parts and their merge.  us by pairs / by runs, 28 over 4 heads of 128, 256 pairs: lengths
        // spread evenly up to 1000 18.7 / 26.2, all of 500 17.7 / 18.5, one of 8000 among 500s 73.8 / 23.0; 1024 pairs: 71.4 / 81.2, 65.9 / 64.4, 106 / 59; 2048: 127 / 147, 123 / 121, 166 / 135.
        // From 1024 pairs on, four blocks a compute unit, they even out by themselves well enough.
        pl.runs = pairs < 4 * RUNS;
        pl.nblocks = pl.runs ? RUNS : (int)pairs;
        pl.ncol = q_len * G; pl.ctx_pad = (max_seq + 63) / 32 * 32 + 32;
        pl.meta = region(pairs * sizeof(int4));
        if (pl.runs) { pl.tmp_out = region((size_t)2 * RUNS * pl.ncol * hd * 4); pl.tmp_ml = region((size_t)2 * RUNS * pl.ncol * 8); }
        if (track) { pl.ml_all = region(pairs * pl.ncol * 8); pl.spill = region(pairs * pl.ncol * pl.ctx_pad * 4); }
    } else {
        const long cols = (long)q_len * G;
        // Four waves a block, two blocks a compute unit: one fills in while the other one starts, ends or waits.  us by eight / by four: 16 x 64 rows 13.0 / 10.5, 4 x 512 29 / 25, 32 x 512
        // 157 / 144, 8 x 512 and 2 x 2048 behind 2048 the same.  Eight, which fetch keys and values half as often, where walks are long (4096 rows behind 12288 slots 895 / 913) and
        // where keys and values are widened on the way (333 rows behind 3001 47 / 60).  Two a block are no form: at 35 to 64 columns behind 1000 to 12000 slots they took 1.01 to 1.27 of four's time,
        // 1.01 to 1.6 over 8 bits, where they spilled most.  Up to 128 columns, where eight would leave half a block idle, four / eight of 35 to 126 columns: 16 bits 13.4 to 32.0 / 13.3 to 29.2 (heads
        // of 128, eight ahead behind 12000 slots and for 32 over 8 heads), 11.0 to 21.1 / 11.3 to 21.5 (64); 8 bits 19.8 to 40.2 / 18.6 to 43.6 (128, eight ahead but for 8 kv heads), 15.7 to 25.1 / 16.0 to 25.4 (64).
        pl.waves = cols <= 128 || (!int8 && max_seq < 8192) ? 4 : 8;
        pl.tiles = (int)((cols + 32 * pl.waves - 1) / (32 * pl.waves));
        const long blocks = (long)pl.tiles * B * nkv, room = 256 * 8 / pl.waves;
        // Parts of at least 256 keys, 64 at most: us by 128 / 256 / 512 keys, 40 rows of 28 over 4 heads behind 1000 slots 15.4 / 16.2 / 18.4, behind 3001 22.5 / 19.0 / 21.9, of 8 over 1 15.1 / 16.3 / 20.9,
        // over 8 bits behind 3001 25.9 / 26.7 / 35.5; by at most 16 / 32 / 64 / 128, 40 rows of 8 over 1 behind 32000 73 / 47 / 39 / 40.
        pl.parts = (int)std::max(1l, std::min({room / std::max(1l, blocks), (max_seq + 255l) / 256, 64l}));
        if (pl.parts > 1) { pl.tmp_out = region((size_t)pl.parts * rows * nh * hd * 4); pl.tmp_ml = region((size_t)pl.parts * rows * nh * 16); }
        if (track) {
            pl.ml_all = region((size_t)rows * nh * sizeof(Col));
            const long kb = (long)cdiv(max_seq, 256) * nkv * B;
            pl.splits = (int)std::max(1l, std::min({1024 / kb, (cols + 1023) / 1024, 8l}));     // at least 8 steps each; us for 2 x 2048 rows behind 2048 by 2 / 4 / 8: 175 / 179 / 169, at best 159 / 165 / 155
            if (pl.splits > 1) pl.spill = region(((size_t)pl.splits * nkv * max_seq + 1) * B * 4);
        }
    }
    pl.bytes = at;
    return pl;
}

template <int HD, bool INT8, int NT, bool BF>
int launch_decode(const DecodeParams& d, hipStream_t st) {
    auto run = [&](auto kernel, int lds) -> int {
        const int rc = raise_dynamic_lds((const void*)kernel, "paged_attn_scored");
        if (rc == MI355_OK) hipLaunchKernelGGL(kernel, dim3(d.nblocks), dim3(64 * Ring<HD, INT8, NT, true>::NW), lds, st, d);
        return rc;
    };
    return d.key_pos ? run(scored_decode_kernel<HD, INT8, NT, BF, true>, Ring<HD, INT8, NT, true>::BYTES) : run(scored_decode_kernel<HD, INT8, NT, BF, false>, Ring<HD, INT8, NT, INT8>::BYTES);
}

template <int HD, bool INT8, bool BF, int FORM>
int launch_chunk(const ChunkParams& c, const Plan& pl, hipStream_t st) {
    auto run = [&](auto kernel, int lds, int threads, long blocks, auto... more) -> int {
        const int rc = raise_dynamic_lds((const void*)kernel, "paged_attn_scored");
        if (rc == MI355_OK) hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(threads), lds, st, c, more...);
        return rc;
    };
    const long blocks = (long)pl.tiles * c.B * c.nkv * pl.parts;
    int rc = pl.waves == 4 ? run(scored_chunk_kernel<HD, INT8, BF, FORM, 4>, Stage<HD, INT8, 4>::LDS, 256, blocks)
                           : run(scored_chunk_kernel<HD, INT8, BF, FORM, 8>, Stage<HD, INT8, 8>::LDS, 512, blocks);
    if (rc != MI355_OK) return rc;
    if (pl.parts > 1) hipLaunchKernelGGL((scored_parts_kernel<HD, BF>), dim3((unsigned)(((long)c.rows * c.nh + 1024 / HD - 1) / (1024 / HD))), dim3(256), 0, st, c);
    if (c.weights) {
        rc = run(scored_sums_kernel<HD, INT8, BF, FORM>, 3 * (128 * HD * 2 + 4096) + 16, 512, (long)cdiv(c.max_seq, 256) * c.nkv * c.B * pl.splits, pl.splits);
        if (rc == MI355_OK && pl.splits > 1) hipLaunchKernelGGL(scored_decay_kernel, dim3(cdiv(c.max_seq, 256), c.nkv, c.B), dim3(256), 0, st, c, pl.splits);
    }
    return rc;
}
template <int HD, bool INT8, bool BF>
int launch_chunk(const ChunkParams& c, const Plan& pl, hipStream_t st) {
    return c.slopes ? launch_chunk<HD, INT8, BF, FORM_BIAS>(c, pl, st) : c.capped ? launch_chunk<HD, INT8, BF, FORM_CAP>(c, pl, st) : launch_chunk<HD, INT8, BF, FORM_PLAIN>(c, pl, st);
}

} // namespace

extern "C" size_t mi355_paged_attn_scored_workspace_bytes(int32_t B, int32_t q_len, int32_t rows, int32_t nh, int32_t nkv, int32_t hd, int32_t max_seq_len, int32_t track) {
    if (B <= 0 || q_len <= 0 || rows <= 0 || nh <= 0 || nkv <= 0 || nh % nkv || hd <= 0 || max_seq_len <= 0) return 0;
    return std::max(plan_of(B, q_len, rows, nh, nkv, hd, max_seq_len, track != 0, false).bytes, plan_of(B, q_len, rows, nh, nkv, hd, max_seq_len, track != 0, true).bytes);
}

extern "C" int mi355_paged_attn_scored(const void* q, int32_t ldq, const mi355_kv_layer_t* kv, const int32_t* block_table, int32_t max_blocks_per_seq,
                                       const int32_t* row_start, int32_t B, int32_t q_len, int32_t rows, int32_t nh, const mi355_attn_score_t* score,
                                       int32_t max_seq_len, void* out, float* lse, float* weights, float decay, void* workspace, size_t workspace_bytes,
                                       mi355_stream_t stream) {
    DecodeParams p;
    const int rc = scored_params(p, q, ldq, kv, block_table, max_blocks_per_seq, row_start, B, q_len, rows, nh, score, max_seq_len, out, lse, weights, decay);
    if (rc != MI355_OK) return rc;
    const Plan pl = plan_of(B, q_len, rows, nh, kv->nkv, kv->hd, max_seq_len, weights != nullptr, kv->kv_dtype == MI355_KV_INT8);
    if (pl.bytes && (pl.bytes > workspace_bytes || !workspace)) {
        mi355_set_error("paged_attn_scored: workspace %zu < %zu", workspace_bytes, pl.bytes);
        return MI355_ERR_WORKSPACE;
    }
    MI355_CHECK_ARG(((uintptr_t)workspace & 15) == 0, "paged_attn_scored: the workspace lies on 16 bytes");
    const bool bf = kv->act_dtype == MI355_ACT_BF16, int8 = kv->kv_dtype == MI355_KV_INT8;
    hipStream_t st = (hipStream_t)stream;
    char* ws = (char*)workspace;
    if (pl.few) {
        const long np = (long)B * kv->nkv;
        MI355_CHECK_ARG(np * (pl.ncol + (long)cdiv(max_seq_len, 256)) < (1l << 31) && (!pl.runs || np * cdiv(max_seq_len, 32) < (1l << 30)) &&
                            pl.nblocks * 512l < GRID_THREADS && ((np * pl.ncol + 3) / 4 + (weights ? np * cdiv(max_seq_len, 1024) : 0)) * 256 < GRID_THREADS,
                        "paged_attn_scored: %d sequences of %d slots and %d heads exceed the grid", B, max_seq_len, nh);
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
        // Four slots a thread, or one where that leaves less than two blocks a compute unit.  us by one / by four, 28 over 4 heads: 2 x 8000 slots (64 blocks of 1024) 17.6 / 18.3, 16 x 4000 (256)
        // 38.3 / 38.9, 32 x 4000 (512) 70.1 / 67.9, 64 x 3000 (768) 102 / 100.
        const int pairs = B * kv->nkv, sl = (long)pairs * cdiv(max_seq_len, 1024) >= 512 ? 4 : 1, chunks = weights ? cdiv(max_seq_len, 256 * sl) : 0;
        // A column a block where a pair has four runs or more, else four: us by four / by one, one row: 8 pairs of 6000 slots 16.6 / 15.6, 16 19.1 / 18.6, 64 of 1000 14.4 / 14.3, 256 31.5 / 32.2; four
        // rows of 1000 slots, whose 28 columns a pair fill the chip sooner: 8 13.3 / 13.1, 32 16.5 / 17.6, 128 25.0 / 27.9.
        const bool wide = pairs < 64;
        const int joins = wide ? pairs * pl.ncol : cdiv(pairs * pl.ncol, 4);
        const dim3 grid(joins + pairs * chunks);
#define LK_(HD_, BF_, SL_) do { if (wide) hipLaunchKernelGGL((scored_join_kernel<HD_, BF_, SL_, 1>), grid, dim3(256), 0, st, p, joins, chunks); \
                                else      hipLaunchKernelGGL((scored_join_kernel<HD_, BF_, SL_, 4>), grid, dim3(256), 0, st, p, joins, chunks); } while (0)
#define LJ_(HD_, BF_) do { if (sl == 4) LK_(HD_, BF_, 4); else LK_(HD_, BF_, 1); } while (0)
        if (kv->hd == 128) { if (bf) LJ_(128, true); else LJ_(128, false); } else { if (bf) LJ_(64, true); else LJ_(64, false); }
#undef LJ_
#undef LK_
        MI355_CHECK_LAUNCH("scored_join_kernel");
        return MI355_OK;
    }
    ChunkParams c;
    static_cast<ScoredParams&>(c) = p;
    c.tiles = pl.tiles; c.parts = pl.parts; c.g_magic = (uint32_t)((1ull << 32) / (unsigned)p.G + 1);
    c.tmp_out = pl.parts > 1 ? (float*)(ws + pl.tmp_out) : nullptr; c.tmp_ml = pl.parts > 1 ? (float4*)(ws + pl.tmp_ml) : nullptr;
    c.cols = weights ? (Col*)(ws + pl.ml_all) : nullptr; c.shares = weights && pl.splits > 1 ? (float*)(ws + pl.spill) : nullptr;
    c.reach = c.shares ? (int*)(c.shares + (size_t)pl.splits * B * kv->nkv * max_seq_len) : nullptr;
    MI355_CHECK_ARG((long)pl.tiles * B * kv->nkv * pl.parts * 64 * pl.waves < GRID_THREADS && (!weights || (long)cdiv(max_seq_len, 256) * kv->nkv * B * pl.splits * 512 < GRID_THREADS) && (long)q_len * p.G * p.G < (1l << 32),
                    "paged_attn_scored: %d rows of %d heads in %d sequences of %d slots exceed the grid", rows, nh, B, max_seq_len);
    int crc;
#define LB_(HD_) do { if (bf) crc = int8 ? launch_chunk<HD_, true, true>(c, pl, st) : launch_chunk<HD_, false, true>(c, pl, st); \
                      else    crc = int8 ? launch_chunk<HD_, true, false>(c, pl, st) : launch_chunk<HD_, false, false>(c, pl, st); } while (0)
    if (kv->hd == 128) LB_(128); else LB_(64);
#undef LB_
    if (crc != MI355_OK) return crc;
    MI355_CHECK_LAUNCH("scored_chunk_kernel");
    return MI355_OK;
}
