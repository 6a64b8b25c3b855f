// A paged cache brought back to its budget by accumulated attention weight, gfx950.
//
// Every (sequence, kv head) with n > keep tokens keeps the `keep` of the largest rank.  A token's rank is a 32-bit number: protected ones (position < sinks or >= next_pos - recent) all
// ones, others their weight's bits in an order that compares as unsigned, 0 for NaN and for tokens in blocks outside the pool; equal ranks go to the lower slot.
// Kept tokens below slot `keep` stay; the i-th kept one behind moves into the i-th hole below.  Sources and holes are disjoint, so no order between moves is needed and nothing else is
// touched: the least that can be moved (a stable compaction would move every token behind the first hole).  The order of slots is lost, which is why positions are kept beside them.
//
// Two launches: the plan (a block per sequence and head) and the moves (as many blocks as there is room for).
#include <algorithm>

#include "common.h"
#include "internal.h"

namespace {

struct EvictParams {
    void*          kv_base;
    float*         scale_base;
    float*         weights;
    int32_t*       key_pos;
    const int32_t* block_table;
    const int32_t* seq_lens;
    const int32_t* next_pos;
    int32_t*       new_lens;
    int32_t*       count;    // [B][nkv] moves
    int32_t*       lists;    // [B][nkv][2][cap]: sources, holes
    int32_t*       first;    // [B][nkv][units + 1]: holes before each 64 slots below keep
    int max_blocks, num_blocks, nkv, page, max_seq, keep, sinks, recent, cap, units;
    uint32_t page_magic;     // 2^32 / page + 1: floor(t / page) = (t magic) >> 32 for t page < 2^32
    __device__ __forceinline__ int page_of(int t) const { return (int)(((unsigned long long)(unsigned)t * page_magic) >> 32); }
};

// LDS of a plan's block, in words: a histogram per pass (copies of it, eight of the first: weights crowd into few exponents), the candidates of the last digit, sums of the waves; behind them the ranks.
constexpr int EV_THREADS = 1024, EV_WAVES = EV_THREADS / 64, EV_COPIES = 4, EV_HIST = 256 * EV_COPIES, EV_CAND = 128, EV_KEYS = 32768, EV_FIXED = 5 * EV_HIST + 2 * EV_CAND + 4 + EV_WAVES;
static_assert((EV_KEYS + EV_FIXED) * 4 <= 160 * 1024, "LDS of a block");

__device__ __forceinline__ uint32_t evict_rank(const EvictParams& p, float w, int pos, int newest) {
    w += 0.f;                                                 // -0 as 0
    if (pos < p.sinks || pos >= newest) return 0xFFFFFFFFu;
    if (w != w) return 0u;
    const uint32_t u = __builtin_bit_cast(uint32_t, w);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ uint32_t evict_rank(const EvictParams& p, int b, int kh, int t, int newest) {
    const int pg = p.page_of(t), blk = p.block_table[(size_t)b * p.max_blocks + pg];
    if (blk < 0 || blk >= p.num_blocks) return 0u;
    const size_t at = ((size_t)blk * p.nkv + kh) * p.page + t - pg * p.page;
    return evict_rank(p, p.weights[at], p.key_pos[at], newest);
}

// IN_LDS: the ranks of the longest sequence that the call allows fit there; else they are formed again by every pass.  Both launches, us by LDS / by passes: 2304 tokens cut to 2048 20.3 / 24.1, 64 x
// 4096 cut to 1024 65.6 / 72.9.
template <bool IN_LDS>
__global__ __launch_bounds__(EV_THREADS) void evict_plan_kernel(const EvictParams p) {
    extern __shared__ __attribute__((aligned(16))) uint32_t ev_sm[];
    uint32_t *hist = ev_sm, *cand = hist + 5 * EV_HIST, *state = cand + 2 * EV_CAND;   // state: candidates, the last kept one's rank and slot
    int* part = reinterpret_cast<int*>(state + 4);
    uint32_t* ranks = state + 4 + EV_WAVES;
    const int kh = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = min(max(p.seq_lens[b], 0), p.max_seq);
    int32_t* cnt = p.count + (size_t)b * p.nkv + kh;
    if (n <= p.keep) { if (tid == 0) *cnt = 0; return; }
    const int newest = p.next_pos[b] - p.recent;
    auto rank = [&](int t) { return IN_LDS ? ranks[t] : evict_rank(p, b, kh, t, newest); };
    for (int i = tid; i < 5 * EV_HIST; i += EV_THREADS) hist[i] = 0;
    if (tid < 4) state[tid] = 0;
    __syncthreads();
    for (int t0 = tid; t0 < n; t0 += 4 * EV_THREADS) {        // the first pass is formed on the way in; four tokens' loads in flight
        int blk[4], pos[4];
        float w[4];
        size_t at[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int t = min(t0 + i * EV_THREADS, n - 1), pg = p.page_of(t);
            blk[i] = p.block_table[(size_t)b * p.max_blocks + pg];
            at[i] = t - pg * p.page;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            at[i] += ((size_t)min(max(blk[i], 0), p.num_blocks - 1) * p.nkv + kh) * p.page;
            pos[i] = p.key_pos[at[i]]; w[i] = p.weights[at[i]];
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int t = t0 + i * EV_THREADS;
            if (t >= n) continue;
            const uint32_t u = blk[i] < 0 || blk[i] >= p.num_blocks ? 0u : evict_rank(p, w[i], pos[i], newest);
            if (IN_LDS) ranks[t] = u;
            atomicAdd(&hist[(lane & (2 * EV_COPIES - 1)) * 256 + (u >> 24)], 1u);
        }
    }
    __syncthreads();
    // The keep-th largest rank, 8 bits at a time; every wave reads the histogram for itself.  Once the digit's ranks are few they are ordered outright, ties with them: weights differ in
    // their upper 16 bits as a rule.
    uint32_t prefix = 0, left = p.keep, bar = 0;
    int ties = 0, bar_slot = -1;                              // kept: rank > bar, and of those at the bar the slots up to bar_slot, or (-1) the first `ties`
    for (int shift = 24; shift >= 0; shift -= 8) {
        uint32_t* h = hist + (shift == 24 ? 0 : 4 - shift / 8) * EV_HIST;
        if (shift < 24) {
            const uint32_t mask = 0xFFFFFFFFu << (shift + 8);
            for (int t = tid; t < n; t += EV_THREADS) {
                const uint32_t u = rank(t);
                if ((u & mask) == prefix) atomicAdd(&h[(lane & (EV_COPIES - 1)) * 256 + (u >> shift & 255)], 1u);
            }
            __syncthreads();
        }
        u32x4 v = {0u, 0u, 0u, 0u};                           // lane: the digits 255 - 4 lane and the three below
#pragma unroll
        for (int c = 0; c < EV_COPIES; ++c) v += *reinterpret_cast<const u32x4*>(&h[c * 256 + 252 - lane * 4]);
        if (shift == 24) {
#pragma unroll
            for (int c = EV_COPIES; c < 2 * EV_COPIES; ++c) v += *reinterpret_cast<const u32x4*>(&h[c * 256 + 252 - lane * 4]);
        }
        const uint32_t own = v[0] + v[1] + v[2] + v[3];
        uint32_t incl = own;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) { const uint32_t up = __shfl_up(incl, o); if (lane >= o) incl += up; }
        uint32_t before = incl - own, digit = 0, rest = 0, many = 0;
        const uint64_t here = __builtin_amdgcn_ballot_w64(before < left && incl >= left);
#pragma unroll
        for (int i = 3; i >= 0; --i) {
            if (before < left && before + v[i] >= left) { digit = 252 - lane * 4 + i; rest = left - before; many = v[i]; }
            before += v[i];
        }
        const int who = __builtin_ctzll(here);
        prefix |= (uint32_t)__builtin_amdgcn_readlane(digit, who) << shift;
        left = __builtin_amdgcn_readlane(rest, who);
        if (__builtin_amdgcn_readlane(many, who) <= EV_CAND) {
            const uint32_t mask = 0xFFFFFFFFu << shift;
            for (int t = tid; t < n; t += EV_THREADS) {
                const uint32_t u = rank(t);
                if ((u & mask) == prefix) { const uint32_t i = atomicAdd(&state[0], 1u); cand[2 * i] = u; cand[2 * i + 1] = t; }
            }
            __syncthreads();
            const int m = state[0];
            if (tid < m) {
                const uint32_t u = cand[2 * tid], t = cand[2 * tid + 1];
                uint32_t ahead = 0;
                for (int i = 0; i < m; ++i) { const uint32_t x = cand[2 * i], y = cand[2 * i + 1]; ahead += x > u || (x == u && y < t); }
                if (ahead + 1 == left) { state[1] = u; state[2] = t; }
            }
            __syncthreads();
            bar = state[1]; bar_slot = state[2];
            break;
        }
        bar = prefix; ties = (int)left;
    }
    // every wave takes a run of slots; what it starts from is the sum over the waves before
    const int run = (n + EV_WAVES * 64 - 1) / (EV_WAVES * 64) * 64, t0 = wave * run, t1 = min(n, t0 + run);
    auto before_of = [&](int mine) {
        __syncthreads();
        if (lane == 0) part[wave] = mine;
        __syncthreads();
        int s = lane < wave ? part[lane & (EV_WAVES - 1)] : 0;
#pragma unroll
        for (int o = 1; o < EV_WAVES; o <<= 1) s += __shfl_xor(s, o);
        return __builtin_amdgcn_readfirstlane(s);
    };
    int eq0 = 0;
    if (bar_slot < 0) {
        int eq = 0;
        for (int t = t0; t < t1; t += 64) eq += __builtin_popcountll(__builtin_amdgcn_ballot_w64(t + lane < t1 && rank(t + lane) == bar));
        eq0 = before_of(eq);
    }
    const uint64_t below = (1ull << lane) - 1;
    auto walk = [&](auto&& each) {                            // each(slots that become holes, kept ones behind keep) as masks of the wave's lanes
        int e = eq0;
        for (int t = t0; t < t1; t += 64) {
            const uint32_t u = t + lane < t1 ? rank(t + lane) : 0u;
            const bool in = t + lane < t1;
            bool kept = u > bar || (u == bar && t + lane <= bar_slot);
            if (bar_slot < 0) {
                const uint64_t at = __builtin_amdgcn_ballot_w64(in && u == bar);
                kept = u > bar || (u == bar && e + __builtin_popcountll(at & below) < ties);
                e += __builtin_popcountll(at);
            }
            each(t, __builtin_amdgcn_ballot_w64(in && !kept && t + lane < p.keep), __builtin_amdgcn_ballot_w64(in && kept && t + lane >= p.keep));
        }
    };
    int holes = 0, late = 0;
    walk([&](int, uint64_t h, uint64_t l) { holes += __builtin_popcountll(h); late += __builtin_popcountll(l); });
    int hole0 = before_of(holes), late0 = before_of(late);
    int32_t* src = p.lists + ((size_t)b * p.nkv + kh) * 2 * p.cap;
    int32_t* dst = src + p.cap;
    int32_t* first = p.first + ((size_t)b * p.nkv + kh) * (p.units + 1);
    if (wave == EV_WAVES - 1 && lane == 0) { *cnt = hole0 + holes; first[p.units] = hole0 + holes; }
    walk([&](int t, uint64_t h, uint64_t l) {
        if (lane == 0 && t < p.keep) first[t >> 6] = hole0;
        if (h >> lane & 1) dst[hole0 + __builtin_popcountll(h & below)] = t + lane;
        if (l >> lane & 1) src[late0 + __builtin_popcountll(l & below)] = t + lane;
        hole0 += __builtin_popcountll(h); late0 += __builtin_popcountll(l);
    });
}

// A block per 64 slots below keep (a block per 16 has the same chain of five dependent reads for a quarter of the bytes).  Keys move by 16 bytes; a value's window of 8 slots is gathered and
// written whole, 16 bytes a thread: by the element, a hole's 2 bytes in each of 128 channels are partial writes of the memory's sectors.  Slots behind keep in the last window get back
// what they hold, which no move changes.  64 sequences of up to 4096 tokens cut to 1024 (4 heads of 128, 16 bits): 76 us for 123 MB read and 105 written, 3.0 TB/s, where 150 MB are tokens'
// own.  Almost all of it are the values (keys alone 11 us), and not the gather's addresses: source windows whole, through LDS, take 77.  By the element both ways 84, by windows with
// conditional loads 86.  Both launches, all 64 of 4096 tokens: 66 us, in 8 bits 47.
constexpr int EV_UNIT = 64;
template <int HD, int ES>
__global__ __launch_bounds__(256) void evict_move_kernel(const EvictParams p) {
    __shared__ int s_at[EV_UNIT][4];                           // of a slot: where its token comes from (block, token), which is itself where there is no hole, and the slot's own place
    __shared__ uint32_t s_hole[EV_UNIT / 32];
    const int unit = blockIdx.x, kh = blockIdx.y, b = blockIdx.z, tid = threadIdx.x;
    if (unit == 0 && kh == 0 && tid == 0 && p.new_lens) p.new_lens[b] = min(min(max(p.seq_lens[b], 0), p.max_seq), p.keep);
    const size_t pair = (size_t)b * p.nkv + kh;
    const int32_t* first = p.first + pair * (p.units + 1) + unit;
    const int all = p.count[pair], m0 = first[0], n = first[1] - m0;
    if (all == 0 || n == 0) return;                            // the plan writes `first` only where there are moves
    const int32_t *src = p.lists + pair * 2 * p.cap + m0, *dst = src + p.cap;
    const int32_t* bt = p.block_table + (size_t)b * p.max_blocks;
    if (tid < EV_UNIT) {
        const int t = unit * EV_UNIT + tid, pg = min(p.page_of(t), p.max_blocks - 1), blk = min(max(bt[pg], 0), p.num_blocks - 1), o = min(t - pg * p.page, p.page - 1);
        s_at[tid][0] = s_at[tid][2] = blk; s_at[tid][1] = s_at[tid][3] = o;
        if (tid < EV_UNIT / 32) s_hole[tid] = 0;
    }
    __syncthreads();
    if (tid < n) {
        const int ts = src[tid], td = dst[tid], ps = p.page_of(ts), pd = p.page_of(td), bs = bt[ps], bd = bt[pd];
        const int os = ts - ps * p.page, od = td - pd * p.page;
        if (bs >= 0 && bs < p.num_blocks && bd >= 0 && bd < p.num_blocks) {
            const int at = td & (EV_UNIT - 1);
            s_at[at][0] = bs; s_at[at][1] = os;
            atomicOr(&s_hole[at >> 5], 1u << (at & 31));
            const size_t ws = ((size_t)bs * p.nkv + kh) * p.page + os, wd = ((size_t)bd * p.nkv + kh) * p.page + od;
            p.weights[wd] = p.weights[ws];
            p.key_pos[wd] = p.key_pos[ws];
            if (ES == 1)                                       // scale plane [block][K, V][nkv][page]
                for (int kv = 0; kv < 2; ++kv)
                    p.scale_base[(((size_t)bd * 2 + kv) * p.nkv + kh) * p.page + od] = p.scale_base[(((size_t)bs * 2 + kv) * p.nkv + kh) * p.page + os];
        }
    }
    __syncthreads();
    // Loads are not conditional, or each would wait for its own: what stays is read in its place.
    constexpr int KV = HD * ES / 16, KI = EV_UNIT * KV / 256;  // 16-byte pieces of a key, of a thread
    u32x4 key[KI];
#pragma unroll
    for (int i = 0; i < KI; ++i) {
        const int* at = s_at[(i * 256 + tid) / KV];
        key[i] = *(reinterpret_cast<const u32x4*>((const char*)p.kv_base + (((size_t)at[0] * 2 * p.nkv + kh) * p.page + at[1]) * HD * ES) + tid % KV);
    }
    using E = std::conditional_t<ES == 2, uint16_t, uint8_t>;
    struct alignas(8 * ES) Window { E v[8]; };
    E* base = reinterpret_cast<E*>(p.kv_base);
    constexpr int WI = EV_UNIT / 8 * HD / 256;                 // windows of a thread: neighbouring threads take a channel's two windows of 16 slots
    Window x[WI];
#pragma unroll
    for (int i = 0; i < WI; ++i) {
        const int item = i * 256 + tid, w = item / (2 * HD) * 2 + (item & 1), d = item % (2 * HD) >> 1;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int* at = s_at[w * 8 + e];
            x[i].v[e] = base[((((size_t)at[0] * 2 + 1) * p.nkv + kh) * HD + d) * p.page + at[1]];
        }
    }
#pragma unroll
    for (int i = 0; i < KI; ++i) {
        const int t = (i * 256 + tid) / KV, *at = s_at[t];
        if (s_hole[t >> 5] >> (t & 31) & 1) *(reinterpret_cast<u32x4*>((char*)p.kv_base + (((size_t)at[2] * 2 * p.nkv + kh) * p.page + at[3]) * HD * ES) + tid % KV) = key[i];
    }
#pragma unroll
    for (int i = 0; i < WI; ++i) {
        const int item = i * 256 + tid, w = item / (2 * HD) * 2 + (item & 1), d = item % (2 * HD) >> 1, *at = s_at[w * 8];   // a window lies in one page
        if (s_hole[w >> 2] >> ((w & 3) * 8) & 0xFF) *reinterpret_cast<Window*>(base + ((((size_t)at[2] * 2 + 1) * p.nkv + kh) * HD + d) * p.page + at[3]) = x[i];
    }
}

inline int evict_cap(int keep, int max_seq) { return std::max(0, std::min(keep, max_seq - keep)); }
inline int evict_units(int keep, int max_seq) { return cdiv(std::min(keep, max_seq), EV_UNIT); }

} // namespace

extern "C" size_t mi355_kv_evict_workspace_bytes(int32_t B, int32_t nkv, int32_t keep, int32_t max_seq_len) {
    if (B <= 0 || nkv <= 0 || keep <= 0 || max_seq_len <= 0) return 0;
    return (size_t)B * nkv * (2 + 2 * (size_t)evict_cap(keep, max_seq_len) + evict_units(keep, max_seq_len)) * sizeof(int32_t);
}

extern "C" int mi355_kv_evict(const mi355_kv_layer_t* kv, float* weights, int32_t* key_pos, const int32_t* block_table, int32_t max_blocks_per_seq, const int32_t* seq_lens,
                              const int32_t* next_pos, int32_t B, int32_t max_seq_len, int32_t keep, int32_t sinks, int32_t recent, int32_t* new_lens, void* workspace,
                              size_t workspace_bytes, mi355_stream_t stream) {
    MI355_CHECK_ARG(kv && kv->kv_base && weights && key_pos && block_table && seq_lens && next_pos, "kv_evict: null pointer");
    MI355_CHECK_ARG(kv->hd == 64 || kv->hd == 128, "kv_evict: hd=%d (64 or 128)", kv->hd);
    MI355_CHECK_ARG(kv->page >= 16 && kv->page % 8 == 0, "kv_evict: page=%d (>= 16, multiple of 8)", kv->page);
    MI355_CHECK_ARG(B > 0 && B <= 65535 && kv->nkv > 0 && kv->nkv <= 65535 && kv->num_blocks > 0, "kv_evict: B=%d nkv=%d num_blocks=%d", B, kv->nkv, kv->num_blocks);
    MI355_CHECK_ARG(max_seq_len > 0 && max_seq_len < (1 << 30) && max_blocks_per_seq > 0 && (long)max_blocks_per_seq * kv->page >= max_seq_len, "kv_evict: max_seq_len=%d exceeds the block table", max_seq_len);
    MI355_CHECK_ARG(((long)max_seq_len + EV_UNIT) * kv->page < (1l << 32), "kv_evict: (max_seq_len=%d + 64) * page=%d >= 2^32", max_seq_len, kv->page);
    MI355_CHECK_ARG(keep > 0 && sinks >= 0 && recent >= 0 && (long)sinks + recent <= keep, "kv_evict: keep=%d of which %d + %d always (keep > 0, sinks + recent <= keep)", keep, sinks, recent);
    const bool int8 = kv->kv_dtype == MI355_KV_INT8;
    MI355_CHECK_ARG(int8 || kv->kv_dtype == MI355_KV_FP16 || kv->kv_dtype == MI355_KV_BF16, "kv_evict: kv_dtype=%d", kv->kv_dtype);
    MI355_CHECK_ARG(!int8 || kv->scale_base, "kv_evict: int8 cache needs scale_base");
    MI355_CHECK_ARG(((uintptr_t)kv->kv_base & 15) == 0, "kv_evict: the cache lies on 16 bytes");
    const size_t need = mi355_kv_evict_workspace_bytes(B, kv->nkv, keep, max_seq_len);
    if (need > workspace_bytes || !workspace) {
        mi355_set_error("kv_evict: workspace %zu < %zu", workspace_bytes, need);
        return MI355_ERR_WORKSPACE;
    }
    EvictParams p;
    p.kv_base = kv->kv_base; p.scale_base = kv->scale_base; p.weights = weights; p.key_pos = key_pos; p.block_table = block_table; p.seq_lens = seq_lens; p.next_pos = next_pos;
    p.new_lens = new_lens; p.max_blocks = max_blocks_per_seq; p.num_blocks = kv->num_blocks; p.nkv = kv->nkv; p.page = kv->page; p.max_seq = max_seq_len;
    p.keep = keep; p.sinks = sinks; p.recent = recent; p.cap = evict_cap(keep, max_seq_len);
    p.page_magic = (uint32_t)((1ull << 32) / (unsigned)kv->page + 1);
    p.units = evict_units(keep, max_seq_len);
    p.count = (int32_t*)workspace; p.first = p.count + (size_t)B * kv->nkv; p.lists = p.first + (size_t)B * kv->nkv * (p.units + 1);
    hipStream_t st = (hipStream_t)stream;
    if (max_seq_len <= EV_KEYS) {
        const int rc = raise_dynamic_lds((const void*)evict_plan_kernel<true>, "kv_evict");
        if (rc != MI355_OK) return rc;
        hipLaunchKernelGGL(evict_plan_kernel<true>, dim3(kv->nkv, B), dim3(EV_THREADS), ((size_t)max_seq_len + EV_FIXED) * 4, st, p);
    } else
        hipLaunchKernelGGL(evict_plan_kernel<false>, dim3(kv->nkv, B), dim3(EV_THREADS), EV_FIXED * 4, st, p);
    MI355_CHECK_LAUNCH("evict_plan_kernel");
    const dim3 grid(p.units, kv->nkv, B);
#define L_(HD_, ES_) hipLaunchKernelGGL((evict_move_kernel<HD_, ES_>), grid, dim3(256), 0, st, p)
    if (kv->hd == 128) { if (int8) L_(128, 1); else L_(128, 2); } else { if (int8) L_(64, 1); else L_(64, 2); }
#undef L_
    MI355_CHECK_LAUNCH("evict_move_kernel");
    return MI355_OK;
}
