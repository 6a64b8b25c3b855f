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
    int max_blocks, num_blocks, nkv, hd, page, max_seq, keep, sinks, recent, cap;
};

constexpr int EV_THREADS = 1024, EV_WAVES = EV_THREADS / 64, EV_COPIES = 8, EV_KEYS = 32768, EV_FIXED = 256 * EV_COPIES + 256 + 2 + EV_WAVES;   // words of LDS beside the ranks
static_assert((EV_KEYS + EV_FIXED) * 4 <= 160 * 1024, "LDS of a block");

__device__ __forceinline__ uint32_t evict_rank(const EvictParams& p, int b, int kh, int t, int newest) {
    const int blk = p.block_table[(size_t)b * p.max_blocks + t / p.page];
    if (blk < 0 || blk >= p.num_blocks) return 0u;
    const size_t at = ((size_t)blk * p.nkv + kh) * p.page + t % p.page;
    const int pos = p.key_pos[at];
    const float w = p.weights[at] + 0.f;                      // -0 as 0
    if (pos < p.sinks || pos >= newest) return 0xFFFFFFFFu;
    if (w != w) return 0u;
    const uint32_t u = __builtin_bit_cast(uint32_t, w);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// IN_LDS: the ranks fit there; else they are formed again by every pass.
template <bool IN_LDS>
__global__ __launch_bounds__(EV_THREADS) void evict_plan_kernel(const EvictParams p) {
    extern __shared__ uint32_t ev_sm[];
    uint32_t *hist = ev_sm, *sum = hist + 256 * EV_COPIES, *found = sum + 256;
    int* part = reinterpret_cast<int*>(found + 2);
    uint32_t* ranks = found + 2 + EV_WAVES;
    const int kh = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = min(max(p.seq_lens[b], 0), p.max_seq);
    int32_t* cnt = p.count + (size_t)b * p.nkv + kh;
    if (n <= p.keep) { if (tid == 0) *cnt = 0; return; }
    const int newest = p.next_pos[b] - p.recent;
    auto rank = [&](int t) { return IN_LDS ? ranks[t] : evict_rank(p, b, kh, t, newest); };
    if (IN_LDS) {
        for (int t = tid; t < n; t += EV_THREADS) ranks[t] = evict_rank(p, b, kh, t, newest);
        __syncthreads();
    }
    // the keep-th largest rank, 8 bits at a time
    uint32_t prefix = 0, left = p.keep;
    for (int shift = 24; shift >= 0; shift -= 8) {
        for (int i = tid; i < 256 * EV_COPIES; i += EV_THREADS) hist[i] = 0;
        __syncthreads();
        const uint32_t mask = shift == 24 ? 0u : 0xFFFFFFFFu << (shift + 8);
        for (int t = tid; t < n; t += EV_THREADS) {
            const uint32_t u = rank(t);
            if ((u & mask) == prefix) atomicAdd(&hist[(u >> shift & 255) * EV_COPIES + (lane & (EV_COPIES - 1))], 1u);
        }
        __syncthreads();
        if (tid < 256) {
            uint32_t s = 0;
#pragma unroll
            for (int c = 0; c < EV_COPIES; ++c) s += hist[tid * EV_COPIES + c];
            sum[tid] = s;
        }
        __syncthreads();
        if (wave == 0) {                                      // lane: four digits, the largest first
            uint32_t v[4], own = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) { v[i] = sum[255 - lane * 4 - i]; own += v[i]; }
            uint32_t incl = own;
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) { const uint32_t up = __shfl_up(incl, o); if (lane >= o) incl += up; }
            uint32_t before = incl - own;
            if (before < left && incl >= left) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (before < left && before + v[i] >= left) { found[0] = 255 - lane * 4 - i; found[1] = left - before; }
                    before += v[i];
                }
            }
        }
        __syncthreads();
        prefix |= found[0] << shift;
        left = found[1];
    }
    const uint32_t bar = prefix;
    const int ties = (int)left;                               // of the tokens at the bar the first `ties` slots stay
    // every wave takes a run of slots; what it starts from is the sum over the waves before
    const int run = (n + EV_WAVES * 64 - 1) / (EV_WAVES * 64) * 64, t0 = wave * run, t1 = min(n, t0 + run);
    auto before_of = [&](int mine) {
        __syncthreads();
        if (lane == 0) part[wave] = mine;
        __syncthreads();
        int s = 0;
        for (int w = 0; w < wave; ++w) s += part[w];
        return s;
    };
    int eq = 0;
    for (int t = t0; t < t1; t += 64) eq += __builtin_popcountll(__builtin_amdgcn_ballot_w64(t + lane < t1 && rank(t + lane) == bar));
    const int eq0 = before_of(eq);
    const uint64_t below = (1ull << lane) - 1;
    auto walk = [&](auto&& each) {                            // each(slots that become holes, kept ones behind keep) as masks of the wave's lanes
        int e = eq0;
        for (int t = t0; t < t1; t += 64) {
            const uint32_t u = t + lane < t1 ? rank(t + lane) : 0u;
            const uint64_t at = __builtin_amdgcn_ballot_w64(t + lane < t1 && u == bar);
            const bool kept = u > bar || (u == bar && e + __builtin_popcountll(at & below) < ties), in = t + lane < t1;
            e += __builtin_popcountll(at);
            each(t, __builtin_amdgcn_ballot_w64(in && !kept && t + lane < p.keep), __builtin_amdgcn_ballot_w64(in && kept && t + lane >= p.keep));
        }
    };
    int holes = 0, late = 0;
    walk([&](int, uint64_t h, uint64_t l) { holes += __builtin_popcountll(h); late += __builtin_popcountll(l); });
    int hole0 = before_of(holes), late0 = before_of(late);
    int32_t* src = p.lists + ((size_t)b * p.nkv + kh) * 2 * p.cap;
    int32_t* dst = src + p.cap;
    if (wave == EV_WAVES - 1 && lane == 0) *cnt = hole0 + holes;
    walk([&](int t, uint64_t h, uint64_t l) {
        if (h >> lane & 1) dst[hole0 + __builtin_popcountll(h & below)] = t + lane;
        if (l >> lane & 1) src[late0 + __builtin_popcountll(l & below)] = t + lane;
        hole0 += __builtin_popcountll(h); late0 += __builtin_popcountll(l);
    });
}

// 32 moves at a time: keys by 16 bytes, values (a channel's tokens lie side by side) a thread 8 moves apart per channel group.
constexpr int EV_MOVES = 32;
template <int HD, int ES>
__global__ __launch_bounds__(256) void evict_move_kernel(const EvictParams p) {
    __shared__ int s_at[2][EV_MOVES][2];                       // source, hole: block (-1: leave it), token
    const int kh = blockIdx.y, b = blockIdx.z, tid = threadIdx.x;
    if (blockIdx.x == 0 && kh == 0 && tid == 0 && p.new_lens) p.new_lens[b] = min(min(max(p.seq_lens[b], 0), p.max_seq), p.keep);
    const size_t pair = (size_t)b * p.nkv + kh;
    const int n = p.count[pair];
    const int32_t* list = p.lists + pair * 2 * p.cap;
    constexpr int KV = HD * ES / 16, CH = HD / 8;              // 16-byte pieces of a key; channels of a thread
    for (int m0 = blockIdx.x * EV_MOVES; m0 < n; m0 += gridDim.x * EV_MOVES) {
        if (tid < 2 * EV_MOVES) {
            const int m = tid & (EV_MOVES - 1), side = tid / EV_MOVES;
            int blk = -1, tok = 0;
            if (m0 + m < n) {
                const int t = list[(size_t)side * p.cap + m0 + m];
                blk = p.block_table[(size_t)b * p.max_blocks + t / p.page];
                tok = t % p.page;
                if (blk >= p.num_blocks) blk = -1;
            }
            s_at[side][m][0] = blk; s_at[side][m][1] = tok;
        }
        __syncthreads();
        for (int i = tid; i < EV_MOVES * KV; i += 256) {
            const int m = i / KV, c = i % KV, bs = s_at[0][m][0], bd = s_at[1][m][0];
            if (bs < 0 || bd < 0) continue;
            const u32x4* from = reinterpret_cast<const u32x4*>((const char*)p.kv_base + (((size_t)bs * 2 * p.nkv + kh) * p.page + s_at[0][m][1]) * HD * ES) + c;
            u32x4* to = reinterpret_cast<u32x4*>((char*)p.kv_base + (((size_t)bd * 2 * p.nkv + kh) * p.page + s_at[1][m][1]) * HD * ES) + c;
            *to = *from;
        }
        {
            using E = std::conditional_t<ES == 2, uint16_t, uint8_t>;
            const int m = tid & (EV_MOVES - 1), d0 = tid / EV_MOVES * CH, bs = s_at[0][m][0], bd = s_at[1][m][0];
            if (bs >= 0 && bd >= 0) {
                const E* from = reinterpret_cast<const E*>(p.kv_base) + (((size_t)bs * 2 + 1) * p.nkv + kh) * p.page * HD + s_at[0][m][1];
                E* to = reinterpret_cast<E*>(p.kv_base) + (((size_t)bd * 2 + 1) * p.nkv + kh) * p.page * HD + s_at[1][m][1];
                E v[CH];
#pragma unroll
                for (int d = 0; d < CH; ++d) v[d] = from[(size_t)(d0 + d) * p.page];
#pragma unroll
                for (int d = 0; d < CH; ++d) to[(size_t)(d0 + d) * p.page] = v[d];
                const size_t ws = ((size_t)bs * p.nkv + kh) * p.page + s_at[0][m][1], wd = ((size_t)bd * p.nkv + kh) * p.page + s_at[1][m][1];
                if (d0 == 0) p.weights[wd] = p.weights[ws];
                if (d0 == CH) p.key_pos[wd] = p.key_pos[ws];
                if (ES == 1 && d0 >= 2 * CH && d0 < 4 * CH) {          // scale plane [block][K, V][nkv][page]
                    const int kv = d0 / CH - 2;
                    p.scale_base[(((size_t)bd * 2 + kv) * p.nkv + kh) * p.page + s_at[1][m][1]] = p.scale_base[(((size_t)bs * 2 + kv) * p.nkv + kh) * p.page + s_at[0][m][1]];
                }
            }
        }
        __syncthreads();
    }
}

inline int evict_cap(int keep, int max_seq) { return std::max(0, std::min(keep, max_seq - keep)); }

} // namespace

extern "C" size_t mi355_kv_evict_workspace_bytes(int32_t B, int32_t nkv, int32_t keep, int32_t max_seq_len) {
    if (B <= 0 || nkv <= 0 || keep <= 0 || max_seq_len <= 0) return 0;
    return (size_t)B * nkv * (1 + 2 * (size_t)evict_cap(keep, max_seq_len)) * sizeof(int32_t);
}

extern "C" int mi355_kv_evict(const mi355_kv_layer_t* kv, float* weights, int32_t* key_pos, const int32_t* block_table, int32_t max_blocks_per_seq, const int32_t* seq_lens,
                              const int32_t* next_pos, int32_t B, int32_t max_seq_len, int32_t keep, int32_t sinks, int32_t recent, int32_t* new_lens, void* workspace,
                              size_t workspace_bytes, mi355_stream_t stream) {
    MI355_CHECK_ARG(kv && kv->kv_base && weights && key_pos && block_table && seq_lens && next_pos, "kv_evict: null pointer");
    MI355_CHECK_ARG(kv->hd == 64 || kv->hd == 128, "kv_evict: hd=%d (64 or 128)", kv->hd);
    MI355_CHECK_ARG(kv->page >= 16 && kv->page % 8 == 0, "kv_evict: page=%d (>= 16, multiple of 8)", kv->page);
    MI355_CHECK_ARG(B > 0 && B <= 65535 && kv->nkv > 0 && kv->nkv <= 65535 && kv->num_blocks > 0, "kv_evict: B=%d nkv=%d num_blocks=%d", B, kv->nkv, kv->num_blocks);
    MI355_CHECK_ARG(max_seq_len > 0 && max_seq_len < (1 << 30) && max_blocks_per_seq > 0 && (long)max_blocks_per_seq * kv->page >= max_seq_len, "kv_evict: max_seq_len=%d exceeds the block table", max_seq_len);
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
    p.new_lens = new_lens; p.max_blocks = max_blocks_per_seq; p.num_blocks = kv->num_blocks; p.nkv = kv->nkv; p.hd = kv->hd; p.page = kv->page; p.max_seq = max_seq_len;
    p.keep = keep; p.sinks = sinks; p.recent = recent; p.cap = evict_cap(keep, max_seq_len);
    p.count = (int32_t*)workspace; p.lists = p.count + (size_t)B * kv->nkv;
    hipStream_t st = (hipStream_t)stream;
    if (max_seq_len <= EV_KEYS) {
        const int rc = raise_dynamic_lds((const void*)evict_plan_kernel<true>, "kv_evict");
        if (rc != MI355_OK) return rc;
        hipLaunchKernelGGL(evict_plan_kernel<true>, dim3(kv->nkv, B), dim3(EV_THREADS), ((size_t)max_seq_len + EV_FIXED) * 4, st, p);
    } else
        hipLaunchKernelGGL(evict_plan_kernel<false>, dim3(kv->nkv, B), dim3(EV_THREADS), EV_FIXED * 4, st, p);
    MI355_CHECK_LAUNCH("evict_plan_kernel");
    const dim3 grid(std::max(1, std::min(cdiv(p.cap, EV_MOVES), std::max(1, 4096 / (B * kv->nkv)))), kv->nkv, B);
#define L_(HD_, ES_) hipLaunchKernelGGL((evict_move_kernel<HD_, ES_>), grid, dim3(256), 0, st, p)
    if (kv->hd == 128) { if (int8) L_(128, 1); else L_(128, 2); } else { if (int8) L_(64, 1); else L_(64, 2); }
#undef L_
    MI355_CHECK_LAUNCH("evict_move_kernel");
    return MI355_OK;
}
