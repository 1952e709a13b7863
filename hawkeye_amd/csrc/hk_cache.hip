// Cutting a cache to the keys that attention has used: the weight every key collects from the queries of a prompt, and the move
// of the keys with the most weight to the front of the cache.
#include "hk_common.h"

namespace {

constexpr float REMOVED = -1.0e4f;   // a key whose bias is at or below this does not exist (the framework's mask value)

// ---------------------------------------------------------------- key weights of a prompt
// w_j = sum_i 2^(s_ij - z_i),  s_ij = q_i . k_j + b_j log2 e,  z_i = log2 sum_j 2^(s_ij).
// Two launches of one structure: a wave keeps 32 rows of one operand in registers and walks 64-row tiles of the other, which the
// four waves of a workgroup share in LDS (two stages, LDS-DMA one tile ahead).  Both compute S^T = K . Q^T with
// v_mfma_f32_32x32x16_bf16: lane -> query lane & 31, register i -> key (i & 3) + 8 (i >> 2) + 4 (lane >> 5).
//   STATS: queries stay, keys pass: running maximum and sum of a query's row in the lane -> z.
//   SUMS:  keys stay, queries pass: 2^(s - z) added up in 16 registers per lane, over the 32 lanes at the end.
// No sum crosses workgroups: every order is fixed.
struct KeyWeightParams {
    const __bf16 *Q, *K;
    const float* bias;
    float* z;                        // [B][H][Nq]; +inf for a query that sees no key
    const float* w_in;
    float* w_out;
    int B, H, Nq, Nk, causal, nblk;
    int64_t ldq, bsq, ldk, bsk, bias_bs, wi_bs, wi_hs, wo_bs, wo_hs;
};

constexpr int BLK = 128;             // rows of the operand that stays, per workgroup
constexpr int TILE = 64;             // rows of the operand that passes, per stage

template <int HD, bool SUMS, bool BIAS>
__global__ __launch_bounds__(256, 2) void hk_key_weights_kernel(const KeyWeightParams p) {
    constexpr int ROWB = HD * 2, CH = HD / 8, NKS = HD / 16;
    constexpr int STAGE = TILE * ROWB;
    constexpr int RPI = 64 / CH;                           // rows one wave-wide LDS-DMA covers
    constexpr int NI = TILE / (4 * RPI);                   // of them per wave and tile
    extern __shared__ __attribute__((aligned(16))) char smem[];      // 2 stages, then [2][TILE] floats: bias (STATS) or z (SUMS)
    float* side = reinterpret_cast<float*>(smem + 2 * STAGE);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r = lane & 31, h = lane >> 5;
    const int nbh = p.B * p.H;
    // causal: the blocks with the most tiles first (keys at the front, queries at the back)
    const int rank = blockIdx.x / nbh, bh = blockIdx.x - rank * nbh;
    const int blk = (!SUMS && p.causal) ? p.nblk - 1 - rank : rank;
    const int b = bh / p.H, head = bh - b * p.H;
    const int off = p.Nk - p.Nq;                           // causal: key <= query + off
    const int n_stay = SUMS ? p.Nk : p.Nq, n_pass = SUMS ? p.Nq : p.Nk;
    const int s0 = blk * BLK + wave * 32;                  // this wave's first row of the operand that stays

    bf16x8 sf[NKS];
    {
        const int row = min(s0 + r, n_stay - 1);
        const __bf16* sp = (SUMS ? p.K + (int64_t)b * p.bsk + (int64_t)row * p.ldk : p.Q + (int64_t)b * p.bsq + (int64_t)row * p.ldq) + head * HD + 8 * h;
#pragma unroll
        for (int s = 0; s < NKS; ++s) sf[s] = *reinterpret_cast<const bf16x8*>(sp + 16 * s);
    }
    const __bf16* pbase = (SUMS ? p.Q + (int64_t)b * p.bsq : p.K + (int64_t)b * p.bsk) + head * HD;
    const int64_t ldp = SUMS ? p.ldq : p.ldk;
    const float* bias = BIAS ? p.bias + (int64_t)b * p.bias_bs : nullptr;
    float* z = p.z + (int64_t)bh * p.Nq;

    // 16-byte chunk c of row x lives at chunk c ^ (x & (CH - 1)): 16 rows x one chunk touch every bank once
    float sr = 0.f;
    auto issue = [&](int t, int stage) {
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            const int lr = (wave * NI + i) * RPI;          // first row of this piece
            const int x = lr + lane / CH, c = (lane % CH) ^ (x & (CH - 1));
            glds16_v(pbase + (int64_t)min(t * TILE + x, n_pass - 1) * ldp + c * 8, smem + stage * STAGE + lr * ROWB);
        }
        if ((SUMS || BIAS) && tid < TILE) {
            const int x = min(t * TILE + tid, n_pass - 1);
            sr = SUMS ? z[x] : bias[x];
        }
    };
    int roff[NKS];
#pragma unroll
    for (int s = 0; s < NKS; ++s) roff[s] = r * ROWB + (((2 * s + h) ^ (r & (CH - 1))) << 4);

    int t0 = 0, t1 = (n_pass + TILE - 1) / TILE;
    if (p.causal) {
        if (SUMS) t0 = max(0, blk * BLK - off) / TILE;                                       // first query that sees the block's first key
        else t1 = min(t1, (min(blk * BLK + BLK, p.Nq) - 1 + off) / TILE + 1);                // last key the block's last query sees
    }
    float kb[16];                                          // SUMS: the bias of this lane's keys, -inf for removed ones
    if (SUMS && BIAS) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const float v = bias[min(s0 + (i & 3) + 8 * (i >> 2) + 4 * h, p.Nk - 1)];
            kb[i] = v <= REMOVED ? -INFINITY : v * HK_LOG2E;
        }
    }
    float acc[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[i] = 0.f;
    float m = -1.0e30f, l = 0.f;

    if (t0 < t1) issue(t0, 0);
    for (int t = t0; t < t1; ++t) {
        const int cur = (t - t0) & 1;
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // the LDS-DMA of this tile, unknown to the compiler
        if ((SUMS || BIAS) && tid < TILE) side[cur * TILE + tid] = sr;
        __syncthreads();                                   // tile t stands; everyone has left tile t - 1
        if (t + 1 < t1) issue(t + 1, cur ^ 1);
        const char* ts = smem + cur * STAGE;
#pragma unroll
        for (int g = 0; g < 2; ++g) {
            f32x16 st;
#pragma unroll
            for (int i = 0; i < 16; ++i) st[i] = 0.f;
#pragma unroll
            for (int s = 0; s < NKS; ++s) {
                const bf16x8 pf = *reinterpret_cast<const bf16x8*>(ts + g * 32 * ROWB + roff[s]);
                st = SUMS ? __builtin_amdgcn_mfma_f32_32x32x16_bf16(sf[s], pf, st, 0, 0, 0)
                          : __builtin_amdgcn_mfma_f32_32x32x16_bf16(pf, sf[s], st, 0, 0, 0);
            }
            const int p0 = t * TILE + g * 32;              // first row of this half tile
            const int q = SUMS ? p0 + r : s0 + r;          // the lane's query
            const int key0 = (SUMS ? s0 : p0) + 4 * h;     // register i: key key0 + (i & 3) + 8 (i >> 2)
            if (BIAS) {
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    if (SUMS) {
                        st[i] = kb[i] == -INFINITY ? -INFINITY : st[i] + kb[i];
                    } else {
                        const float v = side[cur * TILE + g * 32 + 4 * h + (i & 3) + 8 * (i >> 2)];
                        st[i] = v <= REMOVED ? -INFINITY : st[i] + v * HK_LOG2E;
                    }
                }
            }
            const int lim = p.causal ? min(p.Nk - 1, q + off) : p.Nk - 1;    // last key the query sees
            const bool edge = SUMS ? (p0 + 32 > p.Nq || (p.causal && s0 + 31 > p0 + off)) : (p0 + 32 > p.Nk || (p.causal && p0 + 31 > s0 + off));
            if (edge) {
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (key0 + (i & 3) + 8 * (i >> 2) > lim || (SUMS && q >= p.Nq)) st[i] = -INFINITY;
            }
            if (SUMS) {
                const float zq = side[cur * TILE + g * 32 + r];
#pragma unroll
                for (int i = 0; i < 16; ++i) acc[i] += __builtin_amdgcn_exp2f(st[i] - zq);
            } else {
                float mx = fmaxf(st[0], st[1]);
#pragma unroll
                for (int i = 2; i < 16; i += 2) mx = fmaxf(mx, fmaxf(st[i], st[i + 1]));
                if (__builtin_amdgcn_ballot_w64(mx > m + 8.f)) {
                    const float mn = fmaxf(m, mx);
                    l *= __builtin_amdgcn_exp2f(m - mn);
                    m = mn;
                }
#pragma unroll
                for (int i = 0; i < 16; ++i) l += __builtin_amdgcn_exp2f(st[i] - m);
            }
        }
    }
    if (SUMS) {
#pragma unroll
        for (int o = 1; o < 32; o <<= 1)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[i] += __shfl_xor(acc[i], o, 64);
        const float* wi = p.w_in ? p.w_in + (int64_t)b * p.wi_bs + (int64_t)head * p.wi_hs : nullptr;
        float* wo = p.w_out + (int64_t)b * p.wo_bs + (int64_t)head * p.wo_hs;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int key = s0 + (i & 3) + 8 * (i >> 2) + 4 * h;
            if (r == i && key < p.Nk) wo[key] = (wi ? wi[key] : 0.f) + acc[i];
        }
    } else {
        const float mo = __shfl_xor(m, 32, 64), lo = __shfl_xor(l, 32, 64);
        const float M = fmaxf(m, mo);
        const float sum = l * __builtin_amdgcn_exp2f(m - M) + lo * __builtin_amdgcn_exp2f(mo - M);
        if (h == 0 && s0 + r < p.Nq) z[s0 + r] = sum == 0.f ? INFINITY : M + __log2f(sum);
    }
}

template <int HD, bool SUMS, bool BIAS>
int launch_key_weights(KeyWeightParams p, hipStream_t s) {
    constexpr int LDS = 2 * TILE * HD * 2 + 2 * TILE * 4;
    p.nblk = ((SUMS ? p.Nk : p.Nq) + BLK - 1) / BLK;
    hipLaunchKernelGGL((hk_key_weights_kernel<HD, SUMS, BIAS>), dim3((unsigned)((int64_t)p.nblk * p.B * p.H)), dim3(256), LDS, s, p);
    return HK_OK;
}
template <int HD>
void launch_both(const KeyWeightParams& p, hipStream_t s) {
    if (p.bias) {
        launch_key_weights<HD, false, true>(p, s);
        launch_key_weights<HD, true, true>(p, s);
    } else {
        launch_key_weights<HD, false, false>(p, s);
        launch_key_weights<HD, true, false>(p, s);
    }
}

// ---------------------------------------------------------------- eviction
struct EvictParams {
    const __bf16 *K, *V;
    __bf16 *KO, *VO;
    const float *w, *bias;
    float *w_out, *bias_out;
    int32_t* kept;
    int B, H, n, budget, recent, in_place;
    int64_t ldk, bsk, ldv, bsv, ldko, bsko, ldvo, bsvo, w_bs, w_hs, wo_bs, wo_hs, b_bs, b_hs, bo_bs, bo_hs;
};

constexpr int SEL_T = 1024;
constexpr int SEL_LDS = 12288;       // keys whose ranks fit the workgroup's LDS

// fp32 -> a whole number that orders like it: removed < NaN < -inf < ... < -0 = 0 < ... < inf < recent
__device__ __forceinline__ uint32_t rank_of(float w, bool removed, bool recent) {
    const uint32_t u = __builtin_bit_cast(uint32_t, w + 0.f);
    uint32_t k = (u >> 31) ? ~u : u | 0x80000000u;
    if (w != w) k = 1u;
    if (removed) k = 0u;
    return recent ? 0xffffffffu : k;
}

// One workgroup per (sequence, head): the budget-th largest rank by four rounds of an 8-bit histogram, then one ordered pass that
// keeps the ranks above it and, of those equal, the first ones; indices, weights and biases move with it (a round's values are in
// registers before any of its stores, and go to places at or below the ones they came from: in place is safe).
template <bool IN_LDS>
__global__ __launch_bounds__(SEL_T) void hk_evict_select_kernel(const EvictParams p) {
    extern __shared__ uint32_t ranks[];
    __shared__ uint32_t hist[256];
    __shared__ uint32_t pick[2];
    __shared__ uint32_t wsum[SEL_T / 64];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int b = blockIdx.x / p.H, head = blockIdx.x - b * p.H;
    const float* w = p.w + (int64_t)b * p.w_bs + (int64_t)head * p.w_hs;
    const float* bias = p.bias ? p.bias + (int64_t)b * p.b_bs + (int64_t)head * p.b_hs : nullptr;
    float* wo = p.w_out + (int64_t)b * p.wo_bs + (int64_t)head * p.wo_hs;
    float* bo = p.bias ? p.bias_out + (int64_t)b * p.bo_bs + (int64_t)head * p.bo_hs : nullptr;
    int32_t* kept = p.kept + (int64_t)blockIdx.x * p.budget;
    auto rank_at = [&](int j) { return rank_of(w[j], bias && bias[j] <= REMOVED, j >= p.n - p.recent); };
    if (IN_LDS) {
        for (int j = tid; j < p.n; j += SEL_T) ranks[j] = rank_at(j);
    }
    uint32_t prefix = 0, want = (uint32_t)p.budget;        // the want-th largest of the ranks that begin with prefix
    for (int shift = 24; shift >= 0; shift -= 8) {
        if (tid < 256) hist[tid] = 0;
        __syncthreads();
        for (int j = tid; j < p.n; j += SEL_T) {
            const uint32_t k = IN_LDS ? ranks[j] : rank_at(j);
            if (shift == 24 || (k >> (shift + 8)) == prefix) atomicAdd(&hist[(k >> shift) & 255u], 1u);
        }
        __syncthreads();
        if (wave == 0) {                                   // lane L: bins 255 - 4 L downwards
            uint32_t c[4], s = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                c[i] = hist[255 - 4 * lane - i];
                s += c[i];
            }
            uint32_t before = s;
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const uint32_t x = __shfl_up(before, o, 64);
                if (lane >= o) before += x;
            }
            before -= s;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (before < want && want <= before + c[i]) {
                    pick[0] = 255 - 4 * lane - i;
                    pick[1] = want - before;
                }
                before += c[i];
            }
        }
        __syncthreads();
        prefix = (prefix << 8) | pick[0];
        want = pick[1];
    }
    // ---- ordered pass: rank > prefix, and the first `want` of those equal to it ----
    uint32_t above = 0, equal = 0;                         // met so far
    for (int j0 = 0; j0 < p.n; j0 += SEL_T) {
        const int j = j0 + tid;
        const bool in = j < p.n;
        const uint32_t k = !in ? 0u : IN_LDS ? ranks[j] : rank_at(j);
        const float wv = in ? w[j] : 0.f, bv = in && bias ? bias[j] : 0.f;
        const uint64_t ga = __builtin_amdgcn_ballot_w64(in && k > prefix), ge = __builtin_amdgcn_ballot_w64(in && k == prefix);
        const uint64_t lower = (1ull << lane) - 1;
        if (lane == 0) wsum[wave] = (uint32_t)__popcll(ga) | (uint32_t)__popcll(ge) << 16;
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // wv, bv are in registers before anyone stores
        __syncthreads();
        uint32_t ba = above, be = equal;
        for (int x = 0; x < SEL_T / 64; ++x) {
            const uint32_t s = wsum[x];
            if (x < wave) {
                ba += s & 0xffffu;
                be += s >> 16;
            }
            above += s & 0xffffu;
            equal += s >> 16;
        }
        ba += (uint32_t)__popcll(ga & lower);
        be += (uint32_t)__popcll(ge & lower);
        if (in && (k > prefix || (k == prefix && be < want))) {
            const uint32_t at = ba + min(be, want);
            kept[at] = j;
            wo[at] = wv;
            if (bo) bo[at] = bv;
        }
        __syncthreads();
    }
    if (p.in_place)                                        // the places that became free: nothing collected, nothing removed
        for (int j = p.budget + tid; j < p.n; j += SEL_T) {
            wo[j] = 0.f;
            if (bo) bo[j] = 0.f;
        }
}

// Rows into another cache: 16 bytes of K and of V per thread and step, neighbouring heads of one destination row next to each other, so
// that whole destination rows are written; the source rows are HD * 2 byte pieces.
template <int HD>
__global__ __launch_bounds__(256) void hk_evict_copy_kernel(const EvictParams p) {
    constexpr int CH = HD / 8, U = 2;
    const int64_t total = (int64_t)p.B * p.budget * p.H;
    const int64_t first = ((int64_t)blockIdx.x * 256 + threadIdx.x) / CH;
    const int c = threadIdx.x % CH;
    u32x4 kv[U], vv[U];
    int64_t ko[U], vo[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int64_t at = first + u * (int64_t)gridDim.x * (256 / CH);
        const int64_t x = at < total ? at : total - 1;
        const int64_t br = x / p.H;
        const int head = (int)(x - br * p.H), b = (int)(br / p.budget), row = (int)(br - (int64_t)b * p.budget);
        const int64_t src = p.kept[((int64_t)b * p.H + head) * p.budget + row];
        kv[u] = *reinterpret_cast<const u32x4*>(p.K + (int64_t)b * p.bsk + src * p.ldk + head * HD + c * 8);
        vv[u] = *reinterpret_cast<const u32x4*>(p.V + (int64_t)b * p.bsv + src * p.ldv + head * HD + c * 8);
        ko[u] = at < total ? (int64_t)b * p.bsko + row * p.ldko + head * HD + c * 8 : -1;
        vo[u] = (int64_t)b * p.bsvo + row * p.ldvo + head * HD + c * 8;
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
        if (ko[u] >= 0) {
            *reinterpret_cast<u32x4*>(p.KO + ko[u]) = kv[u];
            *reinterpret_cast<u32x4*>(p.VO + vo[u]) = vv[u];
        }
}

// Rows within the cache: one workgroup per (sequence, head, K or V) walks the kept rows upwards.  Row `at` comes from kept[at] >= at, so
// a step's stores can only hit sources of the same or an earlier step: all of a step's loads have arrived before its first store.
template <int HD>
__global__ __launch_bounds__(512) void hk_evict_move_kernel(const EvictParams p) {
    constexpr int CH = HD / 8, RPS = 512 / CH, U = 8;
    const int bh = blockIdx.x >> 1, b = bh / p.H, head = bh - b * p.H;
    const bool is_v = blockIdx.x & 1;
    const int64_t ld = is_v ? p.ldvo : p.ldko;
    __bf16* base = (is_v ? p.VO + (int64_t)b * p.bsvo : p.KO + (int64_t)b * p.bsko) + head * HD + (threadIdx.x % CH) * 8;
    const int32_t* kept = p.kept + (int64_t)bh * p.budget;
    const int g = threadIdx.x / CH;
    for (int r0 = 0; r0 < p.budget; r0 += RPS * U) {
        u32x4 x[U];
        int src[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int at = r0 + u * RPS + g;
            src[u] = kept[min(at, p.budget - 1)];
            x[u] = *reinterpret_cast<const u32x4*>(base + (int64_t)src[u] * ld);
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int at = r0 + u * RPS + g;
            if (at < p.budget && src[u] != at) *reinterpret_cast<u32x4*>(base + (int64_t)at * ld) = x[u];
        }
    }
}

}  // namespace

extern "C" int hk_attn_key_weights_bf16(const hk_key_weights_desc* d, void* stream) {
    HK_REQUIRE(d && d->Q && d->K && d->w_out, "hk_attn_key_weights_bf16: null operand");
    HK_REQUIRE(d->B >= 1 && d->B < 65536 && d->H >= 1 && d->H < 65536 && d->Nq >= 1 && d->Nk >= 1 && d->Nq < (1 << 26) && d->Nk < (1 << 26) &&
                   (d->head_dim == 64 || d->head_dim == 128) && (!d->causal || d->Nk >= d->Nq),
               "hk_attn_key_weights_bf16: bad shape B=%d H=%d Nq=%d Nk=%d head_dim=%d (head size 64 or 128, causal needs Nk >= Nq)", d->B, d->H,
               d->Nq, d->Nk, d->head_dim);
    HK_REQUIRE(((d->ldq | d->bsq | d->ldk | d->bsk) & 7) == 0 && d->ldq >= 0 && d->bsq >= 0 && d->ldk >= 0 && d->bsk >= 0,
               "hk_attn_key_weights_bf16: strides must be multiples of 8 elements, not negative");
    HK_REQUIRE(((uintptr_t)d->Q | (uintptr_t)d->K) % 16 == 0 &&
                   ((uintptr_t)d->key_bias | (uintptr_t)d->w_in | (uintptr_t)d->w_out | (uintptr_t)d->ws) % 4 == 0,
               "hk_attn_key_weights_bf16: operands must be 16-byte aligned");
    HK_REQUIRE((d->H == 1 || d->wo_hs >= d->Nk) && (d->B == 1 || d->wo_bs >= (d->H - 1) * d->wo_hs + d->Nk) && d->wi_bs >= 0 && d->wi_hs >= 0 &&
                   d->bias_bs >= 0,
               "hk_attn_key_weights_bf16: rows of w_out must not overlap, strides must not be negative");
    HK_REQUIRE(d->w_in != d->w_out || (d->wi_bs == d->wo_bs && d->wi_hs == d->wo_hs),
               "hk_attn_key_weights_bf16: weights updated in place must have one layout");
    const size_t need = (size_t)d->B * d->H * d->Nq * 4;
    HK_REQUIRE(d->ws && d->ws_bytes >= need, "hk_attn_key_weights_bf16: workspace of %zu bytes, B * H * Nq floats = %zu needed",
               d->ws ? d->ws_bytes : (size_t)0, need);
    {
        const int64_t row = (int64_t)d->H * d->head_dim;
        const HkSpan wo = hk_span(d->w_out, d->B, d->wo_bs, d->H, d->wo_hs, d->Nk, 4), w = hk_span(d->ws, 1, 0, 1, 0, (int64_t)need, 1);
        const HkSpan in[] = {hk_span(d->Q, d->B, d->bsq, d->Nq, d->ldq, row, 2), hk_span(d->K, d->B, d->bsk, d->Nk, d->ldk, row, 2),
                             hk_span(d->key_bias, d->B, d->bias_bs, 1, 0, d->Nk, 4),
                             d->w_in == d->w_out ? HkSpan{0, 0} : hk_span(d->w_in, d->B, d->wi_bs, d->H, d->wi_hs, d->Nk, 4)};
        for (int i = 0; i < 4; ++i)
            HK_REQUIRE(!hk_overlap(wo, in[i]) && !hk_overlap(w, in[i]), "hk_attn_key_weights_bf16: the output or the workspace overlaps an input");
        HK_REQUIRE(!hk_overlap(wo, w), "hk_attn_key_weights_bf16: the output overlaps the workspace");
    }
    const int64_t most = ((d->Nq > d->Nk ? d->Nq : d->Nk) + BLK - 1) / BLK;
    HK_REQUIRE(most * d->B * d->H < (1LL << 31), "hk_attn_key_weights_bf16: grid too large");
    KeyWeightParams p = {};
    p.Q = reinterpret_cast<const __bf16*>(d->Q);
    p.K = reinterpret_cast<const __bf16*>(d->K);
    p.bias = d->key_bias;
    p.z = reinterpret_cast<float*>(d->ws);
    p.w_in = d->w_in;
    p.w_out = d->w_out;
    p.B = d->B;
    p.H = d->H;
    p.Nq = d->Nq;
    p.Nk = d->Nk;
    p.causal = d->causal != 0;
    p.ldq = d->ldq;
    p.bsq = d->bsq;
    p.ldk = d->ldk;
    p.bsk = d->bsk;
    p.bias_bs = d->bias_bs;
    p.wi_bs = d->wi_bs;
    p.wi_hs = d->wi_hs;
    p.wo_bs = d->wo_bs;
    p.wo_hs = d->wo_hs;
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    if (d->head_dim == 128) launch_both<128>(p, s);
    else launch_both<64>(p, s);
    HK_CHECK_LAUNCH("hk_attn_key_weights_bf16");
    return HK_OK;
}

extern "C" int hk_cache_evict_bf16(const hk_cache_evict_desc* d, void* stream) {
    HK_REQUIRE(d && d->K && d->V && d->k_out && d->v_out && d->weight && d->weight_out && d->kept, "hk_cache_evict_bf16: null operand");
    HK_REQUIRE(d->B >= 1 && d->H >= 1 && d->H < 65536 && (int64_t)d->B * d->H < (1 << 27) && (d->head_dim == 64 || d->head_dim == 128),
               "hk_cache_evict_bf16: bad shape B=%d H=%d head_dim=%d (head size 64 or 128)", d->B, d->H, d->head_dim);
    HK_REQUIRE(d->n_keys >= 1 && d->n_keys < (1 << 28) && d->budget >= 1 && d->budget <= d->n_keys && d->recent >= 0 && d->recent <= d->budget,
               "hk_cache_evict_bf16: n_keys=%d budget=%d recent=%d (0 <= recent <= budget <= n_keys, 1 <= budget)", d->n_keys, d->budget, d->recent);
    HK_REQUIRE((d->key_bias == nullptr) == (d->key_bias_out == nullptr), "hk_cache_evict_bf16: key_bias and key_bias_out come together");
    const int64_t row = (int64_t)d->H * d->head_dim;
    HK_REQUIRE(((d->ldk | d->bsk | d->ldv | d->bsv | d->ldko | d->bsko | d->ldvo | d->bsvo) & 7) == 0 && d->ldk >= 0 && d->bsk >= 0 && d->ldv >= 0 &&
                   d->bsv >= 0 && d->w_bs >= 0 && d->w_hs >= 0 && d->b_bs >= 0 && d->b_hs >= 0,
               "hk_cache_evict_bf16: strides must be multiples of 8 elements, not negative");
    HK_REQUIRE(d->ldko >= row && d->ldvo >= row && (d->B == 1 || (d->bsko >= row && d->bsvo >= row)),
               "hk_cache_evict_bf16: output rows must not overlap");
    HK_REQUIRE(((uintptr_t)d->K | (uintptr_t)d->V | (uintptr_t)d->k_out | (uintptr_t)d->v_out) % 16 == 0 &&
                   ((uintptr_t)d->weight | (uintptr_t)d->weight_out | (uintptr_t)d->key_bias | (uintptr_t)d->key_bias_out | (uintptr_t)d->kept) % 4 == 0,
               "hk_cache_evict_bf16: caches must be 16-byte aligned");
    const bool in_place = d->K == d->k_out;
    HK_REQUIRE(d->k_out != d->v_out, "hk_cache_evict_bf16: K and V need a cache each");
    HK_REQUIRE(in_place == (d->V == d->v_out) && in_place == (d->weight == d->weight_out) &&
                   (d->key_bias == nullptr || in_place == (d->key_bias == d->key_bias_out)),
               "hk_cache_evict_bf16: K, V, weights and biases are cut in place together or not at all");
    HK_REQUIRE(!in_place || (d->ldk == d->ldko && d->bsk == d->bsko && d->ldv == d->ldvo && d->bsv == d->bsvo && d->w_bs == d->wo_bs &&
                             d->w_hs == d->wo_hs && d->b_bs == d->bo_bs && d->b_hs == d->bo_hs),
               "hk_cache_evict_bf16: in place, input and output must have one layout");
    const int64_t wlen = in_place ? d->n_keys : d->budget;
    HK_REQUIRE((d->H == 1 || d->wo_hs >= wlen) && (d->B == 1 || d->wo_bs >= (d->H - 1) * d->wo_hs + wlen) &&
                   (d->key_bias == nullptr || ((d->H == 1 || d->bo_hs >= wlen) && (d->B == 1 || d->bo_bs >= (d->H - 1) * d->bo_hs + wlen))),
               "hk_cache_evict_bf16: rows of the weights and biases written must not overlap");
    {
        const HkSpan out[] = {hk_span(d->k_out, d->B, d->bsko, d->budget, d->ldko, row, 2), hk_span(d->v_out, d->B, d->bsvo, d->budget, d->ldvo, row, 2),
                              hk_span(d->weight_out, d->B, d->wo_bs, d->H, d->wo_hs, wlen, 4),
                              hk_span(d->key_bias_out, d->B, d->bo_bs, d->H, d->bo_hs, wlen, 4),
                              hk_span(d->kept, 1, 0, 1, 0, (int64_t)d->B * d->H * d->budget, 4)};
        const HkSpan in[] = {hk_span(d->K, d->B, d->bsk, d->n_keys, d->ldk, row, 2), hk_span(d->V, d->B, d->bsv, d->n_keys, d->ldv, row, 2),
                             hk_span(d->weight, d->B, d->w_bs, d->H, d->w_hs, d->n_keys, 4),
                             hk_span(d->key_bias, d->B, d->b_bs, d->H, d->b_hs, d->n_keys, 4)};
        for (int i = 0; i < 5; ++i) {
            for (int j = 0; j < 4; ++j)      // in place, an output is its own input
                HK_REQUIRE((in_place && i == j) || !hk_overlap(out[i], in[j]), "hk_cache_evict_bf16: an output overlaps an input");
            for (int j = 0; j < i; ++j) HK_REQUIRE(!hk_overlap(out[i], out[j]), "hk_cache_evict_bf16: two outputs overlap");
        }
    }
    EvictParams p = {};
    p.K = reinterpret_cast<const __bf16*>(d->K);
    p.V = reinterpret_cast<const __bf16*>(d->V);
    p.KO = reinterpret_cast<__bf16*>(d->k_out);
    p.VO = reinterpret_cast<__bf16*>(d->v_out);
    p.w = d->weight;
    p.bias = d->key_bias;
    p.w_out = d->weight_out;
    p.bias_out = d->key_bias_out;
    p.kept = d->kept;
    p.B = d->B;
    p.H = d->H;
    p.n = d->n_keys;
    p.budget = d->budget;
    p.recent = d->recent;
    p.in_place = in_place;
    p.ldk = d->ldk;
    p.bsk = d->bsk;
    p.ldv = d->ldv;
    p.bsv = d->bsv;
    p.ldko = d->ldko;
    p.bsko = d->bsko;
    p.ldvo = d->ldvo;
    p.bsvo = d->bsvo;
    p.w_bs = d->w_bs;
    p.w_hs = d->w_hs;
    p.wo_bs = d->wo_bs;
    p.wo_hs = d->wo_hs;
    p.b_bs = d->b_bs;
    p.b_hs = d->b_hs;
    p.bo_bs = d->bo_bs;
    p.bo_hs = d->bo_hs;
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    const unsigned pairs = (unsigned)(p.B * p.H);
    if (p.n <= SEL_LDS) hipLaunchKernelGGL((hk_evict_select_kernel<true>), dim3(pairs), dim3(SEL_T), (size_t)p.n * 4, s, p);
    else hipLaunchKernelGGL((hk_evict_select_kernel<false>), dim3(pairs), dim3(SEL_T), 0, s, p);
    if (in_place) {
        if (d->head_dim == 128) hipLaunchKernelGGL((hk_evict_move_kernel<128>), dim3(pairs * 2), dim3(512), 0, s, p);
        else hipLaunchKernelGGL((hk_evict_move_kernel<64>), dim3(pairs * 2), dim3(512), 0, s, p);
    } else {
        const int64_t pieces = (int64_t)p.B * p.H * p.budget, per = 256 / (d->head_dim / 8) * 2;
        HK_REQUIRE((pieces + per - 1) / per < (1LL << 31), "hk_cache_evict_bf16: grid too large");
        const unsigned grid = (unsigned)((pieces + per - 1) / per);
        if (d->head_dim == 128) hipLaunchKernelGGL((hk_evict_copy_kernel<128>), dim3(grid), dim3(256), 0, s, p);
        else hipLaunchKernelGGL((hk_evict_copy_kernel<64>), dim3(grid), dim3(256), 0, s, p);
    }
    HK_CHECK_LAUNCH("hk_cache_evict_bf16");
    return HK_OK;
}
