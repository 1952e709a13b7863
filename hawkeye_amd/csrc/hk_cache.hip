// Cutting a cache to the keys that attention has used: the weight every key collects from the queries of a prompt, and the move
// of the keys with the most weight to the front of the cache.
#include <type_traits>
#include "hk_common.h"
#include "hk_overlap.h"

namespace {

constexpr float REMOVED = -1.0e4f;   // a key whose bias is at or below this does not exist (the framework's mask value)

// ---------------------------------------------------------------- key weights of a prompt
// w_j = sum_i 2^(s_ij - z_i),  s_ij = q_i . k_j + b_j log2 e,  z_i = log2 sum_j 2^(s_ij).
// Beyond few keys (hk_key_weights_few_kernel), two launches of one structure (and a small one between them where few queries take their keys in chunks): a wave keeps 32 rows of one operand in registers and walks 64-row tiles of the other, which the
// four waves of a workgroup share in LDS (two stages, LDS-DMA one tile ahead).  Both compute S^T = K . Q^T with
// v_mfma_f32_32x32x16_bf16: lane -> query lane & 31, register i -> key (i & 3) + 8 (i >> 2) + 4 (lane >> 5).
//   STATS: queries stay, keys pass: a reference point m and the sum of 2^(s - m) in the lane -> z.  m is the maximum of the row's first keys and
//     moves only when a tile's partial sum leaves [0, 2^20] (that tile is redone): the common path is exp2 and an addition per score.
//   SUMS:  keys stay, queries pass: 2^(s - z) added up in 16 registers per lane, over the 32 lanes at the end.
// GRP = 2: two such groups of four waves share a workgroup, each with stages of its own, and take every other tile; the second's sums
// join the first's through LDS at the end.  Chunks of keys (key_chunks) leave (m, sum) for a small launch that joins them: every order is fixed.
// Measured: 2 x 2047 tokens, 32 heads of 128, padded 75-86 us for both launches (clock), 800-910 TFLOP/s of the products they make (each makes them
// all).  The matrix unit is busy 21 % of the time, the vector unit 38 %, 1.8 waves per SIMD on average: bound by the chain of a tile within a wave
// (LDS, 16 matrix instructions, 32 exp2: about 2000 cycles) and the uneven lengths of causal blocks.  No gain: 128-row tiles, their products
// spread among the exponentials, fragments read 2-8 steps ahead, starting values kept in registers, long and short blocks paired on a CU by
// their order (each within 3 %); slower: 64 rows per wave, two waves per workgroup (twice the time), 4 and 8 stages.
struct KeyWeightParams {
    const __bf16 *Q, *K;
    const float* bias;
    float* z;                        // [B][H][Nq]; +inf for a query that sees no key
    float2* part;                    // STATS by chunks of keys: [chunk][B][H][Nq] of (reference point, sum)
    int nch, ct;                     // chunks, tiles per chunk
    const float* w_in;
    float* w_out;
    int B, H, Nq, Nk, causal, nblk;
    int64_t ldq, bsq, ldk, bsk, bias_bs, wi_bs, wi_hs, wo_bs, wo_hs;
};

constexpr int NST = 2;               // stages (a power of two): a tile is requested NST - 1 tiles ahead.  4 measured alike (STATS) or 13 % slower (SUMS)
constexpr float OVERFLOW_SUM = 1048576.0f;
constexpr int BLK = 128;             // rows of the operand that stays, per workgroup
constexpr int TILE = 64;             // rows of the operand that passes, per stage

// a[0] of lane r & 15 <- the sum of a[r & 15] over the 32 lanes of a half: each step sends the half of the values that the partner lane keeps.
// Partners differ in the bit that picks the half and share those before it: lane ^ 8, ^ 7, ^ 2, ^ 1 (all within 16 lanes), at last ^ 16.
__device__ __forceinline__ void sum_over_queries(float (&a)[16], int r) {
    auto halve = [&](auto o_c, auto dpp_c) __attribute__((always_inline)) {
        constexpr int o = decltype(o_c)::value;
        const bool up = (r & o) != 0;
#pragma unroll
        for (int i = 0; i < o; ++i) {
            const float keep = up ? a[i + o] : a[i], send = up ? a[i] : a[i + o];
            a[i] = keep + __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, send), decltype(dpp_c)::value, 0xf, 0xf, true));
        }
    };
    halve(std::integral_constant<int, 8>{}, std::integral_constant<int, 0x128>{});      // row_ror:8
    halve(std::integral_constant<int, 4>{}, std::integral_constant<int, 0x141>{});      // row_half_mirror
    halve(std::integral_constant<int, 2>{}, std::integral_constant<int, 0x4e>{});       // quad_perm [2,3,0,1]
    halve(std::integral_constant<int, 1>{}, std::integral_constant<int, 0xb1>{});       // quad_perm [1,0,3,2]
    a[0] += __shfl_xor(a[0], 16, 64);
}

template <int HD, bool SUMS, bool BIAS, int GRP>
__global__ __launch_bounds__(GRP * 256, 2) void hk_key_weights_kernel(const KeyWeightParams p) {
    constexpr int ROWB = HD * 2, CH = HD / 8, NKS = HD / 16;
    constexpr int STAGE = TILE * ROWB;
    constexpr int RPI = 64 / CH;                           // rows one wave-wide LDS-DMA covers
    constexpr int NI = TILE / (4 * RPI);                   // of them per wave and tile
    constexpr bool SIDE = SUMS || BIAS;                    // 64 floats come with a tile: its queries' z (SUMS), its keys' biases (STATS)
    constexpr int PER = NI + (SIDE ? 1 : 0);               // LDS-DMAs per wave and tile
    extern __shared__ __attribute__((aligned(16))) char smem[];      // NST stages, then [NST][wave][TILE] floats (each wave its own copy); the same for the next group
    constexpr int GROUP = NST * (STAGE + 4 * TILE * 4);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane((tid >> 6) & 3);
    const int grp = GRP == 1 ? 0 : __builtin_amdgcn_readfirstlane(tid >> 8);
    char* gs = smem + grp * GROUP;
    const int r = lane & 31, h = lane >> 5;
    const int nbh = p.B * p.H;
    // causal: the blocks with the most tiles first (keys at the front, queries at the back)
    int rank = blockIdx.x / nbh;
    const int bh = blockIdx.x - rank * nbh;
    const int c = SUMS ? 0 : rank % p.nch;
    if (!SUMS) rank /= p.nch;
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

    // 16-byte chunk c of row x lives at chunk c ^ swz(x): 16 rows x one chunk touch every bank once
    auto swz = [](int x) { return HD == 128 ? x & 15 : (x >> 1) & 7; };
    float* side = reinterpret_cast<float*>(gs + NST * STAGE) + wave * TILE;
    const int lx = lane / CH, lc = (lane % CH) ^ swz(lx);  // this lane's row and (source) chunk of a piece of RPI rows from lr:
    // swz(lr + lx) == swz(lr) ^ swz(lx), as RPI is 4 (HD 128) or 8
    const uint32_t lane_off = (uint32_t)((lx * ldp) * 2);
    int t0 = 0, t1 = (n_pass + TILE - 1) / TILE;
    if (p.causal) {
        if (SUMS) t0 = max(0, blk * BLK - off) / TILE;                                       // first query that sees the block's first key
        else t1 = min(t1, (min(blk * BLK + BLK, p.Nq) - 1 + off) / TILE + 1);                // last key the block's last query sees
    }
    if (!SUMS && p.nch > 1) {
        t0 = c * p.ct;
        t1 = max(t0, min(t1, t0 + p.ct));
    }
    auto issue = [&](int u) {                              // the group's tile of step u
        const int t = t0 + u * GRP + grp;
        if (GRP > 1 && t >= t1) return;
        char* st = gs + (u & (NST - 1)) * STAGE;
        if ((t + 1) * TILE <= n_pass) {                    // scalar base + 32-bit lane offset
#pragma unroll
            for (int i = 0; i < NI; ++i) {
                const int lr = (wave * NI + i) * RPI;      // first row of this piece
                glds16_s(pbase + (int64_t)(t * TILE + lr) * ldp, lane_off + (uint32_t)((lc ^ swz(lr)) << 4), st + lr * ROWB);
            }
        } else {
#pragma unroll
            for (int i = 0; i < NI; ++i) {
                const int lr = (wave * NI + i) * RPI;
                glds16_v(pbase + (int64_t)min(t * TILE + lr + lx, n_pass - 1) * ldp + (lc ^ swz(lr)) * 8, st + lr * ROWB);
            }
        }
        if (SIDE) glds4_s(SUMS ? z : bias, (uint32_t)min(t * TILE + lane, n_pass - 1) * 4u, side + (u & (NST - 1)) * 4 * TILE);
    };
    const int steps = (t1 - t0 + GRP - 1) / GRP;
#pragma unroll
    for (int i = 0; i < NST - 1; ++i)
        if (i < steps) issue(i);
    // The loads above are waited for here: left pending, the compiler would wait for them inside the loop, with counts that take the
    // LDS-DMA in flight there (which it does not know) along.
#pragma unroll
    for (int s = 0; s < NKS; ++s) asm volatile("" : "+v"(sf[s]));
    const int ro = r * ROWB + ((h ^ swz(r)) << 4);         // chunk 2 s + h: the 2 s joins by exclusive or

    float kb[16];                                          // SUMS: the bias of this lane's keys, -inf for removed ones
    bool kplain = true, kall = false;                      // all of the wave's biases are 0, all of its keys are removed
    if (SUMS && BIAS) {
        const float kv = bias[min(s0 + r, p.Nk - 1)];
        kplain = __builtin_amdgcn_ballot_w64(kv != 0.f) == 0;
        kall = __builtin_amdgcn_ballot_w64(kv <= REMOVED || s0 + r >= p.Nk) == ~0ull;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const float v = bias[min(s0 + (i & 3) + 8 * (i >> 2) + 4 * h, p.Nk - 1)];
            kb[i] = v <= REMOVED ? -INFINITY : v * HK_LOG2E;
            asm volatile("" : "+v"(kb[i]));
        }
    }
    float acc[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[i] = 0.f;
    float m = 0.f, l = 0.f;                                // STATS: everything is relative to m
    bool unset = true, pending = true;                     // STATS: this half row / some row of the wave has met no key yet

    for (int u = 0; u < steps; ++u) {
        const int cur = u & (NST - 1), t = t0 + u * GRP + grp;
        // this tile's LDS-DMA has arrived, those of the NST - 2 tiles behind it may be on their way (the compiler knows of none)
        if (GRP == 1 && u + NST - 2 < steps) asm volatile("s_waitcnt vmcnt(%0)" ::"n"((NST - 2) * PER) : "memory");
        else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");      // tile t stands; everyone has left the tile before
        if (u + NST - 1 < steps) issue(u + NST - 1);
        if (GRP > 1 && t >= t1) continue;
        const char* ts = gs + cur * STAGE;
        const float* sd = side + cur * 4 * TILE;
        // edges: rows of the passing operand that do not exist, keys behind the query's last
        const int p0 = t * TILE;
        const bool edge = SUMS ? (p0 + TILE > p.Nq || (p.causal && s0 + 31 > p0 + off)) : (p0 + TILE > p.Nk || (p.causal && p0 + TILE - 1 > s0 + off));
        // What the biases do to this tile, for all its keys at once: nothing (the rule: zeros), everything (all removed: no work), or some.
        // Likewise a tile of queries that see no key (padding: z = inf).
        bool plain = !BIAS;
        if (BIAS && !SUMS) {
            const float v = sd[lane];
            if (__builtin_amdgcn_ballot_w64(v <= REMOVED || p0 + lane >= p.Nk) == ~0ull) continue;
            plain = __builtin_amdgcn_ballot_w64(v != 0.f) == 0;
        }
        if (BIAS && SUMS) {
            if (kall || __builtin_amdgcn_ballot_w64(sd[lane] == INFINITY) == ~0ull) continue;
            plain = kplain;
        }
        for (bool take = !SUMS && pending;; take = true) { // STATS: a second time if a partial sum left the range; SUMS: once
            f32x16 st[2];                                  // the half tiles' products: two independent chains
            // The products start from -m only where they are of its size: added to a reference point far away, or one that biases make large, they
            // would lose bits at every step.  base: what the biases, added afterwards, are taken relative to.
            const float base = SUMS || take ? 0.f : m, start = plain ? -base : 0.f;
#pragma unroll
            for (int s = 0; s < NKS; ++s)
#pragma unroll
                for (int g = 0; g < 2; ++g) {
                    if (s == 0) {
#pragma unroll
                        for (int i = 0; i < 16; ++i) st[g][i] = SUMS ? 0.f : start;
                    }
                    const bf16x8 pf = *reinterpret_cast<const bf16x8*>(ts + g * 32 * ROWB + (ro ^ (32 * s)));
                    st[g] = SUMS ? __builtin_amdgcn_mfma_f32_32x32x16_bf16(sf[s], pf, st[g], 0, 0, 0)
                                 : __builtin_amdgcn_mfma_f32_32x32x16_bf16(pf, sf[s], st[g], 0, 0, 0);
                }
            if (!plain) {
#pragma unroll
                for (int g = 0; g < 2; ++g)
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        if (SUMS) {
                            st[g][i] = kb[i] == -INFINITY ? -INFINITY : st[g][i] + kb[i];
                        } else {
                            const float v = sd[g * 32 + 4 * h + (i & 3) + 8 * (i >> 2)];
                            st[g][i] = v <= REMOVED ? -INFINITY : st[g][i] + fmaf(v, HK_LOG2E, -base);
                        }
                    }
            }
            if (edge) {
#pragma unroll
                for (int g = 0; g < 2; ++g) {
                    const int q = SUMS ? p0 + g * 32 + r : s0 + r;                           // the lane's query
                    int lim = p.causal ? min(p.Nk - 1, q + off) : p.Nk - 1;                  // last key it sees
                    if (SUMS && q >= p.Nq) lim = -1;
                    lim -= (SUMS ? s0 : p0 + g * 32) + 4 * h;                                // register i: key (i & 3) + 8 (i >> 2) from here
                    asm volatile("" : "+v"(lim));     // (left to itself the compiler makes the comparisons for every tile)
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        if ((i & 3) + 8 * (i >> 2) > lim) st[g][i] = -INFINITY;
                }
            }
            if (SUMS) {
#pragma unroll
                for (int g = 0; g < 2; ++g) {
                    const float zq = sd[g * 32 + r];
#pragma unroll
                    for (int i = 0; i < 16; ++i) acc[i] += __builtin_amdgcn_exp2f(st[g][i] - zq);
                }
                break;
            }
            if (take) {
                float mx = fmaxf(st[0][0], st[1][0]);
#pragma unroll
                for (int i = 1; i < 16; ++i) mx = fmaxf(mx, fmaxf(st[0][i], st[1][i]));
                const float mn = unset ? (mx == -INFINITY ? 0.f : mx) : fmaxf(m, mx);
                l *= unset ? 0.f : __builtin_amdgcn_exp2f(m - mn);
                unset = unset && mx == -INFINITY;
                pending = __builtin_amdgcn_ballot_w64(unset) != 0;
                m = mn;
#pragma unroll
                for (int g = 0; g < 2; ++g)
#pragma unroll
                    for (int i = 0; i < 16; ++i) st[g][i] -= mn;
            }
            float rs = 0.f;
#pragma unroll
            for (int g = 0; g < 2; ++g)
#pragma unroll
                for (int i = 0; i < 16; ++i) rs += __builtin_amdgcn_exp2f(st[g][i]);
            if (take || __builtin_amdgcn_ballot_w64(!(rs <= OVERFLOW_SUM)) == 0) {
                l += rs;
                break;
            }
        }
    }
    if (SUMS) {
        sum_over_queries(acc, r);
        if (GRP > 1) {
            float* js = reinterpret_cast<float*>(smem) + wave * 64 + lane;
            __syncthreads();                               // everyone has left the last tiles
            if (grp) js[(grp - 1) * 256] = acc[0];
            __syncthreads();
            if (grp) return;
#pragma unroll
            for (int g = 0; g < GRP - 1; ++g) acc[0] += js[g * 256];
        }
        const int key = s0 + (r & 3) + 8 * ((r & 15) >> 2) + 4 * h;
        if (r < 16 && key < p.Nk) {
            const int64_t at = (int64_t)b * p.wi_bs + (int64_t)head * p.wi_hs + key;
            p.w_out[(int64_t)b * p.wo_bs + (int64_t)head * p.wo_hs + key] = (p.w_in ? p.w_in[at] : 0.f) + acc[0];
        }
    } else {
        if (unset) m = -1.0e30f;                           // this lane half met no key
        if (GRP > 1) {
            float* js = reinterpret_cast<float*>(smem) + (wave * 64 + lane) * 2;
            __syncthreads();                               // everyone has left the last tiles
            if (grp) {
                js[(grp - 1) * 512] = m;
                js[(grp - 1) * 512 + 1] = l;
            }
            __syncthreads();
            if (grp) return;
#pragma unroll
            for (int g = 0; g < GRP - 1; ++g) {
                const float mg = js[g * 512], lg = js[g * 512 + 1], M = fmaxf(m, mg);
                l = l * __builtin_amdgcn_exp2f(m - M) + lg * __builtin_amdgcn_exp2f(mg - M);
                m = M;
            }
        }
        const float mo = __shfl_xor(m, 32, 64), lo = __shfl_xor(l, 32, 64);
        const float M = fmaxf(m, mo);
        const float sum = l * __builtin_amdgcn_exp2f(m - M) + lo * __builtin_amdgcn_exp2f(mo - M);
        if (h == 0 && s0 + r < p.Nq) {
            if (p.nch > 1) p.part[((int64_t)c * nbh + bh) * p.Nq + s0 + r] = make_float2(M, sum);
            else z[s0 + r] = sum == 0.f ? INFINITY : M + __log2f(sum);
        }
    }
}

// z of the queries whose keys went by chunks, in chunk order.
__global__ __launch_bounds__(256) void hk_key_weights_join_kernel(const KeyWeightParams p) {
    const int64_t n = (int64_t)p.B * p.H * p.Nq, i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    float M = -1.0e30f, sum = 0.f;
#pragma unroll 4
    for (int c = 0; c < p.nch; ++c) {
        const float2 x = p.part[c * n + i];
        const float N = fmaxf(M, x.x);
        sum = sum * __builtin_amdgcn_exp2f(M - N) + x.y * __builtin_amdgcn_exp2f(x.x - N);
        M = N;
    }
    p.z[i] = sum == 0.f ? INFINITY : M + __log2f(sum);
}

// Few keys: one launch, a workgroup per (sequence, head), no second pass over the products.  A wave takes 32 queries at a time and keeps their
// scores of ALL keys in registers (NB blocks of 32; S^T = K . Q^T as above), so the softmax is the plain one: maximum, exponentials, sum.
// K lies in LDS as the fragments that the matrix instruction takes.  A block's weights are added over its 32 queries by halving exchanges (as
// above) into the wave's own sums in LDS; the eight waves' sums are added in order at the end.
template <int HD, int NB, bool BIAS>
__global__ __launch_bounds__(512, 2) void hk_key_weights_few_kernel(const KeyWeightParams p) {
    constexpr int NKS = HD / 16, NW = 8;
    extern __shared__ __attribute__((aligned(16))) char smem[];      // fragments [NB][NKS][64 lanes] of 16 bytes, then sums [NW][NB * 32], biases [NB * 32]
    bf16x8* kl = reinterpret_cast<bf16x8*>(smem);
    float* sums = reinterpret_cast<float*>(smem + NB * NKS * 1024);
    float* bl = sums + NW * NB * 32;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r = lane & 31, h = lane >> 5;
    const int b = blockIdx.x / p.H, head = blockIdx.x - b * p.H;
    const int off = p.Nk - p.Nq, nkb = (p.Nk + 31) / 32, nqb = (p.Nq + 31) / 32;
    const __bf16* kp = p.K + (int64_t)b * p.bsk + head * HD + 8 * h;
    const __bf16* qp = p.Q + (int64_t)b * p.bsq + head * HD + 8 * h;
    bf16x8 qf[NKS];
    auto load_q = [&](int qb) {
        const __bf16* x = qp + (int64_t)min(qb * 32 + r, p.Nq - 1) * p.ldq;
#pragma unroll
        for (int s = 0; s < NKS; ++s) qf[s] = *reinterpret_cast<const bf16x8*>(x + 16 * s);
    };
    if (wave < nqb) load_q(nqb - 1 - wave);
    for (int g = wave; g < nkb; g += NW) {
        const __bf16* x = kp + (int64_t)min(g * 32 + r, p.Nk - 1) * p.ldk;
        bf16x8 kf[NKS];
#pragma unroll
        for (int s = 0; s < NKS; ++s) kf[s] = *reinterpret_cast<const bf16x8*>(x + 16 * s);
#pragma unroll
        for (int s = 0; s < NKS; ++s) kl[(g * NKS + s) * 64 + lane] = kf[s];
    }
    for (int j = tid; j < NW * NB * 32; j += NW * 64) sums[j] = 0.f;
    if (BIAS)
        for (int j = tid; j < nkb * 32; j += NW * 64) {
            const float v = p.bias[(int64_t)b * p.bias_bs + min(j, p.Nk - 1)];
            bl[j] = v <= REMOVED ? -INFINITY : v * HK_LOG2E;
        }
    __syncthreads();
    for (int u = 0; u * NW < nqb; ++u) {                   // causal: the longest blocks first, to and fro over the waves
        const int qb = nqb - 1 - (u * NW + (u & 1 ? NW - 1 - wave : wave));
        if (qb < 0) break;
        if (u) load_q(qb);
        const int q = qb * 32 + r, last = p.causal ? min(p.Nk - 1, q + off) : p.Nk - 1;      // the last key the lane's query sees
        const int gn = p.causal ? min(nkb, (qb * 32 + 31 + off) / 32 + 1) : nkb;
        const int clear = p.causal ? min(p.Nk - 1, qb * 32 + off) : p.Nk - 1;                // keys up to here every query of the block sees
        f32x16 st[NB];
        float mx = -INFINITY;
#pragma unroll
        for (int g0 = 0; g0 < NB; g0 += 2)
            if (g0 < gn) {                                 // two blocks: independent chains (one behind the keys: its scores are masked, all of them)
#pragma unroll
                for (int g = g0; g < g0 + 2; ++g)
#pragma unroll
                    for (int i = 0; i < 16; ++i) st[g][i] = 0.f;
#pragma unroll
                for (int s = 0; s < NKS; ++s)
#pragma unroll
                    for (int g = g0; g < g0 + 2; ++g)
                        st[g] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kl[(g * NKS + s) * 64 + lane], qf[s], st[g], 0, 0, 0);
#pragma unroll
                for (int g = g0; g < g0 + 2; ++g) {
                    if (BIAS) {
#pragma unroll
                        for (int x = 0; x < 4; ++x) {      // register 4 x + j <-> key 32 g + 8 x + 4 h + j
                            const f32x4 v = *reinterpret_cast<const f32x4*>(bl + g * 32 + 8 * x + 4 * h);
#pragma unroll
                            for (int j = 0; j < 4; ++j) st[g][4 * x + j] = v[j] == -INFINITY ? -INFINITY : st[g][4 * x + j] + v[j];
                        }
                    }
                    if (g * 32 + 31 > clear) {
                        const int lim = last - g * 32 - 4 * h;
#pragma unroll
                        for (int i = 0; i < 16; ++i)
                            if ((i & 3) + 8 * (i >> 2) > lim) st[g][i] = -INFINITY;
                    }
#pragma unroll
                    for (int i = 0; i < 16; ++i) mx = fmaxf(mx, st[g][i]);
                }
            }
        mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
        if (mx == -INFINITY) mx = 0.f;                     // no key: every exponential is 0
        float l = 0.f;
#pragma unroll
        for (int g0 = 0; g0 < NB; g0 += 2)
            if (g0 < gn) {
                float x[2] = {0.f, 0.f};
#pragma unroll
                for (int i = 0; i < 16; ++i)
#pragma unroll
                    for (int g = 0; g < 2; ++g) {
                        st[g0 + g][i] = __builtin_amdgcn_exp2f(st[g0 + g][i] - mx);
                        x[g] += st[g0 + g][i];
                    }
                l += x[0] + x[1];
            }
        l += __shfl_xor(l, 32, 64);
        float inv = l > 0.f ? 1.0f / l : (l == 0.f ? 0.f : l);       // NaN stays
        if (q >= p.Nq) inv = 0.f;
#pragma unroll
        for (int g = 0; g < NB; ++g)
            if (g < gn) {
                float a[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) a[i] = st[g][i] * inv;
                sum_over_queries(a, r);
                if (r < 16) sums[wave * NB * 32 + g * 32 + (r & 3) + 8 * (r >> 2) + 4 * h] += a[0];
            }
    }
    __syncthreads();
    const float* wi = p.w_in ? p.w_in + (int64_t)b * p.wi_bs + (int64_t)head * p.wi_hs : nullptr;
    float* wo = p.w_out + (int64_t)b * p.wo_bs + (int64_t)head * p.wo_hs;
    for (int j = tid; j < p.Nk; j += NW * 64) {
        float x = 0.f;
#pragma unroll
        for (int w = 0; w < NW; ++w) x += sums[w * NB * 32 + j];
        wo[j] = (wi ? wi[j] : 0.f) + x;
    }
}

// STATS of few queries over many keys: chunks of the keys, a workgroup per CU, four tiles at least.  The last 32 / 512 of so many tokens,
// 32 heads of 128, without : with chunks (us, all launches): 1000 17.0 : 13.0, 23.8 : 21.7; 2047 27.5 : 15.2, 37.9 : 31.0; 16000 170 : 52, 219 : 164;
// 4 sequences of 16000 285 : 231 (K is read twice: 216), 665 : 670.  Twice as many chunks: 16000 tokens 57 and 169; eight tiles at least: 1000 tokens 14.8.
int key_chunks(int64_t blocks, int Nk, int* ct) {
    const int tiles = (Nk + TILE - 1) / TILE;
    int64_t n = 256 / blocks < tiles / 4 ? 256 / blocks : tiles / 4;
    if (n < 1) n = 1;
    *ct = (int)((tiles + n - 1) / n);
    return (tiles + *ct - 1) / *ct;
}
// hk_key_weights_few_kernel or two launches?  The former as long as its waves have up to 12 blocks of 32 x 32 products each.  Few : two, 32 heads of 128
// (us): prompts of 20 / 65 / 128 / 256 / 352 tokens 4.2 : 7.6, 5.6 : 9.9, 6.5 : 10.2, 10.5 : 13.6, 14.6 : 15.8, 32 of them 7 : 13, 13 : 20, 17 : 28, 44 : 57,
// 61 : 88; without a diagonal, 128 keys and 400 / 800 / 1600 queries 9.9 : 13.3, 15.6 : 16.6, 23.4 : 24.5, 256 keys and 200 / 400 11.5 : 13.5, 17.0 : 15.3,
// 384 keys and 200 15.3 : 14.6; heads of 64, 256 keys and 400 14.2 : 11.9.
bool few_keys(int64_t Nq, int64_t Nk, bool causal) {
    const int64_t nqb = (Nq + 31) / 32, nkb = (Nk + 31) / 32;
    return Nk <= 384 && nqb * nkb - (causal ? nqb * (nqb - 1) / 2 : 0) <= 96;
}
// Whole multiples of 64 bytes: the sums of a few rows could otherwise come to HK_NO_WS, which says that there are none.
size_t key_weights_bytes(int64_t B, int64_t H, int64_t Nq, int Nk, bool causal) {
    static_assert(HK_NO_WS % 64 != 0, "a workspace's size must not be the value that stands for none");
    if (few_keys(Nq, Nk, causal)) return HK_NO_WS;
    int ct;
    const int nch = key_chunks((Nq + BLK - 1) / BLK * B * H, Nk, &ct);
    return ((size_t)(B * H * Nq) * (nch > 1 ? 8 * nch + 4 : 4) + 63) / 64 * 64;
}

template <int HD, bool SUMS, bool BIAS, int GRP>
int launch_groups(const KeyWeightParams& p, hipStream_t s) {
    constexpr int LDS = GRP * NST * (TILE * HD * 2 + 4 * TILE * 4);
    static std::atomic<unsigned long long> attr_done{0};   // per device
    const hipError_t e = hk_lds_attr_once(attr_done, reinterpret_cast<const void*>(&hk_key_weights_kernel<HD, SUMS, BIAS, GRP>), LDS);
    if (e != hipSuccess) {
        hk_set_error("hk_attn_key_weights_bf16: hipFuncSetAttribute(%d B LDS): %s", LDS, hipGetErrorString(e));
        return HK_ELAUNCH;
    }
    hipLaunchKernelGGL((hk_key_weights_kernel<HD, SUMS, BIAS, GRP>), dim3((unsigned)((int64_t)p.nblk * p.B * p.H * (SUMS ? 1 : p.nch))),
                       dim3(GRP * 256), LDS, s, p);
    return HK_OK;
}
template <int HD, bool SUMS, bool BIAS>
int launch_key_weights(KeyWeightParams p, hipStream_t s) {
    p.nblk = ((SUMS ? p.Nk : p.Nq) + BLK - 1) / BLK;
    // A second group where it finds CUs idle and tiles enough.  One : two groups, both launches, heads of 128 (us at so many blocks): 65 rows (32
    // blocks) 10.0 : 10.1, 128 (32) 10.2 : 11.0, 200 (64) 13.7 : 13.4, 352 (96) 17.0 : 15.7, 1000 (256) 34.4 : 28.0, 2047 (128) 59.9 : 45.1;
    // 352 (384) 18.7 : 20.3, 500 (512) 23.7 : 25.7, 700 (384) 27.9 : 27.1, 1500 (384) 49.9 : 41.0, 2047 (512) 65.2 : 57.9; 700 (768) 33 : 43.
    const int64_t blocks = (int64_t)p.nblk * p.B * p.H * (SUMS ? 1 : p.nch), n_pass = SUMS ? p.Nq : p.nch > 1 ? p.ct * TILE : p.Nk;
    const bool two = blocks <= 256 ? n_pass > 2 * TILE : blocks <= 512 && n_pass > 10 * TILE;
    return two ? launch_groups<HD, SUMS, BIAS, 2>(p, s) : launch_groups<HD, SUMS, BIAS, 1>(p, s);
}
template <int HD, int NB, bool BIAS>
int launch_few(const KeyWeightParams& p, hipStream_t s) {
    constexpr int LDS = NB * 32 * (HD * 2 + 9 * 4);
    static std::atomic<unsigned long long> attr_done{0};   // per device
    const hipError_t e = hk_lds_attr_once(attr_done, reinterpret_cast<const void*>(&hk_key_weights_few_kernel<HD, NB, BIAS>), LDS);
    if (e != hipSuccess) {
        hk_set_error("hk_attn_key_weights_bf16: hipFuncSetAttribute(%d B LDS): %s", LDS, hipGetErrorString(e));
        return HK_ELAUNCH;
    }
    hipLaunchKernelGGL((hk_key_weights_few_kernel<HD, NB, BIAS>), dim3((unsigned)(p.B * p.H)), dim3(512), LDS, s, p);
    return HK_OK;
}
template <int HD>
int launch_both(const KeyWeightParams& p, hipStream_t s) {
    if (few_keys(p.Nq, p.Nk, p.causal)) {
        if (p.Nk <= 128) return p.bias ? launch_few<HD, 4, true>(p, s) : launch_few<HD, 4, false>(p, s);
        if (p.Nk <= 256) return p.bias ? launch_few<HD, 8, true>(p, s) : launch_few<HD, 8, false>(p, s);
        return p.bias ? launch_few<HD, 12, true>(p, s) : launch_few<HD, 12, false>(p, s);
    }
    const int rc = p.bias ? launch_key_weights<HD, false, true>(p, s) : launch_key_weights<HD, false, false>(p, s);
    if (rc != HK_OK) return rc;
    if (p.nch > 1) hipLaunchKernelGGL(hk_key_weights_join_kernel, dim3((unsigned)(((int64_t)p.B * p.H * p.Nq + 255) / 256)), dim3(256), 0, s, p);
    return p.bias ? launch_key_weights<HD, true, true>(p, s) : launch_key_weights<HD, true, false>(p, s);
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
constexpr int REG_KEYS = 16 * 1024;  // keys per (sequence, head) up to which a workgroup keeps all ranks in registers

// fp32 -> a whole number that orders like it: removed < NaN < -inf < ... < -0 = 0 < ... < inf < recent
__device__ __forceinline__ uint32_t rank_of(float w, bool removed, bool recent) {
    const uint32_t u = __builtin_bit_cast(uint32_t, w + 0.f);
    uint32_t k = (u >> 31) ? ~u : u | 0x80000000u;
    if (w != w) k = 1u;
    if (removed) k = 0u;
    return recent ? 0xffffffffu : k;
}

// Kept rows within one (sequence, head), walked upwards by a workgroup of T threads.  Row `at` comes from src(at) >= at, so a step's stores
// can only hit sources of the same or an earlier step: all of a step's loads have arrived before its first store.  Not in place: copied.
// (W of the head's HD values, from w0 on: what different workgroups move does not meet.)
template <int HD, int T, int W, typename Src>
__device__ __forceinline__ void move_rows(const EvictParams& p, int b, int head, bool is_v, int w0, Src src) {
    constexpr int CH = W / 8, RPS = T / CH, U = 8;
    const int col = head * HD + w0 + ((int)threadIdx.x % CH) * 8, g = threadIdx.x / CH;
    const __bf16* from = is_v ? p.V + (int64_t)b * p.bsv + col : p.K + (int64_t)b * p.bsk + col;
    __bf16* to = is_v ? p.VO + (int64_t)b * p.bsvo + col : p.KO + (int64_t)b * p.bsko + col;
    const int64_t ldf = is_v ? p.ldv : p.ldk, ldt = is_v ? p.ldvo : p.ldko;
    for (int r0 = 0; r0 < p.budget; r0 += RPS * U) {
        u32x4 x[U];
        int s[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            s[u] = src(min(r0 + u * RPS + g, p.budget - 1));
            x[u] = *reinterpret_cast<const u32x4*>(from + (int64_t)s[u] * ldf);
        }
        if (p.in_place) {
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __syncthreads();
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int at = r0 + u * RPS + g;
            if (at < p.budget && !(p.in_place && s[u] == at)) *reinterpret_cast<u32x4*>(to + (int64_t)at * ldt) = x[u];
        }
    }
}

// One workgroup per (sequence, head), every rank in a register (key u * T + thread in slot u).  The budget-th largest rank is found bit by
// bit: count the ranks at or above the candidate (a comparison, a ballot and a bit count per slot; the waves add up through LDS), keep the
// bit if there are enough; done as soon as there are exactly enough.  An ordered pass then keeps the ranks above the threshold and, of those
// equal to it, the first ones: positions from a scan over the (slot, wave) counts.  Weights and biases move through registers (in place is
// safe), and MOVE moves K and V in the same launch.  Bound by latency without it (512 pairs of 2047 keys 10-15 us), by the moved rows with it.
template <int T, int KPT, int HD, bool MOVE>
__global__ __launch_bounds__(T) void hk_evict_kernel(const EvictParams p) {
    constexpr int NW = T / 64, NC = KPT * NW;              // (slot, wave) pairs
    static_assert(NC <= 256, "one wave scans four counts per lane");
    __shared__ uint32_t part[2][NW];
    __shared__ uint32_t cnt[NC];
    extern __shared__ uint16_t rows[];                     // MOVE: [budget] the kept rows
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int b = blockIdx.x / p.H, head = blockIdx.x - b * p.H;
    const float* w = p.w + (int64_t)b * p.w_bs + (int64_t)head * p.w_hs;
    const float* bias = p.bias ? p.bias + (int64_t)b * p.b_bs + (int64_t)head * p.b_hs : nullptr;
    float* wo = p.w_out + (int64_t)b * p.wo_bs + (int64_t)head * p.wo_hs;
    float* bo = p.bias ? p.bias_out + (int64_t)b * p.bo_bs + (int64_t)head * p.bo_hs : nullptr;
    int32_t* kept = p.kept + (int64_t)blockIdx.x * p.budget;
    float wv[KPT], bv[KPT];
    uint32_t k[KPT];
#pragma unroll
    for (int u = 0; u < KPT; ++u) {
        const int j = min(u * T + tid, p.n - 1);
        wv[u] = w[j];
        bv[u] = bias ? bias[j] : 0.f;
    }
#pragma unroll
    for (int u = 0; u < KPT; ++u) {
        const int j = u * T + tid;
        k[u] = rank_of(wv[u], bv[u] <= REMOVED, j >= p.n - p.recent);
        if (j >= p.n) k[u] = 0u;                           // behind the last key: never counted (candidates are above 0), never kept
    }
    const uint32_t want = (uint32_t)p.budget;
    uint32_t thr = 0;                                      // the largest value that at least `want` ranks reach, so far
    bool exact = false;
    for (int bit = 31; bit >= 0 && !exact; --bit) {
        const uint32_t cand = thr | (1u << bit);
        uint32_t c = 0;
#pragma unroll
        for (int u = 0; u < KPT; ++u) c += (uint32_t)__popcll(__builtin_amdgcn_ballot_w64(k[u] >= cand));
        if (lane == 0) part[bit & 1][wave] = c;            // two turns: the next round's counts do not meet this round's readers
        __syncthreads();
        c = 0;
#pragma unroll
        for (int x = 0; x < NW; ++x) c += part[bit & 1][x];
        if (c >= want) thr = cand;
        exact = c == want;
    }
    // ranks above thr - all of them are kept - and those equal to it, of which the first `want - above` are
    uint64_t ga[KPT], ge[KPT];
#pragma unroll
    for (int u = 0; u < KPT; ++u) {
        const bool in = u * T + tid < p.n;
        ga[u] = __builtin_amdgcn_ballot_w64(in && k[u] > thr);
        ge[u] = __builtin_amdgcn_ballot_w64(in && k[u] == thr);
        if (lane == 0) cnt[u * NW + wave] = (uint32_t)__popcll(ga[u]) | (uint32_t)__popcll(ge[u]) << 16;   // at most 2^14 of each in all
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");       // every weight and bias is in a register before any is stored
    __syncthreads();
    if (wave == 0) {
        constexpr int CPL = (NC + 63) / 64;
        uint32_t c[CPL], s = 0;
#pragma unroll
        for (int i = 0; i < CPL; ++i) {
            c[i] = lane * CPL + i < NC ? cnt[lane * CPL + i] : 0u;
            s += c[i];
        }
        uint32_t before = s;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const uint32_t x = __shfl_up(before, o, 64);
            if (lane >= o) before += x;
        }
        if (lane == 63) part[0][0] = before & 0xffffu;     // ranks above thr in all
        before -= s;
#pragma unroll
        for (int i = 0; i < CPL; ++i) {
            if (lane * CPL + i < NC) cnt[lane * CPL + i] = before;
            before += c[i];
        }
    }
    __syncthreads();
    const uint32_t ties = want - part[0][0];
    const uint64_t lower = (1ull << lane) - 1;
#pragma unroll
    for (int u = 0; u < KPT; ++u) {
        const int j = u * T + tid;
        const uint32_t base = cnt[u * NW + wave];
        const uint32_t ba = (base & 0xffffu) + (uint32_t)__popcll(ga[u] & lower), be = (base >> 16) + (uint32_t)__popcll(ge[u] & lower);
        if (j < p.n && (k[u] > thr || (k[u] == thr && be < ties))) {
            const uint32_t at = ba + min(be, ties);
            kept[at] = j;
            wo[at] = wv[u];
            if (bo) bo[at] = bv[u];
            if (MOVE) rows[at] = (uint16_t)j;
        }
    }
    if (p.in_place)                                        // the places that became free: nothing collected, nothing removed
        for (int j = p.budget + tid; j < p.n; j += T) {
            wo[j] = 0.f;
            if (bo) bo[j] = 0.f;
        }
    if (MOVE) {
        __syncthreads();
        auto src = [&](int at) { return (int)rows[at]; };
        move_rows<HD, T, HD>(p, b, head, false, 0, src);
        move_rows<HD, T, HD>(p, b, head, true, 0, src);
    }
}

// More keys than registers hold: the budget-th largest rank by four rounds of an 8-bit histogram over the weights in memory, then the ordered
// pass chunk by chunk (a chunk's values are in registers before any of its stores, and go to places at or below the ones they came from).
// Bound by the passes' waits for memory: 40000 keys 77 us (one rank in flight per thread and 1024 keys per ordered step: 118).
__global__ __launch_bounds__(SEL_T) void hk_evict_select_kernel(const EvictParams p) {
    constexpr int U = 8;                                   // ranks in flight per thread: one at a time, the passes wait for memory
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
    uint32_t prefix = 0, want = (uint32_t)p.budget;        // the want-th largest of the ranks that begin with prefix
    for (int shift = 24; shift >= 0; shift -= 8) {
        if (tid < 256) hist[tid] = 0;
        __syncthreads();
        for (int j0 = tid; j0 < p.n; j0 += SEL_T * U) {
            uint32_t k[U];
#pragma unroll
            for (int u = 0; u < U; ++u) k[u] = rank_at(min(j0 + u * SEL_T, p.n - 1));
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const bool in = j0 + u * SEL_T < p.n && (shift == 24 || (k[u] >> (shift + 8)) == prefix);
                const uint32_t bin = (k[u] >> shift) & 255u;
                // a wave's ranks often begin alike: the first lane's bin is counted once for all lanes that share it
                const uint64_t any = __builtin_amdgcn_ballot_w64(in);
                if (any == 0) continue;
                const int lead = __ffsll((unsigned long long)any) - 1;
                const uint32_t b0 = __builtin_amdgcn_readlane(bin, lead);
                const uint64_t same = __builtin_amdgcn_ballot_w64(in && bin == b0);
                if (lane == lead) atomicAdd(&hist[b0], (uint32_t)__popcll(same));
                else if (in && bin != b0) atomicAdd(&hist[bin], 1u);
            }
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
    constexpr int W = 4;                                   // consecutive keys per thread and step
    for (int j0 = 0; j0 < p.n; j0 += SEL_T * W) {
        uint32_t k[W], c = 0;
        float wv[W], bv[W];
#pragma unroll
        for (int i = 0; i < W; ++i) {
            const int j = min(j0 + tid * W + i, p.n - 1);
            wv[i] = w[j];
            bv[i] = bias ? bias[j] : 0.f;
        }
#pragma unroll
        for (int i = 0; i < W; ++i) {
            const int j = j0 + tid * W + i;
            k[i] = rank_of(wv[i], bias && bv[i] <= REMOVED, j >= p.n - p.recent);
            if (j < p.n) c += (k[i] > prefix ? 1u : 0u) + (k[i] == prefix ? 1u << 16 : 0u);
        }
        uint32_t x = c;                                    // above | equal << 16, of the lanes up to this one
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const uint32_t y = __shfl_up(x, o, 64);
            if (lane >= o) x += y;
        }
        if (lane == 63) wsum[wave] = x;
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // wv, bv are in registers before anyone stores
        __syncthreads();
        uint32_t ba = above + ((x - c) & 0xffffu), be = equal + ((x - c) >> 16);
        for (int v = 0; v < SEL_T / 64; ++v) {
            const uint32_t s = wsum[v];
            if (v < wave) {
                ba += s & 0xffffu;
                be += s >> 16;
            }
            above += s & 0xffffu;
            equal += s >> 16;
        }
#pragma unroll
        for (int i = 0; i < W; ++i) {
            const int j = j0 + tid * W + i;
            const bool gt = j < p.n && k[i] > prefix, eq = j < p.n && k[i] == prefix;
            if (gt || (eq && be < want)) {
                const uint32_t at = ba + min(be, want);
                kept[at] = j;
                wo[at] = wv[i];
                if (bo) bo[at] = bv[i];
            }
            ba += gt;
            be += eq;
        }
        __syncthreads();
    }
    if (p.in_place)
        for (int j = p.budget + tid; j < p.n; j += SEL_T) {
            wo[j] = 0.f;
            if (bo) bo[j] = 0.f;
        }
}

// Rows into another cache: 16 bytes of K and of V per thread and step, neighbouring heads of one destination row next to each other, so
// that whole destination rows are written; the source rows are HD * 2 byte pieces.  16384 rows of 8 KB, K and V: 99 us, 5.4 TB/s read and written.
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

// Rows within the cache, the kept list in memory: a workgroup per (sequence, head, K or V, W values of the head).
template <int HD, int W>
__global__ __launch_bounds__(512) void hk_evict_move_kernel(const EvictParams p) {
    constexpr int N = HD / W;
    const int bh = blockIdx.x / (2 * N), part = blockIdx.x % (2 * N), b = bh / p.H, head = bh - b * p.H;
    const int32_t* kept = p.kept + (int64_t)bh * p.budget;
    move_rows<HD, 512, W>(p, b, head, part & 1, (part >> 1) * W, [&](int at) { return kept[at]; });
}

template <int T, int KPT, int HD, bool MOVE>
int launch_evict(const EvictParams& p, hipStream_t s) {
    hipLaunchKernelGGL((hk_evict_kernel<T, KPT, HD, MOVE>), dim3((unsigned)(p.B * p.H)), dim3(T), MOVE ? (size_t)p.budget * 2 : 0, s, p);
    return HK_OK;
}
template <int HD, bool MOVE>
int launch_evict_any(const EvictParams& p, hipStream_t s) {
    if constexpr (MOVE || HD == 128)       // (heads of 64 move so few rows in the same launch, always)
        if (p.n <= 512) return launch_evict<256, 2, HD, MOVE>(p, s);
    // moving rows wants more in flight than selecting them: 500 of 1000 keys, 256 : 512 threads 11.9 : 8.9 us (32 pairs, in place), 20.1 : 17.3 (128 pairs)
    if (p.n <= 2048) return launch_evict<MOVE ? 512 : 256, MOVE ? 4 : 8, HD, MOVE>(p, s);
    if (p.n <= 4096) return launch_evict<512, 8, HD, MOVE>(p, s);
    return launch_evict<1024, 16, HD, MOVE>(p, s);
}
template <int HD>
int launch_evict_all(const EvictParams& p, hipStream_t s) {
    const unsigned pairs = (unsigned)(p.B * p.H);
    // One launch or two?  A workgroup per pair moves its rows in pieces of one head; the copy kernel writes whole rows with the whole chip
    // (5.5 TB/s against 4.6) and costs a launch (2.6 us of the host's).  One : two, heads of 128 (us).  Budget 256 of 353: 9.5 : 9.2 (32 pairs),
    // 11.3 : 12.1 (128), 24.5 : 28.5 (512); 500 of 1000: 15.7 : 11.7, 20.0 : 20.0, 51.3 : 52.7; 1024 of 2047: 26 : 15, 31 : 31, 118 : 113; 8000 of
    // 16000: 200 : 66, 312 : 217.  Heads of 64, 1024 of 2047: 17 : 13 (32 pairs), 28 : 32 (256), 60 : 59 (512).
    const int64_t bytes = (int64_t)p.budget * HD * 2;
    const bool one = bytes <= (pairs < 128 ? 64 << 10 : 128 << 10);
    // In place, rows may only move within what one workgroup walks, but slices of the head's values are apart: few pairs spread over the CUs by
    // slices of 32, and many lose by their 64-byte pieces.  One : two launches, 1024 of 2047 rows 14.0 : 12.7 (32 pairs), 18.1 : 21.2 (64), 23.5 : 33.4 (128);
    // 8000 of 16000 97 : 63 (32), 201 : 253 (128); 500 of 1000 8.9 : 8.2 (32).
    const bool sliced = pairs <= 32;
    if (p.n <= REG_KEYS && (p.in_place ? one || !sliced : one)) return launch_evict_any<HD, true>(p, s);
    if (p.n <= REG_KEYS) launch_evict_any<HD, false>(p, s);
    else hipLaunchKernelGGL(hk_evict_select_kernel, dim3(pairs), dim3(SEL_T), 0, s, p);
    if (p.in_place) {
        if (sliced) hipLaunchKernelGGL((hk_evict_move_kernel<HD, 32>), dim3(pairs * 2 * (HD / 32)), dim3(512), 0, s, p);
        else hipLaunchKernelGGL((hk_evict_move_kernel<HD, HD>), dim3(pairs * 2), dim3(512), 0, s, p);
    } else {
        const int64_t pieces = (int64_t)p.B * p.H * p.budget, per = 256 / (HD / 8) * 2;
        HK_REQUIRE((pieces + per - 1) / per < (1LL << 31), "hk_cache_evict_bf16: grid too large");
        hipLaunchKernelGGL((hk_evict_copy_kernel<HD>), dim3((unsigned)((pieces + per - 1) / per)), dim3(256), 0, s, p);
    }
    return HK_OK;
}

}  // namespace

extern "C" size_t hk_attn_key_weights_ws(int32_t B, int32_t H, int32_t Nq, int32_t Nk, int32_t causal) {
    if (B < 1 || B >= 65536 || H < 1 || H >= 65536 || Nq < 1 || Nk < 1 || Nq >= (1 << 26) || Nk >= (1 << 26) || (causal && Nk < Nq)) return 0;
    return key_weights_bytes(B, H, Nq, Nk, causal != 0);
}

extern "C" int hk_attn_key_weights_bf16(const hk_key_weights_desc* d, void* stream) {
    HK_REQUIRE(d && d->Q && d->K && d->w_out, "hk_attn_key_weights_bf16: null operand");
    HK_REQUIRE(d->B >= 1 && d->B < 65536 && d->H >= 1 && d->H < 65536 && d->Nq >= 1 && d->Nk >= 1 && d->Nq < (1 << 26) && d->Nk < (1 << 26) &&
                   (d->head_dim == 64 || d->head_dim == 128) && (!d->causal || d->Nk >= d->Nq),
               "hk_attn_key_weights_bf16: bad shape B=%d H=%d Nq=%d Nk=%d head_dim=%d (head size 64 or 128, causal needs Nk >= Nq)", d->B, d->H,
               d->Nq, d->Nk, d->head_dim);
    HK_REQUIRE(((d->ldq | d->bsq | d->ldk | d->bsk) & 7) == 0 && d->ldq >= 0 && d->bsq >= 0 && d->ldk >= 0 && d->bsk >= 0,
               "hk_attn_key_weights_bf16: strides must be multiples of 8 elements, not negative");
    HK_REQUIRE(d->ldq < (1 << 25) && d->ldk < (1 << 25), "hk_attn_key_weights_bf16: token strides of 2^25 elements and more are not supported");
    HK_REQUIRE(((uintptr_t)d->Q | (uintptr_t)d->K | (uintptr_t)d->ws) % 16 == 0 &&
                   ((uintptr_t)d->key_bias | (uintptr_t)d->w_in | (uintptr_t)d->w_out) % 4 == 0,
               "hk_attn_key_weights_bf16: operands must be 16-byte aligned");
    HK_REQUIRE(hk_rows_apart(d->B, d->wo_bs, d->H, d->wo_hs, d->Nk) && d->wi_bs >= 0 && d->wi_hs >= 0 && d->bias_bs >= 0,
               "hk_attn_key_weights_bf16: rows of w_out must not overlap, strides must not be negative");
    HK_REQUIRE(d->w_in != d->w_out || (d->wi_bs == d->wo_bs && d->wi_hs == d->wo_hs),
               "hk_attn_key_weights_bf16: weights updated in place must have one layout");
    const size_t need = key_weights_bytes(d->B, d->H, d->Nq, d->Nk, d->causal != 0);
    const bool few = few_keys(d->Nq, d->Nk, d->causal != 0);
    HK_REQUIRE(few || (d->ws && d->ws_bytes >= need), "hk_attn_key_weights_bf16: workspace of %zu bytes, %zu needed (hk_attn_key_weights_ws)",
               d->ws ? d->ws_bytes : (size_t)0, need);
    {
        const int64_t row = (int64_t)d->H * d->head_dim;
        const HkSpan wo = hk_span(d->w_out, d->B, d->wo_bs, d->H, d->wo_hs, d->Nk, 4), w = hk_span(few ? nullptr : d->ws, 1, 0, 1, 0, (int64_t)need, 1);
        const HkSpan in[] = {hk_span(d->Q, d->B, d->bsq, d->Nq, d->ldq, row, 2), hk_span(d->K, d->B, d->bsk, d->Nk, d->ldk, row, 2),
                             hk_span(d->key_bias, d->B, d->bias_bs, 1, 0, d->Nk, 4),
                             d->w_in == d->w_out ? HkSpan{} : hk_span(d->w_in, d->B, d->wi_bs, d->H, d->wi_hs, d->Nk, 4)};
        for (int i = 0; i < 4; ++i)
            HK_REQUIRE(!hk_overlap(wo, in[i]) && !hk_overlap(w, in[i]), "hk_attn_key_weights_bf16: the output or the workspace overlaps an input");
        HK_REQUIRE(!hk_overlap(wo, w), "hk_attn_key_weights_bf16: the output overlaps the workspace");
    }
    const int64_t most = ((d->Nq > d->Nk ? d->Nq : d->Nk) + BLK - 1) / BLK;      // (chunks only where that leaves few workgroups)
    HK_REQUIRE(most * d->B * d->H < (1LL << 31) && (int64_t)d->B * d->H * d->Nq < (1LL << 38), "hk_attn_key_weights_bf16: grid too large");
    KeyWeightParams p = {};
    p.Q = reinterpret_cast<const __bf16*>(d->Q);
    p.K = reinterpret_cast<const __bf16*>(d->K);
    p.bias = d->key_bias;
    p.nch = key_chunks(((int64_t)d->Nq + BLK - 1) / BLK * d->B * d->H, d->Nk, &p.ct);
    p.part = reinterpret_cast<float2*>(d->ws);             // z behind it (8-byte aligned)
    p.z = reinterpret_cast<float*>(d->ws) + (p.nch > 1 ? (int64_t)2 * p.nch * d->B * d->H * d->Nq : 0);
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
    const int rc = d->head_dim == 128 ? launch_both<128>(p, s) : launch_both<64>(p, s);
    if (rc != HK_OK) return rc;
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
    const int64_t wlen = in_place ? d->n_keys : d->budget;       // in place, what one sequence writes another must not read either
    HK_REQUIRE(hk_rows_apart(d->B, d->bsko, wlen, d->ldko, row) && hk_rows_apart(d->B, d->bsvo, wlen, d->ldvo, row),
               "hk_cache_evict_bf16: output rows must not overlap");
    HK_REQUIRE(hk_rows_apart(d->B, d->wo_bs, d->H, d->wo_hs, wlen) && (d->key_bias == nullptr || hk_rows_apart(d->B, d->bo_bs, d->H, d->bo_hs, wlen)),
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
    const int rc = d->head_dim == 128 ? launch_evict_all<128>(p, s) : launch_evict_all<64>(p, s);
    if (rc != HK_OK) return rc;
    HK_CHECK_LAUNCH("hk_cache_evict_bf16");
    return HK_OK;
}
