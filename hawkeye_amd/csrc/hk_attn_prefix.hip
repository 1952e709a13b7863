// Attention of a batch whose sequences share one prefix, and the decode step that adds its softmax weights to what the keys
// have collected.  Both are bound by reading K and V: the prefix's rows are read once for ALL rows of the batch.
//
//   s_j = q . k_j (+ bias_j log2 e),  p_j = 2^(s_j - M),  o = sum_j p_j v_j / sum_j p_j
//
// over the prefix's keys and the row's own; softmax sums are associative, so the keys are cut into chunks, a chunk leaves
// (m, l, o) = (its maximum, sum_j 2^(s_j - m), sum_j 2^(s_j - m) v_j) in 32 bits, and a second launch joins the chunks of a
// row.  Tiles go to waves, and chunks to groups of threads, in turn; every sum's order follows from the sizes alone (bit-reproducible).
//
// hk_prefix_part_kernel: a workgroup = one (head, key chunk, group of query rows).  Prefix chunks take rows of ALL
// sequences (row r = sequence r / Nq, token r % Nq), a sequence's own chunks take its Nq rows.  Its four waves walk 32-key tiles
// of the chunk, each for itself:
//   S^T = K . Q^T  (v_mfma_f32_16x16x32_bf16: 16 keys x 16 rows; lane -> row lane & 15, keys 4 (lane >> 4) + i)
//   O^T += V^T . P^T, where the S^T accumulators of two 16-key blocks ARE the B operand (contraction index 8 q + j <-> key
//   4 q + j of block 0, j < 4, or 4 q + j - 4 of block 1), and V^T comes in that key order from ds_read_b64_tr_b16.
// K goes from memory straight to the A operand's registers, V through 32 keys of LDS that belong to the wave (no barrier in
// the loop).  The next tile's K is requested as soon as this one's scores stand, its V as soon as this one's is in LDS: a
// wave keeps about 16 KB in flight, 8 waves per CU.  Bound by memory: 16 sequences' step over 1500 own keys each (398 MB) 80 us, 5.0 TB/s;
// 64 sequences' over 333 own keys each beside the prefix (350 MB) 67 us.
// Many sequences with few own keys each: a wave takes a sequence's keys alone (by_wave).
// ONE: a workgroup of eight waves per (sequence, head) for all its keys, the prefix's tiles first; no chunks, no second launch, a step's scores
// stay in LDS.  Bound by latency (a chain of dependent tiles per wave): one sequence over 353 keys 7.7 us, and the host needs 10 for the call.
#include <type_traits>
#include "hk_common.h"
#include "hk_overlap.h"

namespace {

constexpr float REMOVED = -1.0e4f;   // a key whose bias is at or below this does not exist (the framework's mask value)
constexpr float M_NONE = -1.0e30f;   // running maximum of a row that has met no key
constexpr int TK = 32;               // keys per tile
constexpr int NWV = 4;               // waves per workgroup
constexpr int MAX_CHUNK = 1024;      // keys per chunk at most: the chunk's bias lives in LDS
// Workgroups the chunks are cut for.  256 / 512 / 1024 / 2048 measured within 2 % of each other for shared prefixes, 91 / 91 / 80 / 79 us for 16
// sequences' own 1500 keys.  128-row blocks (one per CU) want as many as there are CUs: see cut_rows.
constexpr int PART_WANT = 1024, ROWS_WANT = 256;

struct PrefixParams {
    const __bf16 *Q, *KP, *VP, *K, *V;
    __bf16* O;
    const float* bias;               // own keys: bias[b * bias_bs + h * bias_hs + j]
    float* part_o;                   // [row][head][slot][HD]
    float* part_ml;                  // [row][head][slot][2]
    float* raw;                      // WEIGHTS: scores [B][H][raw_ld], raw_ld = Nk rounded up to whole tiles
    int B, H, Nq, P, Nk, R;          // R = B * Nq
    int64_t ldq, bsq, ldkp, ldvp, ldk, bsk, ldv, bsv, ldo, bso, bias_bs, bias_hs, raw_ld;
    int pc, npc, nprg;               // prefix: keys per chunk, chunks, row groups
    int oc, noc, norg;               // own keys: the same, per sequence
    int ns;                          // slots of a row: npc + noc
    int by_wave;                     // own keys: a (sequence, head, row group) per wave instead of per workgroup (noc = 1)
    int64_t pjobs;                   // workgroups of the prefix: H * npc * nprg (below 2^31 once checked)
};

__device__ __forceinline__ void wave_lds_sync() {   // LDS written by this wave's lanes is read by its other lanes
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

__device__ __forceinline__ float inverse_sum(float l) { return l > 0.f ? 1.0f / l : (l == 0.f ? 0.f : l); }     // no key: 0; NaN stays

// A decode step's weights: w_out[j] = w_in[j] + 2^(s_j - M) / l from its scores.
struct StepWeights {
    const float* w_in;               // may be w_out; NULL = zeros
    float* w_out;
    int64_t wi_bs, wi_hs, wo_bs, wo_hs;
};
__device__ __forceinline__ void add_weights(const PrefixParams& p, const StepWeights& sw, int b, int head, const float* raw, float M, float inv,
                                            int j0, int step) {
    const float* wi = sw.w_in ? sw.w_in + (int64_t)b * sw.wi_bs + (int64_t)head * sw.wi_hs : nullptr;
    float* wo = sw.w_out + (int64_t)b * sw.wo_bs + (int64_t)head * sw.wo_hs;
    for (int j = j0; j < p.Nk; j += step) wo[j] = (wi ? wi[j] : 0.f) + __builtin_amdgcn_exp2f(raw[j] - M) * inv;
}

// (Three waves per SIMD where the registers allow them without a spill: at two, 178 VGPRs, 16 sequences' step over 1985 + 61 keys takes 15.6 us, not 14.6.)
template <int HD, int RT, bool BIAS, bool RAW, int NW, bool ONE>
__global__ __launch_bounds__(NW * 64, HD == 128 && RT == 1 && !BIAS && !ONE ? 3 : 2) void hk_prefix_part_kernel(const PrefixParams p, const StepWeights sw) {
    constexpr int CH = HD / 8;            // 16-byte chunks per key row
    constexpr int KS = HD / 32;           // contraction steps of S^T
    constexpr int DT = HD / 16;           // 16-dim blocks of O^T
    constexpr int RPL = 64 / CH;          // key rows one 64-lane load covers
    constexpr int NL = TK / RPL;          // loads per lane for a tile of V
    constexpr int VB = TK * HD * 2;       // bytes of a wave's V tile
    constexpr int OB = RT * 16 * HD * 4;  // bytes of a wave's O block at the end
    constexpr int WB = VB > OB ? VB : OB;
    __shared__ __attribute__((aligned(16))) char vlds[NW * WB];
    __shared__ float ml[NW][RT * 16][2];
    __shared__ __attribute__((aligned(16))) float blds[BIAS ? MAX_CHUNK : 4];
    __shared__ __attribute__((aligned(16))) float rawl[ONE && RAW ? MAX_CHUNK : 4];

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int l15 = lane & 15, quad = lane >> 4;

    // ---- which rows, which keys ----
    int head, row0, nrows, k0, k1, slot, lim0 = 0x3fffffff, brow = 0;
    const __bf16 *kb, *vb;
    int64_t ldk, ldv;
    bool shared_keys, alone = false, live = true;          // alone: this wave has keys and rows of its own, if live
    const int pA = ONE ? p.P : 0, nA = (pA + TK - 1) / TK;      // ONE: tiles [0, nA) are the prefix's, the own keys' follow
    if (!ONE && blockIdx.x < p.pjobs) {      // row groups of one (head, chunk) follow each other: the later ones find K and V in L2
        const int rg = blockIdx.x % p.nprg, hc = blockIdx.x / p.nprg;
        head = hc % p.H;
        slot = hc / p.H;
        k0 = slot * p.pc;
        k1 = min(k0 + p.pc, p.P);
        row0 = rg * RT * 16;
        nrows = min(RT * 16, p.R - row0);
        kb = p.KP + head * HD;
        vb = p.VP + head * HD;
        ldk = p.ldkp;
        ldv = p.ldvp;
        shared_keys = true;
    } else {
        int j = (int)(blockIdx.x - (ONE ? 0 : p.pjobs));
        if (!ONE && !RAW && p.by_wave) {
            const int jobs = p.B * p.H * p.norg;
            alone = true;
            j = j * NW + wave;
            live = j < jobs;
            j = min(j, jobs - 1);
        }
        const int rg = j % p.norg;
        j /= p.norg;
        head = j % p.H;
        j /= p.H;
        brow = ONE ? j : j / p.noc;
        const int c = ONE ? 0 : j - brow * p.noc;
        slot = p.npc + c;
        k0 = ONE ? 0 : c * p.oc;
        k1 = ONE ? p.Nk : min(k0 + p.oc, p.Nk);
        const int i0 = rg * RT * 16;
        row0 = brow * p.Nq + i0;
        nrows = min(RT * 16, p.Nq - i0);
        lim0 = i0 + p.Nk - p.Nq;          // last key the group's first row sees
        k1 = min(k1, lim0 + nrows);       // no row of the group sees a key behind its last row's
        kb = p.K + (int64_t)brow * p.bsk + head * HD;
        vb = p.V + (int64_t)brow * p.bsv + head * HD;
        ldk = p.ldk;
        ldv = p.ldv;
        shared_keys = false;
    }
    const bool has_bias = BIAS && !shared_keys;
    const float* bls = blds + (alone ? wave * (MAX_CHUNK / NW) : 0);
    if (has_bias) {
        const float* bp = p.bias + (int64_t)brow * p.bias_bs + (int64_t)head * p.bias_hs;
        if (alone) {
            for (int i = lane; i < MAX_CHUNK / NW && k0 + i < k1; i += 64) blds[wave * (MAX_CHUNK / NW) + i] = bp[k0 + i];
        } else {
            for (int i = tid; i < MAX_CHUNK && k0 + i < k1; i += NW * 64) blds[i] = bp[k0 + i];
        }
        __syncthreads();
    }

    bf16x8 qf[RT][KS];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const int row = row0 + min(rt * 16 + l15, nrows - 1);
        const int b = row / p.Nq, i = row - b * p.Nq;
        const __bf16* qp = p.Q + (int64_t)b * p.bsq + (int64_t)i * p.ldq + head * HD + 8 * quad;
#pragma unroll
        for (int s = 0; s < KS; ++s) qf[rt][s] = *reinterpret_cast<const bf16x8*>(qp + 32 * s);
    }

    f32x4 ot[RT][DT];
    float m[RT], l[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        m[rt] = M_NONE;
        l[rt] = 0.f;
#pragma unroll
        for (int d = 0; d < DT; ++d) ot[rt][d] = f32x4{0.f, 0.f, 0.f, 0.f};
    }

    bf16x8 kr[2][KS];
    u32x4 vr[NL];
    const int vrow = lane / CH, vch = lane % CH;
    auto load_k = [&](int t) {
        const bool pre = ONE && t < nA;
        const __bf16* base = pre ? p.KP + head * HD : kb;
        const int64_t ld = pre ? p.ldkp : ldk;
        const int first = pre ? t * TK : k0 + (t - nA) * TK, last = (pre ? pA : k1) - 1;
#pragma unroll
        for (int g = 0; g < 2; ++g) {
            const __bf16* kp = base + (int64_t)min(first + 16 * g + l15, last) * ld + 8 * quad;
#pragma unroll
            for (int s = 0; s < KS; ++s) kr[g][s] = *reinterpret_cast<const bf16x8*>(kp + 32 * s);
        }
    };
    auto load_v = [&](int t) {
        const bool pre = ONE && t < nA;
        const __bf16* base = pre ? p.VP + head * HD : vb;
        const int64_t ld = pre ? p.ldvp : ldv;
        const int first = pre ? t * TK : k0 + (t - nA) * TK, last = (pre ? pA : k1) - 1;
#pragma unroll
        for (int i = 0; i < NL; ++i)
            vr[i] = *reinterpret_cast<const u32x4*>(base + (int64_t)min(first + i * RPL + vrow, last) * ld + vch * 8);
    };
    // 16-byte chunk c of key row r lives at chunk c ^ swz(r): the 16 key rows x 32 bytes of one transposing read then touch every
    // bank twice, the least there is (512 bytes at 128 a cycle)
    auto swz = [](int r) { return HD == 128 ? (r & 7) << 1 : ((r >> 1) & 3) << 1; };
    char* vw = vlds + wave * WB;
    const int trow = 4 * quad + (l15 >> 2);               // transposing read: this lane's key row (and + 16), 8 bytes of it
    int toff[DT];
#pragma unroll
    for (int d = 0; d < DT; ++d) toff[d] = trow * HD * 2 + (((2 * d + ((lane & 3) >> 1)) ^ swz(trow)) << 4) + 8 * (lane & 1);

    const int nt = live ? nA + (k1 > k0 ? (k1 - k0 + TK - 1) / TK : 0) : 0;
    const int tf = alone ? 0 : wave, ts = alone ? 1 : NW;  // the wave's tiles: tf, tf + ts, ...
    if (tf < nt) {
        load_k(tf);
        load_v(tf);
    }
    for (int t = tf; t < nt; t += ts) {
        f32x4 st[RT][2];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
            for (int g = 0; g < 2; ++g) {
                st[rt][g] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int s = 0; s < KS; ++s) st[rt][g] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kr[g][s], qf[rt][s], st[rt][g], 0, 0, 0);
            }
        const bool more = t + ts < nt;
        if (more) load_k(t + ts);
        // ---- bias, removed and invisible keys ----
        const bool pre = ONE && t < nA;
        const int kt = pre ? t * TK : k0 + (t - nA) * TK, ke = pre ? pA : k1;
        uint32_t gone = 0;                                // keys of this tile that no row has: their V rows are made zero
        if (has_bias && !pre) {
            const float* bl = bls + (t - nA) * TK;
            const bool rem = lane < TK && (kt + lane >= ke || bl[lane] <= REMOVED);
            gone = (uint32_t)__builtin_amdgcn_ballot_w64(rem);
#pragma unroll
            for (int g = 0; g < 2; ++g) {
                const f32x4 bv = *reinterpret_cast<const f32x4*>(bl + 16 * g + 4 * quad);
#pragma unroll
                for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        st[rt][g][i] = (gone >> (16 * g + 4 * quad + i)) & 1 ? -INFINITY : st[rt][g][i] + bv[i] * HK_LOG2E;
            }
        } else if (kt + TK > ke) {
            gone = 0xffffffffu << (ke - kt);              // ke - kt is 1 .. 31 here
        }
        if (kt + TK > ke || (!pre && kt + TK - 1 > lim0)) {
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                const int lim = pre ? ke - 1 : min(ke - 1, lim0 + rt * 16 + l15);
#pragma unroll
                for (int g = 0; g < 2; ++g)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (kt + 16 * g + 4 * quad + i > lim) st[rt][g][i] = -INFINITY;
            }
        }
        if (RAW && l15 == 0) {                            // one row: its scores, for the weights
            float* rp = ONE ? rawl + kt : p.raw + ((int64_t)brow * p.H + head) * p.raw_ld + kt;
            *reinterpret_cast<f32x4*>(rp + 4 * quad) = st[0][0];
            *reinterpret_cast<f32x4*>(rp + 16 + 4 * quad) = st[0][1];
        }
        // ---- running maximum: moved only when some row outgrows it by 8 bits ----
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            float mx = fmaxf(fmaxf(fmaxf(st[rt][0][0], st[rt][0][1]), fmaxf(st[rt][0][2], st[rt][0][3])),
                             fmaxf(fmaxf(st[rt][1][0], st[rt][1][1]), fmaxf(st[rt][1][2], st[rt][1][3])));
            if (__builtin_amdgcn_ballot_w64(mx > m[rt] + 8.f)) {
                mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
                mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
                const float mn = fmaxf(m[rt], mx);
                const float a = __builtin_amdgcn_exp2f(m[rt] - mn);
                m[rt] = mn;
                l[rt] *= a;
#pragma unroll
                for (int d = 0; d < DT; ++d)
#pragma unroll
                    for (int i = 0; i < 4; ++i) ot[rt][d][i] *= a;
            }
        }
        // P as two bf16 numbers (the matrix instruction's operand), its value and what that rounding left: off by 2^-16 of itself.  Reading K and V
        // bounds these calls, so the second product is nearly free, and a step keeps what a softmax in 32 bits has.  One : two (us, in a graph):
        // 16 sequences' step over 1985 + 61 keys 15.0 : 14.6, padded 16.4 : 16.7; 4 over 352 + 20 7.3 : 7.4; 5 x 3 over 907 (64) 7.6 : 7.8; weights, 16 x 1500 85.9 : 86.2.
        bf16x8 pf[RT], pl[RT];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            float e[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                e[i] = __builtin_amdgcn_exp2f(st[rt][i >> 2][i & 3] - m[rt]);
                l[rt] += e[i];
            }
            u32x4 w, x;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                w[i] = pack_bf16x2(e[2 * i], e[2 * i + 1]);
                x[i] = pack_bf16x2(e[2 * i] - bf16_lo(w[i]), e[2 * i + 1] - bf16_hi(w[i]));
            }
            pf[rt] = __builtin_bit_cast(bf16x8, w);
            pl[rt] = __builtin_bit_cast(bf16x8, x);
        }
        // ---- V through LDS ----
        if (gone) {
#pragma unroll
            for (int i = 0; i < NL; ++i)
                if ((gone >> (i * RPL + vrow)) & 1) vr[i] = u32x4{0, 0, 0, 0};
        }
#pragma unroll
        for (int i = 0; i < NL; ++i) {
            const int r = i * RPL + vrow;
            *reinterpret_cast<u32x4*>(vw + r * HD * 2 + ((vch ^ swz(r)) << 4)) = vr[i];
        }
        wave_lds_sync();
        if (more) load_v(t + ts);
#pragma unroll
        for (int d = 0; d < DT; d += 2) {                 // two blocks: independent chains
            bf16x8 vf[2];
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const bf16x4 v0 = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((__attribute__((address_space(3))) bf16x4*)(vw + toff[d + x]));
                const bf16x4 v1 = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((__attribute__((address_space(3))) bf16x4*)(vw + toff[d + x] + 16 * HD * 2));
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    vf[x][i] = v0[i];
                    vf[x][i + 4] = v1[i];
                }
            }
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                for (int x = 0; x < 2; ++x) ot[rt][d + x] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf[x], pf[rt], ot[rt][d + x], 0, 0, 0);
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                for (int x = 0; x < 2; ++x) ot[rt][d + x] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf[x], pl[rt], ot[rt][d + x], 0, 0, 0);
        }
        wave_lds_sync();
    }

    // ---- join the waves (in wave order), leave the chunk's (m, l, o) ----
    float* ow = reinterpret_cast<float*>(vw);
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        l[rt] += __shfl_xor(l[rt], 16, 64);
        l[rt] += __shfl_xor(l[rt], 32, 64);
        if (quad == 0) {
            ml[wave][rt * 16 + l15][0] = m[rt];
            ml[wave][rt * 16 + l15][1] = l[rt];
        }
#pragma unroll
        for (int d = 0; d < DT; ++d)     // element (row, dim) at row * HD + dim; 16-byte pieces rotated by the row against bank conflicts
            *reinterpret_cast<f32x4*>(ow + (rt * 16 + l15) * HD + (((4 * d + quad) ^ (l15 & 7)) << 2)) = ot[rt][d];
    }
    __syncthreads();
    constexpr int TPR = HD / 4;                            // threads per row, four dims each
    if (alone) {
        for (int r = lane / TPR; live && r < nrows; r += 64 / TPR) {
            const int c = lane % TPR;
            const int64_t at = ((int64_t)(row0 + r) * p.H + head) * p.ns + slot;
            *reinterpret_cast<f32x4*>(p.part_o + at * HD + 4 * c) = *reinterpret_cast<const f32x4*>(ow + r * HD + ((c ^ (r & 7)) << 2));
            if (c == 0) {
                p.part_ml[at * 2] = ml[wave][r][0];
                p.part_ml[at * 2 + 1] = ml[wave][r][1];
            }
        }
        return;
    }
    for (int r = tid / TPR; r < nrows; r += NW * 64 / TPR) {
        const int c = tid % TPR;
        float M = ml[0][r][0];
#pragma unroll
        for (int w = 1; w < NW; ++w) M = fmaxf(M, ml[w][r][0]);
        f32x4 o = {0.f, 0.f, 0.f, 0.f};
        float ls = 0.f;
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            const float a = __builtin_amdgcn_exp2f(ml[w][r][0] - M);
            const f32x4 x = *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(vlds + w * WB) + r * HD + ((c ^ (r & 7)) << 2));
            ls += a * ml[w][r][1];
#pragma unroll
            for (int i = 0; i < 4; ++i) o[i] += a * x[i];
        }
        if (ONE) {
            const float inv = inverse_sum(ls);
            const int row = row0 + r, b = row / p.Nq, i = row - b * p.Nq;
            u32x2 w;
            w[0] = pack_bf16x2(o[0] * inv, o[1] * inv);
            w[1] = pack_bf16x2(o[2] * inv, o[3] * inv);
            *reinterpret_cast<u32x2*>(p.O + (int64_t)b * p.bso + (int64_t)i * p.ldo + head * HD + 4 * c) = w;
            continue;
        }
        const int64_t at = ((int64_t)(row0 + r) * p.H + head) * p.ns + slot;
        *reinterpret_cast<f32x4*>(p.part_o + at * HD + 4 * c) = o;
        if (c == 0) {
            p.part_ml[at * 2] = M;
            p.part_ml[at * 2 + 1] = ls;
        }
    }
    if (ONE && RAW) {                                      // the weights of the one row
        float M = ml[0][0][0], ls = 0.f;
#pragma unroll
        for (int w = 1; w < NW; ++w) M = fmaxf(M, ml[w][0][0]);
#pragma unroll
        for (int w = 0; w < NW; ++w) ls += __builtin_amdgcn_exp2f(ml[w][0][0] - M) * ml[w][0][1];
        add_weights(p, sw, brow, head, rawl, M, inverse_sum(ls), tid, NW * 64);
    }
}

// ---------------------------------------------------------------- many rows
// hk_prefix_rows_kernel: a workgroup = 128 query rows of one head (four waves of 32) that share 64-key tiles in LDS (two stages,
// LDS-DMA one tile ahead, two workgroups per CU).  With 32 rows per wave the matrix instructions, not memory, are the bound:
// v_mfma_f32_32x32x16_bf16, transposed as above (lane -> row lane & 31; the S^T accumulator is the B operand of O^T += V^T . P^T).
// The running maximum enters as the first instruction's accumulator and is taken again only when a tile's partial row sum leaves
// [0, 2^20] (that tile is redone): the common path is exp2 and an addition per score.  A row that has met no key yet takes the
// maximum of every tile until it does.
// Rows are a sequence's (its keys: the prefix, then its own up to the diagonal; or its own alone) or, for the prefix alone, rows of
// all sequences packed: whichever leaves fewer 128-row blocks part empty (make_plan).
// GRP = 2: two such groups of waves share a workgroup, each with stages of its own, and take every other tile; the second's (m, l, o) joins the
// first's through LDS at the end (where CUs would be idle: make_plan).
// A tile with nothing to mask goes by halves, the second half's products among the first half's exponentials.
// TWO: P as two bf16 numbers, as in hk_prefix_part_kernel, for steps (MIXED, Nq = 1), which reading bounds: one : two (us, in a graph), 64 sequences
// over 16384 + 333 keys 129.3 : 130.2, 128 over 2000 + 20 32.1 : 33.8.  One, off by 2^-8, for questions, as in hk_flash_attn_bf16: the feed of the
// matrix unit bounds those (32 x 16 tokens over 1600 39.2 : 44.4).
// Measured (32 heads of 128): 8 sequences of 512 rows over 1400 shared keys and their own 116-125 us, 890-960 TFLOP/s; the matrix unit is busy half of
// the time.  Copies of the loop without one part, in-bounds and for timing only: without LDS-DMA and barriers 107-116 us, without the reads of
// K from LDS 84, without those of V too 79, without exp2 101: bound by feeding the matrix unit from LDS (each wave reads every tile), at the clock that the
// card holds under it.  Slower: 32-key tiles at 3-4 waves per SIMD (10-40 %), LDS-DMA spread over the matrix steps (141), K read before
// the LDS-DMA is issued (130), four stages instead of two (10-40 % where a CU holds two workgroups, the same elsewhere).  64 sequences' single rows over 16384 shared keys
// (268 MB, one workgroup per CU): 59-69 us, 3.9-4.5 TB/s, P as two numbers (54-59 as one).
struct RowsParams {
    int packed;                      // prefix by packed row blocks and key chunks, own keys apart; else both in one workgroup
    int npb, nob;                    // row blocks: of all rows (packed prefix), of a sequence
    int64_t pjobs;                   // packed: workgroups of the prefix = npb * npc * H
};

constexpr int RB = 128;
constexpr int KT = 64;               // keys per tile
constexpr float OVERFLOW_SUM = 1048576.0f;

__device__ __forceinline__ float half_max(float x) {    // the larger of the two lane halves' values (rows live on lane & 31)
    float a = x, b = x;
    asm volatile("s_nop 1\n\tv_permlane32_swap_b32 %0, %1" : "+v"(a), "+v"(b));
    return fmaxf(a, b);
}

template <int HD, bool BIAS, int GRP, bool TWO>
__global__ __launch_bounds__(GRP * 256, 2) void hk_prefix_rows_kernel(const PrefixParams p, const RowsParams q) {
    constexpr int ROWB = HD * 2, CH = HD / 8, NKS = HD / 16, NDT = HD / 32;
    constexpr int STAGE = 2 * KT * ROWB;
    constexpr int RPP = 256 / CH;                          // key rows one workgroup-wide LDS-DMA covers
    constexpr int NP = KT / RPP;                           // of them per operand and tile
    extern __shared__ __attribute__((aligned(16))) char smem[];      // per group: [2][K | V][KT keys][ROWB]; then per group [2][KT] biases
    const int tid = threadIdx.x & 255, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int grp = GRP == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x >> 8);
    char* gs = smem + grp * 2 * STAGE;
    float* blds = reinterpret_cast<float*>(smem + GRP * 2 * STAGE) + grp * 2 * KT;
    const int r = lane & 31, h = lane >> 5;

    // ---- which rows, which keys (blockIdx = ... * H + head: the row blocks of a head share an XCD's L2 where H is a multiple of 8) ----
    const int head = blockIdx.x % p.H;
    int rest = blockIdx.x / p.H;
    int row0, nrows, a0 = 0, a1 = 0, k1 = 0, slot = -1, brow = 0, b0 = 0;
    int off = 0x3fffffff;                                  // row i of the block sees own keys <= i + off
    if (q.packed && blockIdx.x < q.pjobs) {
        const int rb = rest % q.npb;
        slot = rest / q.npb;
        row0 = rb * RB;
        nrows = min(RB, p.R - row0);
        a0 = slot * p.pc;
        a1 = min(a0 + p.pc, p.P);
    } else {
        if (q.packed) {
            rest -= (int)(q.pjobs / p.H);
            slot = p.npc;
        } else {
            a1 = p.P;
        }
        brow = rest % p.B;
        rest /= p.B;
        const int rb = q.nob - 1 - rest % q.nob;           // longest first
        const int c = rest / q.nob;                        // packed: the own keys' chunk
        if (q.packed) {
            slot += c;
            b0 = c * p.oc;
        }
        const int i0 = rb * RB;
        row0 = brow * p.Nq + i0;
        nrows = min(RB, p.Nq - i0);
        off = i0 + p.Nk - p.Nq - b0;                       // own keys are counted from the chunk's first
        k1 = max(0, min(q.packed ? min(p.oc, p.Nk - b0) : p.Nk, off + nrows));
    }
    const int nA = (a1 - a0 + KT - 1) / KT, NT = nA + (k1 + KT - 1) / KT;
    const int q0 = wave * 32;                              // the wave's first row within the block
    const bool active = q0 < nrows;

    bf16x8 qf[NKS];
    {
        const int row = row0 + min(q0 + r, nrows - 1);
        const int b = row / p.Nq, i = row - b * p.Nq;
        const __bf16* qp = p.Q + (int64_t)b * p.bsq + (int64_t)i * p.ldq + head * HD + 8 * h;
#pragma unroll
        for (int s = 0; s < NKS; ++s) qf[s] = *reinterpret_cast<const bf16x8*>(qp + 16 * s);
    }
    // The loads above are waited for here: left pending, the compiler would wait for them inside the loop, with counts that take the
    // LDS-DMA in flight there (which it does not know) along.
#pragma unroll
    for (int s = 0; s < NKS; ++s) asm volatile("" : "+v"(qf[s]));
    const __bf16* kA = p.KP + (int64_t)a0 * p.ldkp + head * HD;
    const __bf16* vA = p.VP + (int64_t)a0 * p.ldvp + head * HD;
    const __bf16* kB = p.K + (int64_t)brow * p.bsk + (int64_t)b0 * p.ldk + head * HD;
    const __bf16* vB = p.V + (int64_t)brow * p.bsv + (int64_t)b0 * p.ldv + head * HD;
    const float* bias = BIAS ? p.bias + (int64_t)brow * p.bias_bs + (int64_t)head * p.bias_hs + b0 : nullptr;

    // K: 16-byte chunk c of key row x at c ^ swk(x): 16 rows x one chunk touch every bank once; V: at c ^ swv(x): so do the 4 key rows x
    // 64 bytes that half a wave's transposing read takes
    auto swk = [](int x) { return HD == 128 ? x & 15 : (x >> 1) & 7; };
    auto swv = [](int x) { return HD == 128 ? (x & 3) << 2 : ((x >> 1) & 1) << 2; };
    const int lrow = tid / CH, lch = tid % CH;
    const uint32_t klA = (uint32_t)((lrow * p.ldkp + (lch ^ swk(lrow)) * 8) * 2), klB = (uint32_t)((lrow * p.ldk + (lch ^ swk(lrow)) * 8) * 2);
    const uint32_t vlA = (uint32_t)((lrow * p.ldvp + (lch ^ swv(lrow)) * 8) * 2), vlB = (uint32_t)((lrow * p.ldv + (lch ^ swv(lrow)) * 8) * 2);
    float br = 0.f;
    auto load_tile = [&](const __bf16* kb, const __bf16* vb, int64_t ldk, int64_t ldv, uint32_t kl, uint32_t vl, int kt, int n, int stage)
        __attribute__((always_inline)) {
        char* ks = gs + stage * STAGE + wave * (64 / CH) * ROWB;
        char* vs = ks + KT * ROWB;
        // the swizzle goes on the source chunk (the LDS image is lane-linear); RPP is a multiple of every swizzle's period
        if (kt + KT <= n) {
#pragma unroll
            for (int i = 0; i < NP; ++i) {
                glds16_s(kb + (int64_t)(kt + i * RPP) * ldk, kl, ks + i * RPP * ROWB);
                glds16_s(vb + (int64_t)(kt + i * RPP) * ldv, vl, vs + i * RPP * ROWB);
            }
        } else {
#pragma unroll
            for (int i = 0; i < NP; ++i) {
                const int64_t key = min(kt + i * RPP + lrow, n - 1);
                glds16_v(kb + key * ldk + (lch ^ swk(lrow)) * 8, ks + i * RPP * ROWB);
                glds16_v(vb + key * ldv + (lch ^ swv(lrow)) * 8, vs + i * RPP * ROWB);
            }
        }
    };
    auto issue = [&](int t, int stage) __attribute__((always_inline)) {
        if (GRP > 1 && t >= NT) return;
        if (t < nA) {
            load_tile(kA, vA, p.ldkp, p.ldvp, klA, vlA, t * KT, a1 - a0, stage);
        } else {
            load_tile(kB, vB, p.ldk, p.ldv, klB, vlB, (t - nA) * KT, k1, stage);
            if (BIAS && tid < KT) br = bias[min((t - nA) * KT + tid, k1 - 1)];
        }
    };
    // K fragment (g, s): row 32 g + r, chunk 2 s + h; V fragment (s, d): rows 16 s + vrow (and + 8), dims 32 d + 16 ((lane >> 4) & 1) + ...:
    // chunk numbers are joined to the swizzle by exclusive or, so one register per operand holds every offset
    const int vrow = 4 * h + ((lane & 15) >> 2);
    const int koff0 = r * ROWB + ((h ^ swk(r)) << 4);
    const int voff0 = vrow * ROWB + (((2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) ^ swv(vrow)) << 4) + 8 * (lane & 1);

    f32x16 ot[NDT];
#pragma unroll
    for (int d = 0; d < NDT; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) ot[d][i] = 0.f;
    float m = 0.f, l = 0.f;                                // everything stored is relative to m
    bool unset = true, pending = true;                     // this row / some row of the wave has met no key yet

    if (NT > 0) {
        issue(grp, 0);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        if (BIAS && grp >= nA && tid < KT) blds[tid] = br;
        __syncthreads();
    }
    for (int u = 0; u * GRP < NT; ++u) {
        const int cur = u & 1, t = u * GRP + grp;
        if (t + GRP < NT) issue(t + GRP, cur ^ 1);
        const bool own = t >= nA;
        const int kt = (own ? t - nA : t) * KT, n = own ? k1 : a1 - a0;
        if (active && (GRP == 1 || t < NT) && (!own || kt <= q0 + 31 + off)) {
            int ko = koff0, vo = voff0;
            asm volatile("" : "+v"(ko), "+v"(vo));          // the offsets are made from these here, not kept across tiles in registers
            const char* ks = gs + cur * STAGE;
            const char* vs = ks + KT * ROWB;
            uint64_t gone = 0;                             // keys of this tile that no row has
            bool biased = false, added = false;            // some key is biased or removed / some key that stays is biased
            if (BIAS && own) {
                const float v = blds[cur * KT + lane];
                gone = __builtin_amdgcn_ballot_w64(kt + lane >= n || v <= REMOVED);
                biased = __builtin_amdgcn_ballot_w64(v != 0.f) != 0;
                added = __builtin_amdgcn_ballot_w64(v != 0.f && !(v <= REMOVED)) != 0;
            }
            const bool edge = kt + KT > n || (own && kt + KT - 1 > q0 + off);
            f32x16 st[2];
            auto kread = [&](int i) __attribute__((always_inline)) {   // K fragment of step i: half i / NKS, contraction step i % NKS
                return *reinterpret_cast<const bf16x8*>(ks + (i / NKS) * 32 * ROWB + (ko ^ (32 * (i % NKS))));
            };
            auto vread = [&](int j) __attribute__((always_inline)) {   // V fragment of step j: 16 keys j / NDT, 32 dims j % NDT
                const char* vp = vs + (j / NDT) * 16 * ROWB + (vo ^ (64 * (j % NDT)));
                const bf16x4 v0 = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((__attribute__((address_space(3))) bf16x4*)(vp));
                const bf16x4 v1 = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((__attribute__((address_space(3))) bf16x4*)(vp + 8 * ROWB));
                bf16x8 vf;
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    vf[x] = v0[x];
                    vf[x + 4] = v1[x];
                }
                return vf;
            };
            auto rest = [&](int s, bf16x8 hi) __attribute__((always_inline)) {      // what rounding left of the values in piece s of P
                const u32x4 w = __builtin_bit_cast(u32x4, hi);
                u32x4 x;
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    x[j] = pack_bf16x2(st[s >> 1][8 * (s & 1) + 2 * j] - bf16_lo(w[j]), st[s >> 1][8 * (s & 1) + 2 * j + 1] - bf16_hi(w[j]));
                return __builtin_bit_cast(bf16x8, x);
            };
            const bool plain = !pending && !edge && !(BIAS && (biased || gone));
            int from = 0;                                  // the tile's keys from here on are left to the general form below
            if (plain) {
                // The ordinary tile, by halves of 32 keys, one matrix instruction after the other with what fits beside it:
                //   S(0)   |   S(1), exp of half 0   |   P(0) . V, exp of half 1   |   P(1) . V
                // fragments are read four instructions ahead; sched_barrier keeps the order (left to itself the compiler reads into one
                // set of registers and waits for every read right before its use).  A wave that feeds the matrix unit goes before one that does not
                // (8 x 512 questions' tokens over 1400: 130 us without the priorities, 124 with).
                __builtin_amdgcn_s_setprio(1);
                bf16x8 kf[4], vf[4];
                float e0 = 0.f, e1 = 0.f;
#pragma unroll
                for (int i = 0; i < 4; ++i) kf[i] = kread(i);
                f32x16 c0;
#pragma unroll
                for (int i = 0; i < 16; ++i) c0[i] = -m;
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int i = 0; i < 2 * NKS; ++i) {
                    const int g = i / NKS, s = i % NKS;
                    st[g] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[i & 3], qf[s], s == 0 ? c0 : st[g], 0, 0, 0);
                    if (i + 4 < 2 * NKS) kf[i & 3] = kread(i + 4);
                    else vf[i + 4 - 2 * NKS] = vread(i + 4 - 2 * NKS);
                    if (g == 1 && s >= NKS / 4) {          // half 0's scores have left the matrix unit
                        constexpr int ST = NKS - NKS / 4;
                        const int x = s - NKS / 4;
#pragma unroll
                        for (int y = 16 * x / ST; y < 16 * (x + 1) / ST; ++y) {
                            st[0][y] = __builtin_amdgcn_exp2f(st[0][y]);
                            e0 += st[0][y];
                        }
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
                auto pack = [&](int s) __attribute__((always_inline)) {
                    u32x4 w;
#pragma unroll
                    for (int j = 0; j < 4; ++j) w[j] = pack_bf16x2(st[s >> 1][8 * (s & 1) + 2 * j], st[s >> 1][8 * (s & 1) + 2 * j + 1]);
                    return __builtin_bit_cast(bf16x8, w);
                };
                if (__builtin_amdgcn_ballot_w64(!(e0 <= OVERFLOW_SUM)) == 0) {
                    l += e0;
                    bf16x8 pf[2] = {pack(0), pack(1)}, pl[2];
                    if (TWO) pl[0] = rest(0, pf[0]), pl[1] = rest(1, pf[1]);
                    __builtin_amdgcn_s_setprio(2);
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int j = 0; j < 2 * NDT; ++j) {
                        ot[j % NDT] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf[j & 3], pf[j / NDT], ot[j % NDT], 0, 0, 0);
                        if (TWO) ot[j % NDT] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf[j & 3], pl[j / NDT], ot[j % NDT], 0, 0, 0);
                        if (j + 4 < 4 * NDT) vf[j & 3] = vread(j + 4);
#pragma unroll
                        for (int y = 16 * j / (2 * NDT); y < 16 * (j + 1) / (2 * NDT); ++y) {
                            st[1][y] = __builtin_amdgcn_exp2f(st[1][y]);
                            e1 += st[1][y];
                        }
                        __builtin_amdgcn_sched_barrier(0);
                    }
                    from = 32;
                    if (__builtin_amdgcn_ballot_w64(!(e1 <= OVERFLOW_SUM)) == 0) {
                        l += e1;
                        pf[0] = pack(2);
                        pf[1] = pack(3);
                        if (TWO) pl[0] = rest(2, pf[0]), pl[1] = rest(3, pf[1]);
                        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                        for (int j = 2 * NDT; j < 4 * NDT; ++j) {
                            ot[j % NDT] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf[j & 3], pf[j / NDT - 2], ot[j % NDT], 0, 0, 0);
                            if (TWO) ot[j % NDT] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf[j & 3], pl[j / NDT - 2], ot[j % NDT], 0, 0, 0);
                            if (j + 4 < 4 * NDT) vf[j & 3] = vread(j + 4);
                            __builtin_amdgcn_sched_barrier(0);
                        }
                        from = 64;
                    }
                }
                __builtin_amdgcn_s_setprio(0);
            }
            if (from < 64) {
                // ends, diagonals, biases, rows without a key so far, scores that outgrew m: the tile as a whole, masks and all
                float rs;
                // base: what the scores are relative to.  The products start from it only where they are of its size: added to a reference point far
                // away, or one that biases make large, they would lose bits at every step.
                auto scores = [&](float base) __attribute__((always_inline)) {
                    int kz = ko, bz = cur * KT + 4 * h;
                    uint64_t gz = gone;
                    asm volatile("" : "+v"(kz), "+v"(bz), "+s"(gz));        // read again each time: kept, the fragments, biases and masks of a tile fill the registers
                    f32x16 c0;
#pragma unroll
                    for (int i = 0; i < 16; ++i) c0[i] = BIAS && biased ? 0.f : -base;
#pragma unroll
                    for (int s = 0; s < NKS; ++s)              // two independent chains
#pragma unroll
                        for (int g = 0; g < 2; ++g)
                            st[g] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(*reinterpret_cast<const bf16x8*>(ks + g * 32 * ROWB + (kz ^ (32 * s))), qf[s],
                                                                            s == 0 ? c0 : st[g], 0, 0, 0);
                    if (BIAS && biased) {                      // register 4 x + j of st[g] <-> key 32 g + 8 x + 4 h + j
#pragma unroll
                        for (int g = 0; g < 2; ++g)
#pragma unroll
                            for (int x = 0; x < 4; ++x) {
                                const f32x4 bv = *reinterpret_cast<const f32x4*>(blds + bz + 32 * g + 8 * x);
                                const uint32_t gb = (uint32_t)(gz >> (32 * g + 8 * x)) >> (4 * h);
#pragma unroll
                                for (int j = 0; j < 4; ++j) st[g][4 * x + j] = (gb >> j) & 1 ? -INFINITY : st[g][4 * x + j] + fmaf(bv[j], HK_LOG2E, -base);
                            }
                    }
                    if (edge || from) {
                        int lim = min(n - 1, own ? q0 + r + off : n - 1) - kt - 4 * h;
                        asm volatile("" : "+v"(lim));
#pragma unroll
                        for (int g = 0; g < 2; ++g)
#pragma unroll
                            for (int i = 0; i < 16; ++i)
                                if (32 * g + (i & 3) + 8 * (i >> 2) > lim || (g == 0 && from)) st[g][i] = -INFINITY;
                    }
                };
                auto exp_sum = [&]() __attribute__((always_inline)) {
                    rs = 0.f;
#pragma unroll
                    for (int g = 0; g < 2; ++g)
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            const float e = __builtin_amdgcn_exp2f(st[g][i]);
                            st[g][i] = e;
                            rs += e;
                        }
                };
                auto move_max = [&]() __attribute__((always_inline)) {
                    float mx = fmaxf(st[0][0], st[1][0]);
#pragma unroll
                    for (int i = 1; i < 16; ++i) mx = fmaxf(mx, fmaxf(st[0][i], st[1][i]));
                    mx = half_max(mx);
                    const float mn = unset ? (mx == -INFINITY ? 0.f : mx) : fmaxf(m, mx);
                    const float a = unset ? 0.f : __builtin_amdgcn_exp2f(m - mn);
                    unset = unset && mx == -INFINITY;
                    pending = __builtin_amdgcn_ballot_w64(unset) != 0;
                    m = mn;
                    l *= a;
#pragma unroll
                    for (int d = 0; d < NDT; ++d)
#pragma unroll
                        for (int i = 0; i < 16; ++i) ot[d][i] *= a;
                };
                auto pv = [&](const bf16x8* pf, const bf16x8* pl, auto masked_c) __attribute__((always_inline)) {
#pragma unroll
                    for (int s = 0; s < 4; ++s) {
                        u32x4 keep = {~0u, ~0u, ~0u, ~0u};
                        if (decltype(masked_c)::value) {       // elements 0-3: keys 16 s + 4 h + j, elements 4-7: 8 further
                            const uint32_t g = (uint32_t)(gone >> (16 * s)) >> (4 * h);
#pragma unroll
                            for (int j = 0; j < 2; ++j) {
                                keep[j] = ((g >> (2 * j)) & 1 ? 0u : 0xffffu) | ((g >> (2 * j + 1)) & 1 ? 0u : 0xffff0000u);
                                keep[j + 2] = ((g >> (8 + 2 * j)) & 1 ? 0u : 0xffffu) | ((g >> (8 + 2 * j + 1)) & 1 ? 0u : 0xffff0000u);
                            }
                        }
#pragma unroll
                        for (int d = 0; d < NDT; ++d) {
                            bf16x8 vf = vread(s * NDT + d);
                            if (decltype(masked_c)::value) vf = __builtin_bit_cast(bf16x8, __builtin_bit_cast(u32x4, vf) & keep);
                            ot[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf, pf[s], ot[d], 0, 0, 0);
                            if (TWO) ot[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf, pl[s], ot[d], 0, 0, 0);
                        }
                    }
                };
                for (bool take = pending || plain;; take = true) {      // at most twice
                    scores(take ? 0.f : m);
                    if (take) {
                        move_max();
                        if (BIAS && added) {               // once more, relative to the new m: beside their biases the scores have lost bits
                            scores(m);
                        } else {
#pragma unroll
                            for (int g = 0; g < 2; ++g)
#pragma unroll
                                for (int i = 0; i < 16; ++i) st[g][i] -= m;
                        }
                    }
                    exp_sum();
                    if (take || __builtin_amdgcn_ballot_w64(!(rs <= OVERFLOW_SUM)) == 0) break;
                }
                l += rs;
                bf16x8 pf[4], pl[4];                           // P in bf16, the matrix instruction's operand; l sums the unrounded values
#pragma unroll
                for (int s = 0; s < 4; ++s) {
                    u32x4 w;
#pragma unroll
                    for (int j = 0; j < 4; ++j) w[j] = pack_bf16x2(st[s >> 1][8 * (s & 1) + 2 * j], st[s >> 1][8 * (s & 1) + 2 * j + 1]);
                    pf[s] = __builtin_bit_cast(bf16x8, w);
                    if (TWO) pl[s] = rest(s, pf[s]);
                }
                if (BIAS && gone) pv(pf, pl, std::true_type{});
                else pv(pf, pl, std::false_type{});
            }
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // the next tile's LDS-DMA, unknown to the compiler
        if (BIAS && t + GRP >= nA && t + GRP < NT && tid < KT) blds[(cur ^ 1) * KT + tid] = br;
        __syncthreads();
    }

    if (GRP > 1) {                                         // the second group's part joins the first's (everyone has left the last tiles)
        float* js = reinterpret_cast<float*>(smem) + tid;  // [NDT * 16 + 2][256 threads]
        if (unset) m = M_NONE;
        if (grp) {
            js[0] = m;
            js[256] = l;
#pragma unroll
            for (int d = 0; d < NDT; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i) js[(2 + 16 * d + i) * 256] = ot[d][i];
        }
        __syncthreads();
        if (grp) return;
        const float m1 = js[0], M = fmaxf(m, m1), f0 = __builtin_amdgcn_exp2f(m - M), f1 = __builtin_amdgcn_exp2f(m1 - M);
        l = l * f0 + js[256] * f1;
#pragma unroll
        for (int d = 0; d < NDT; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) ot[d][i] = ot[d][i] * f0 + js[(2 + 16 * d + i) * 256] * f1;
        unset = M <= M_NONE;
        m = M;
    }
    l += __shfl_xor(l, 32, 64);
    if (q0 + r >= nrows) return;
    const int row = row0 + q0 + r;
    if (slot >= 0) {                                       // register 4 x + j of ot[d] <-> dim 32 d + 8 x + 4 h + j
        const int64_t at = ((int64_t)row * p.H + head) * p.ns + slot;
#pragma unroll
        for (int d = 0; d < NDT; ++d)
#pragma unroll
            for (int x = 0; x < 4; ++x)
                *reinterpret_cast<f32x4*>(p.part_o + at * HD + 32 * d + 8 * x + 4 * h) =
                    f32x4{ot[d][4 * x], ot[d][4 * x + 1], ot[d][4 * x + 2], ot[d][4 * x + 3]};
        if (h == 0) {
            p.part_ml[at * 2] = unset ? M_NONE : m;
            p.part_ml[at * 2 + 1] = l;
        }
    } else {
        const float inv = inverse_sum(l);
        const int b = row / p.Nq, i = row - b * p.Nq;
        __bf16* op = p.O + (int64_t)b * p.bso + (int64_t)i * p.ldo + head * HD + 4 * h;
#pragma unroll
        for (int d = 0; d < NDT; ++d)
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                u32x2 w;
                w[0] = pack_bf16x2(ot[d][4 * x] * inv, ot[d][4 * x + 1] * inv);
                w[1] = pack_bf16x2(ot[d][4 * x + 2] * inv, ot[d][4 * x + 3] * inv);
                *reinterpret_cast<u32x2*>(op + 32 * d + 8 * x) = w;
            }
    }
}

// ---------------------------------------------------------------- joining the chunks
// One thread group's share of a row's slots (s0, s0 + SG, ...): running (M, l, o) in one pass over (m, l, o) of the slots.
template <int HD, int SG>
__device__ __forceinline__ void join_share(const float* mlp, const float* op, int s0, int ns, float& M, float& l, f32x4& o) {
    M = M_NONE;
    l = 0.f;
    o = f32x4{0.f, 0.f, 0.f, 0.f};
    constexpr int U = 4;                                   // slots in flight
    for (int s = s0; s < ns; s += U * SG) {
        float ms[U], ls[U];
        f32x4 x[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int at = min(s + u * SG, ns - 1);
            ms[u] = s + u * SG < ns ? mlp[2 * at] : M_NONE;
            ls[u] = s + u * SG < ns ? mlp[2 * at + 1] : 0.f;
            x[u] = *reinterpret_cast<const f32x4*>(op + (int64_t)at * HD);
        }
        float mn = M;
#pragma unroll
        for (int u = 0; u < U; ++u) mn = fmaxf(mn, ms[u]);
        float a = __builtin_amdgcn_exp2f(M - mn);
        M = mn;
        l *= a;
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] *= a;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            a = s + u * SG < ns ? __builtin_amdgcn_exp2f(ms[u] - M) : 0.f;
            l += a * ls[u];
#pragma unroll
            for (int i = 0; i < 4; ++i) o[i] += s + u * SG < ns ? a * x[u][i] : 0.f;
        }
    }
}
// o = sum_s o_s 2^(m_s - M) / sum_s l_s 2^(m_s - M), no key at all: zeros.  HD / 4 threads per row and slot group (four dims each),
// SG groups per row, joined in group order.
template <int HD, int SG>
__global__ __launch_bounds__(256) void hk_prefix_join_kernel(const PrefixParams p) {
    constexpr int TPR = HD / 4, RPB = 256 / (TPR * SG);
    __shared__ float ml[RPB * SG][2];
    __shared__ __attribute__((aligned(16))) float os[RPB * SG][HD];
    const int c = threadIdx.x % TPR, g = threadIdx.x / TPR, rl = g / SG;
    const int64_t rh = (int64_t)blockIdx.x * RPB + rl;
    const bool in = rh < (int64_t)p.R * p.H;
    const int64_t at = (in ? rh : 0) * p.ns;
    float M, l;
    f32x4 o;
    join_share<HD, SG>(p.part_ml + at * 2, p.part_o + at * HD + 4 * c, g % SG, p.ns, M, l, o);
    if (SG > 1) {
        if (c == 0) {
            ml[g][0] = M;
            ml[g][1] = l;
        }
        *reinterpret_cast<f32x4*>(&os[g][4 * c]) = o;
        __syncthreads();
        if (g % SG) return;
        M = M_NONE;
#pragma unroll
        for (int x = 0; x < SG; ++x) M = fmaxf(M, ml[g + x][0]);
        l = 0.f;
        o = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int x = 0; x < SG; ++x) {
            const float a = __builtin_amdgcn_exp2f(ml[g + x][0] - M);
            l += a * ml[g + x][1];
#pragma unroll
            for (int i = 0; i < 4; ++i) o[i] += a * os[g + x][4 * c + i];
        }
    }
    if (!in) return;
    const float inv = inverse_sum(l);
    const int row = (int)(rh / p.H), head = (int)(rh - (int64_t)row * p.H);
    const int b = row / p.Nq, i = row - b * p.Nq;
    u32x2 w;
    w[0] = pack_bf16x2(o[0] * inv, o[1] * inv);
    w[1] = pack_bf16x2(o[2] * inv, o[3] * inv);
    *reinterpret_cast<u32x2*>(p.O + (int64_t)b * p.bso + (int64_t)i * p.ldo + head * HD + 4 * c) = w;
}

// The same for one decode step, and its weights from the scores the first launch left.  One workgroup per (sequence, head) and 2048 keys; all
// its groups share the slots.
template <int HD>
__global__ __launch_bounds__(256) void hk_step_join_kernel(const PrefixParams p, const StepWeights sw) {
    constexpr int TPR = HD / 4, SG = 256 / TPR;
    __shared__ float ml[SG][2];
    __shared__ __attribute__((aligned(16))) float os[SG][HD];
    const int head = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, c = tid % TPR, g = tid / TPR;
    const int64_t rh = (int64_t)b * p.H + head, at = rh * p.ns;
    float M, l;
    f32x4 o;
    join_share<HD, SG>(p.part_ml + at * 2, p.part_o + at * HD + 4 * c, g, p.ns, M, l, o);
    if (c == 0) {
        ml[g][0] = M;
        ml[g][1] = l;
    }
    *reinterpret_cast<f32x4*>(&os[g][4 * c]) = o;
    __syncthreads();
    M = M_NONE;
    l = 0.f;
#pragma unroll
    for (int x = 0; x < SG; ++x) M = fmaxf(M, ml[x][0]);
#pragma unroll
    for (int x = 0; x < SG; ++x) l += __builtin_amdgcn_exp2f(ml[x][0] - M) * ml[x][1];
    const float inv = inverse_sum(l);
    if (blockIdx.z == 0 && g == 0) {
        o = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int x = 0; x < SG; ++x) {
            const float a = __builtin_amdgcn_exp2f(ml[x][0] - M);
#pragma unroll
            for (int i = 0; i < 4; ++i) o[i] += a * os[x][4 * c + i];
        }
        u32x2 w;
        w[0] = pack_bf16x2(o[0] * inv, o[1] * inv);
        w[1] = pack_bf16x2(o[2] * inv, o[3] * inv);
        *reinterpret_cast<u32x2*>(p.O + (int64_t)b * p.bso + head * HD + 4 * c) = w;
    }
    add_weights(p, sw, b, head, p.raw + rh * p.raw_ld, M, inv, blockIdx.z * 256 + tid, gridDim.z * 256);
}

// ---------------------------------------------------------------- host side
enum { ONCE, SMALL, MIXED, PACKED, FUSED };
struct Plan {
    int mode, rt, groups;            // groups: of four waves per workgroup of hk_prefix_rows_kernel, if two
    RowsParams rows;
};

// n chunks of `keys` such that `per` workgroups each come to about `want`; a chunk is whole multiples of `unit`, at most `most` keys.
int cut(int keys, int64_t per, int64_t want, int unit, int most, int* chunk) {
    *chunk = unit;
    if (keys <= 0) return 0;
    int64_t n = want / (per < 1 ? 1 : per);
    if (n < 1) n = 1;
    int64_t c = (keys + n - 1) / n;
    c = (c + unit - 1) / unit * unit;
    if (c > most) c = most;
    *chunk = (int)c;
    return (int)((keys + c - 1) / c);
}

// The same for 128-row blocks: the nearest count to ROWS_WANT, but two chunks rather than one wherever a launch leaves CUs without a block.
// Measured, 32 heads of 128 (us at so many chunks): 1 block of rows over 16384 keys 187 / 158 / 160 / 161 at 4 / 8 / 12 / 16, 2 over 1201
// 22.9 / 21.8 / 21.8 / 22.9 at 2 / 3 / 4 / 5, 3 over 1985 48 / 33 / 28 / 31 at 1 / 2 / 3 / 4, 5 over 1201 37 / 32 / 36 at 1 / 2 / 3, 6 over
// 2500 62 / 53 / 65 at 1 / 2 / 3; 8 heads of 64, 13 blocks over 1500 32 / 25 / 27 at 1 / 2 / 3.
int cut_rows(int keys, int64_t per, int* chunk) {
    int64_t n = (ROWS_WANT + per / 2) / per;
    if (n < 2 && per < ROWS_WANT) n = 2;
    return cut(keys, per, per * n, KT, 1 << 28, chunk);
}

// Which kernel takes what.  Up to 32 queries per sequence, own keys are bound by reading them: hk_prefix_part_kernel.  So is the prefix as long
// as few rows share it (SMALL); beyond, its rows fill 128-row blocks (MIXED).  More queries: hk_prefix_rows_kernel for both, in one
// workgroup (FUSED) or apart (PACKED), whichever the estimate below finds shorter.
Plan make_plan(PrefixParams& p, int hd, bool raw) {
    Plan m = {};
    p.R = p.B * p.Nq;
    m.rt = !raw && (p.Nq > 16 || (p.P > 0 && p.R > 16)) ? 2 : 1;
    m.rows.npb = (p.R + RB - 1) / RB;
    m.rows.nob = (p.Nq + RB - 1) / RB;
    p.nprg = (p.R + m.rt * 16 - 1) / (m.rt * 16);
    p.norg = (p.Nq + m.rt * 16 - 1) / (m.rt * 16);
    const int64_t H = p.H, B = p.B;
    // One launch, a workgroup per (sequence, head) for all its keys, or chunks and a join?  Measured in a graph, 32 heads of 128 (us, one : two
    // launches).  One sequence, 55 / 372 / 520 / 720 keys: 4.6 : 6.3, 7.3 : 6.8, 8.8 : 7.0, 10.8 : 7.1 - and the second launch and the workspace
    // cost the host 4.3, so up to 1.5 are given for them.  The prefix is
    // read once per sequence here: 16 sequences over 352 + 20 keys 13.0 : 8.8.  Heads of 64, 55 / 520 / 700 / 907 keys: 4.0 : 5.8, 6.0 : 6.5, 6.9 : 6.6,
    // 8.0 : 6.7 (16 waves instead of eight: 0.2 more).  Without one nothing is read twice, and 256 pairs fill the
    // chip: 8 sequences' step over 353 / 1000 keys 11.3 : 15.8, 23.5 : 26.3; 4 sequences' over 1000 15.9 : 18.4, one's 13.7 : 8.0; 32 sequences'
    // over 100 20.7 : 16.6.
    const int64_t pairs = H * B, keys = (int64_t)p.P + p.Nk;
    if (p.Nq <= 16 && (p.P > 0 ? pairs <= 256 && keys * hd <= 480 * 128 : pairs <= 512 && (keys <= 384 || (pairs >= 128 && keys <= MAX_CHUNK)))) {
        m.mode = ONCE;
        m.rt = 1;
        p.norg = 1;
        p.ns = 0;
        return m;
    }
    if (p.Nq <= 32) {
        // hk_prefix_part_kernel goes over the prefix again for every 32 rows, hk_prefix_rows_kernel for every 128, but is a launch more and
        // leaves blocks part empty.  SMALL : MIXED, 32 heads of 128 (us): 64 rows over 1000 / 1985 / 16384 keys 27.5 : 31.5, 36.4 : 34.4, 153 : 136;
        // 128 rows over 200 / 1000 / 1985 15.0 : 21.4, 27.2 : 27.0, 35.0 : 27.8; 256 over 200 / 1000 19.2 : 29.4, 37.5 : 30.9;
        // heads of 64, 128 rows over 1000 / 4096 16.9 : 19.0, 31.5 : 25.1.
        const int64_t again = ((p.R + 31) / 32 - m.rows.npb) * (int64_t)p.P * hd * H;
        m.mode = again >= 9600000 ? MIXED : SMALL;
        if (m.mode == SMALL) p.npc = cut(p.P, H * p.nprg, PART_WANT, NWV * TK, MAX_CHUNK, &p.pc);
        else p.npc = cut_rows(p.P, H * m.rows.npb, &p.pc);
        if (m.mode == MIXED && p.Nq <= 16) {               // 16 rows are enough for the own keys then
            m.rt = 1;
            p.norg = 1;
        }
        p.noc = cut(p.Nk, B * H * p.norg, PART_WANT, NWV * TK, MAX_CHUNK, &p.oc);
        // Own keys by wave: nothing of a workgroup is idle where they are few, but a wave walks them alone.  By workgroup : by wave, 32 heads of 128, prefix of
        // 1985 (us): 16 sequences' 20 / 61 / 100 own keys 14.1 : 13.7, 15.3 : 15.3, 16.6 : 17.6, 32 sequences' 21.6 : 17.3, 22.1 : 19.9, 25.0 : 24.3, 64
        // sequences' 35 : 28, 36 : 33, 41 : 40; 128 own keys 43 : 44; heads of 64, 32 sequences' 14.1 : 11.7, 14.3 : 12.4, 15.5 : 14.5.
        p.by_wave = !raw && p.noc == 1 && p.Nk <= 96 && B * H * p.norg >= 1024;
    } else {
        // time of a 128-row x 64-key tile when 512 workgroups (two per CU) run: about 1 us; a lone workgroup's is not much shorter
        p.npc = cut_rows(p.P, H * m.rows.npb, &p.pc);
        p.noc = cut_rows(p.Nk, H * B * m.rows.nob, &p.oc);
        const double own = (double)H * B * m.rows.nob * ((p.Nk + KT - 1) / KT), pre = (double)((p.P + KT - 1) / KT);
        const double fused_n = (double)H * B * m.rows.nob;
        double fused = (own + fused_n * pre) / (fused_n < 512 ? fused_n : 512);
        // Two groups of waves where CUs would be idle.  One : two, 32 heads of 128 (us): one sequence's 37 rows over 100 / 350 / 1201 9.5 : 9.7, 13.8 : 13.1,
        // 28.2 : 22.9, 200 over 350 18.9 : 16.7, 512 over 1400 43.5 : 36.2; chunks of a prefix (PACKED), 37 rows over 350 / 1201 11.2 : 12.5, 13.4 : 14.5.
        const bool two = fused_n <= 256 && (p.P + KT - 1) / KT + (p.Nk + KT - 1) / KT >= 6;
        if (two) fused = 0.8 * fused + 1.0;
        const double packed_n = (double)H * m.rows.npb * p.npc + (double)H * B * m.rows.nob * p.noc;
        double packed = (own + (double)H * m.rows.npb * pre) / (packed_n < 512 ? packed_n : 512);
        packed += 4.0 + (double)p.R * H * (p.npc + p.noc) * hd * 8 / 4.5e6;      // the join: a launch, partial sums written and read at 4.5 TB/s
        m.mode = p.P > 0 && packed < fused ? PACKED : FUSED;
        if (p.P == 0 && packed < fused && p.noc > 1) m.mode = PACKED;
        if (m.mode == FUSED && two) m.groups = 2;
    }
    m.rows.packed = m.mode != FUSED;
    m.rows.pjobs = m.mode == MIXED || m.mode == PACKED ? H * m.rows.npb * p.npc : 0;
    p.pjobs = m.mode == SMALL ? H * p.npc * p.nprg : 0;
    p.ns = m.mode == FUSED ? 0 : p.npc + p.noc;
    return m;
}

size_t up16(size_t x) { return (x + 15) / 16 * 16; }
size_t part_bytes(const PrefixParams& p, int hd) {
    return p.ns == 0 ? HK_NO_WS : up16((size_t)p.ns * p.R * p.H * hd * 4) + up16((size_t)p.ns * p.R * p.H * 8);
}
size_t step_bytes(const PrefixParams& p, int hd) {      // chunks, and every key's score (one launch keeps those in LDS)
    return part_bytes(p, hd) + (p.ns == 0 ? 0 : (size_t)p.B * p.H * p.raw_ld * 4);
}
void set_parts(PrefixParams& p, void* ws, int hd) {
    p.part_o = reinterpret_cast<float*>(ws);
    p.part_ml = reinterpret_cast<float*>(reinterpret_cast<char*>(ws) + up16((size_t)p.ns * p.R * p.H * hd * 4));
}
int64_t part_grid(const PrefixParams& p) {
    const int64_t own = (int64_t)p.B * p.H * p.norg;
    return p.ns == 0 ? (int64_t)p.B * p.H : p.pjobs + (p.by_wave ? (own + NWV - 1) / NWV : own * p.noc);
}
int64_t rows_grid(const PrefixParams& p, const Plan& m) {
    const int64_t own = (int64_t)p.B * m.rows.nob * p.H;
    return m.mode == MIXED ? m.rows.pjobs : m.mode == PACKED ? m.rows.pjobs + own * p.noc : own;
}

template <int HD, int RT, bool BIAS, bool RAW>
void launch_part(const PrefixParams& p, hipStream_t s) {
    hipLaunchKernelGGL((hk_prefix_part_kernel<HD, RT, BIAS, RAW, NWV, false>), dim3((unsigned)part_grid(p)), dim3(NWV * 64), 0, s, p, StepWeights{});
}
template <int HD, bool RAW>
void launch_once(const PrefixParams& p, const StepWeights& sw, hipStream_t s) {
    const dim3 grid((unsigned)(p.B * p.H));
    if (p.bias) hipLaunchKernelGGL((hk_prefix_part_kernel<HD, 1, true, RAW, 8, true>), grid, dim3(512), 0, s, p, sw);
    else hipLaunchKernelGGL((hk_prefix_part_kernel<HD, 1, false, RAW, 8, true>), grid, dim3(512), 0, s, p, sw);
}
template <int HD, bool BIAS, int GRP, bool TWO>
int launch_rows_groups(const PrefixParams& p, const Plan& m, hipStream_t s) {
    constexpr int LDS = GRP * (2 * 2 * KT * HD * 2 + (BIAS ? 2 * KT * 4 : 0));
    static std::atomic<unsigned long long> attr_done{0};   // per device
    const hipError_t e = hk_lds_attr_once(attr_done, reinterpret_cast<const void*>(&hk_prefix_rows_kernel<HD, BIAS, GRP, TWO>), LDS);
    if (e != hipSuccess) {
        hk_set_error("hk_prefix_attn_bf16: hipFuncSetAttribute(%d B LDS): %s", LDS, hipGetErrorString(e));
        return HK_ELAUNCH;
    }
    hipLaunchKernelGGL((hk_prefix_rows_kernel<HD, BIAS, GRP, TWO>), dim3((unsigned)rows_grid(p, m)), dim3(GRP * 256), LDS, s, p, m.rows);
    return HK_OK;
}
template <int HD, bool BIAS>
int launch_rows(const PrefixParams& p, const Plan& m, hipStream_t s) {
    return m.groups == 2 ? launch_rows_groups<HD, BIAS, 2, false>(p, m, s) : launch_rows_groups<HD, BIAS, 1, false>(p, m, s);
}
template <int HD, int SG>
void launch_join(const PrefixParams& p, hipStream_t s) {
    const int64_t rh = (int64_t)p.R * p.H, per = 256 / (HD / 4 * SG);
    hipLaunchKernelGGL((hk_prefix_join_kernel<HD, SG>), dim3((unsigned)((rh + per - 1) / per)), dim3(256), 0, s, p);
}
template <int HD>
int launch_prefix(const PrefixParams& p, const Plan& m, hipStream_t s) {
    if (m.mode == ONCE) {
        launch_once<HD, false>(p, StepWeights{}, s);
        return HK_OK;
    }
    if (m.mode != SMALL) {
        // MIXED: the rows kernel reads the prefix only, which has no bias
        const int rc = m.mode == MIXED && p.Nq == 1 ? launch_rows_groups<HD, false, 1, true>(p, m, s)
                       : p.bias && m.mode != MIXED  ? launch_rows<HD, true>(p, m, s)
                                                    : launch_rows<HD, false>(p, m, s);
        if (rc != HK_OK || m.mode == FUSED) return rc;
    }
    if (m.mode != PACKED) {
        if (m.rt == 2) {
            if (p.bias) launch_part<HD, 2, true, false>(p, s);
            else launch_part<HD, 2, false, false>(p, s);
        } else {
            if (p.bias) launch_part<HD, 1, true, false>(p, s);
            else launch_part<HD, 1, false, false>(p, s);
        }
    }
    if (p.ns <= 4) launch_join<HD, 1>(p, s);
    else launch_join<HD, 4>(p, s);
    return HK_OK;
}
template <int HD>
void launch_step(const PrefixParams& p, const Plan& m, const StepWeights& sw, hipStream_t s) {
    if (m.mode == ONCE) {
        launch_once<HD, true>(p, sw, s);
        return;
    }
    if (p.bias) launch_part<HD, 1, true, true>(p, s);
    else launch_part<HD, 1, false, true>(p, s);
    const int z = p.Nk < 2048 * 64 ? (p.Nk + 2047) / 2048 : 64;
    hipLaunchKernelGGL((hk_step_join_kernel<HD>), dim3((unsigned)p.H, (unsigned)p.B, (unsigned)z), dim3(256), 0, s, p, sw);
}

bool shape_ok(int64_t B, int64_t H, int64_t Nq, int64_t P, int64_t Nk, int hd) {
    return B >= 1 && B < 65536 && H >= 1 && H < 65536 && Nq >= 1 && P >= 0 && Nk >= Nq && P < (1 << 28) && Nk < (1 << 28) &&
           (hd == 64 || hd == 128) && B * Nq * H < (1LL << 27);
}

}  // namespace

extern "C" size_t hk_prefix_attn_ws(int32_t B, int32_t H, int32_t Nq, int32_t P, int32_t Nk, int32_t head_dim) {
    if (!shape_ok(B, H, Nq, P, Nk, head_dim)) return 0;
    PrefixParams p = {};
    p.B = B;
    p.H = H;
    p.Nq = Nq;
    p.P = P;
    p.Nk = Nk;
    make_plan(p, head_dim, false);
    return part_bytes(p, head_dim);
}

extern "C" int hk_prefix_attn_bf16(const hk_prefix_attn_desc* d, void* stream) {
    HK_REQUIRE(d && d->Q && d->K && d->V && d->O, "hk_prefix_attn_bf16: null operand");
    HK_REQUIRE(shape_ok(d->B, d->H, d->Nq, d->P, d->Nk, d->head_dim),
               "hk_prefix_attn_bf16: bad shape B=%d H=%d Nq=%d P=%d Nk=%d head_dim=%d (head size 64 or 128, Nk >= Nq >= 1, P >= 0)", d->B,
               d->H, d->Nq, d->P, d->Nk, d->head_dim);
    HK_REQUIRE(d->P == 0 || (d->KP && d->VP), "hk_prefix_attn_bf16: null prefix");
    const int64_t row = (int64_t)d->H * d->head_dim;
    HK_REQUIRE(((d->ldq | d->bsq | d->ldkp | d->ldvp | d->ldk | d->bsk | d->ldv | d->bsv) & 7) == 0 && ((d->ldo | d->bso) & 3) == 0,
               "hk_prefix_attn_bf16: strides must keep 16-byte rows (8 elements; 4 for the output)");
    HK_REQUIRE(d->ldkp < (1 << 25) && d->ldvp < (1 << 25) && d->ldk < (1 << 25) && d->ldv < (1 << 25),
               "hk_prefix_attn_bf16: token strides of 2^25 elements and more are not supported");
    HK_REQUIRE(d->ldq >= 0 && d->ldkp >= 0 && d->ldvp >= 0 && d->ldk >= 0 && d->ldv >= 0 && d->bsq >= 0 && d->bsk >= 0 && d->bsv >= 0 &&
                   hk_rows_apart(d->B, d->bso, d->Nq, d->ldo, row) && d->bias_bs >= 0,
               "hk_prefix_attn_bf16: strides must not be negative, output rows must not overlap");
    HK_REQUIRE(((uintptr_t)d->Q | (uintptr_t)d->KP | (uintptr_t)d->VP | (uintptr_t)d->K | (uintptr_t)d->V | (uintptr_t)d->ws) % 16 == 0 &&
                   (uintptr_t)d->O % 8 == 0 && (uintptr_t)d->key_bias % 4 == 0,
               "hk_prefix_attn_bf16: operands must be 16-byte aligned");
    PrefixParams p = {};
    p.Q = reinterpret_cast<const __bf16*>(d->Q);
    p.KP = reinterpret_cast<const __bf16*>(d->KP);
    p.VP = reinterpret_cast<const __bf16*>(d->VP);
    p.K = reinterpret_cast<const __bf16*>(d->K);
    p.V = reinterpret_cast<const __bf16*>(d->V);
    p.O = reinterpret_cast<__bf16*>(d->O);
    p.bias = d->key_bias;
    p.B = d->B;
    p.H = d->H;
    p.Nq = d->Nq;
    p.P = d->P;
    p.Nk = d->Nk;
    p.ldq = d->ldq;
    p.bsq = d->bsq;
    p.ldkp = d->ldkp;
    p.ldvp = d->ldvp;
    p.ldk = d->ldk;
    p.bsk = d->bsk;
    p.ldv = d->ldv;
    p.bsv = d->bsv;
    p.ldo = d->ldo;
    p.bso = d->bso;
    p.bias_bs = d->bias_bs;
    const Plan m = make_plan(p, d->head_dim, false);
    HK_REQUIRE(p.ns == 0 || (d->ws && d->ws_bytes >= part_bytes(p, d->head_dim)),
               "hk_prefix_attn_bf16: workspace of %zu bytes, %zu needed (hk_prefix_attn_ws)", d->ws ? d->ws_bytes : (size_t)0,
               part_bytes(p, d->head_dim));
    HK_REQUIRE(part_grid(p) < (1LL << 31) && rows_grid(p, m) < (1LL << 31), "hk_prefix_attn_bf16: grid too large");
    {
        const HkSpan o = hk_span(p.O, p.B, p.bso, p.Nq, p.ldo, row, 2), w = hk_span(p.ns ? d->ws : nullptr, 1, 0, 1, 0, (int64_t)part_bytes(p, d->head_dim), 1);
        const HkSpan in[] = {hk_span(p.KP, 1, 0, p.P, p.ldkp, row, 2), hk_span(p.VP, 1, 0, p.P, p.ldvp, row, 2),
                             hk_span(p.K, p.B, p.bsk, p.Nk, p.ldk, row, 2), hk_span(p.V, p.B, p.bsv, p.Nk, p.ldv, row, 2),
                             hk_span(p.bias, p.B, p.bias_bs, 1, 0, p.Nk, 4), hk_span(p.Q, p.B, p.bsq, p.Nq, p.ldq, row, 2)};
        for (int i = 0; i < 6; ++i)
            HK_REQUIRE(!hk_overlap(w, in[i]) && !hk_overlap(o, in[i]), "hk_prefix_attn_bf16: the output or the workspace overlaps an input");
        HK_REQUIRE(!hk_overlap(o, w), "hk_prefix_attn_bf16: the output overlaps the workspace");
    }
    set_parts(p, d->ws, d->head_dim);
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    const int rc = d->head_dim == 128 ? launch_prefix<128>(p, m, s) : launch_prefix<64>(p, m, s);
    if (rc != HK_OK) return rc;
    HK_CHECK_LAUNCH("hk_prefix_attn_bf16");
    return HK_OK;
}

extern "C" size_t hk_decode_attn_weights_ws(int32_t B, int32_t H, int32_t head_dim, int32_t n_keys) {
    if (!shape_ok(B, H, 1, 0, n_keys, head_dim)) return 0;
    PrefixParams p = {};
    p.B = B;
    p.H = H;
    p.Nq = 1;
    p.Nk = n_keys;
    p.raw_ld = (n_keys + TK - 1) / TK * TK;
    make_plan(p, head_dim, true);
    return step_bytes(p, head_dim);
}

extern "C" int hk_decode_attn_weights_bf16(const hk_step_weights_desc* d, void* stream) {
    HK_REQUIRE(d && d->q && d->k_cache && d->v_cache && d->out && d->w_out, "hk_decode_attn_weights_bf16: null operand");
    HK_REQUIRE(shape_ok(d->B, d->H, 1, 0, d->n_keys, d->head_dim) && d->n_keys <= d->cache_rows,
               "hk_decode_attn_weights_bf16: bad shape B=%d H=%d head_dim=%d n_keys=%d cache_rows=%ld", d->B, d->H, d->head_dim, d->n_keys,
               (long)d->cache_rows);
    HK_REQUIRE(((uintptr_t)d->q | (uintptr_t)d->k_cache | (uintptr_t)d->v_cache | (uintptr_t)d->ws) % 16 == 0 && (uintptr_t)d->out % 8 == 0 &&
                   ((uintptr_t)d->w_in | (uintptr_t)d->w_out | (uintptr_t)d->key_bias) % 4 == 0,
               "hk_decode_attn_weights_bf16: operands must be 16-byte aligned");
    HK_REQUIRE(hk_rows_apart(d->B, d->wo_bs, d->H, d->wo_hs, d->n_keys) && d->wi_bs >= 0 && d->wi_hs >= 0 && d->bias_bs >= 0 && d->bias_hs >= 0,
               "hk_decode_attn_weights_bf16: rows of w_out must not overlap, strides must not be negative");
    HK_REQUIRE(d->w_in != d->w_out || (d->wi_bs == d->wo_bs && d->wi_hs == d->wo_hs),
               "hk_decode_attn_weights_bf16: weights updated in place must have one layout");
    const int64_t D = (int64_t)d->H * d->head_dim;
    PrefixParams p = {};
    p.Q = reinterpret_cast<const __bf16*>(d->q);
    p.K = reinterpret_cast<const __bf16*>(d->k_cache);
    p.V = reinterpret_cast<const __bf16*>(d->v_cache);
    p.O = reinterpret_cast<__bf16*>(d->out);
    p.bias = d->key_bias;
    p.B = d->B;
    p.H = d->H;
    p.Nq = 1;
    p.Nk = d->n_keys;
    p.ldq = p.bsq = p.ldo = p.bso = p.ldk = p.ldv = D;
    p.bsk = p.bsv = d->cache_rows * D;
    p.bias_bs = d->bias_bs;
    p.bias_hs = d->bias_hs;
    p.raw_ld = (d->n_keys + TK - 1) / TK * TK;
    const Plan m = make_plan(p, d->head_dim, true);
    const size_t need = step_bytes(p, d->head_dim);
    HK_REQUIRE(p.ns == 0 || (d->ws && d->ws_bytes >= need), "hk_decode_attn_weights_bf16: workspace of %zu bytes, %zu needed (hk_decode_attn_weights_ws)",
               d->ws ? d->ws_bytes : (size_t)0, need);
    HK_REQUIRE(part_grid(p) < (1LL << 31), "hk_decode_attn_weights_bf16: grid too large");
    {
        const HkSpan wo = hk_span(d->w_out, p.B, d->wo_bs, p.H, d->wo_hs, p.Nk, 4), o = hk_span(p.O, p.B, D, 1, 0, D, 2),
                     w = hk_span(p.ns ? d->ws : nullptr, 1, 0, 1, 0, (int64_t)need, 1);
        const HkSpan in[] = {hk_span(p.Q, p.B, D, 1, 0, D, 2), hk_span(p.K, p.B, p.bsk, p.Nk, D, D, 2), hk_span(p.V, p.B, p.bsv, p.Nk, D, D, 2),
                             hk_span(p.bias, p.B, p.bias_bs, p.H, p.bias_hs, p.Nk, 4),
                             d->w_in == d->w_out ? HkSpan{} : hk_span(d->w_in, p.B, d->wi_bs, p.H, d->wi_hs, p.Nk, 4)};
        for (int i = 0; i < 5; ++i)
            HK_REQUIRE(!hk_overlap(wo, in[i]) && !hk_overlap(o, in[i]) && !hk_overlap(w, in[i]),
                       "hk_decode_attn_weights_bf16: an output or the workspace overlaps an input");
        HK_REQUIRE(!hk_overlap(o, wo) && !hk_overlap(o, w) && !hk_overlap(wo, w), "hk_decode_attn_weights_bf16: outputs and workspace overlap");
    }
    set_parts(p, d->ws, d->head_dim);
    p.raw = reinterpret_cast<float*>(reinterpret_cast<char*>(d->ws) + part_bytes(p, d->head_dim));
    StepWeights sw = {d->w_in, d->w_out, d->wi_bs, d->wi_hs, d->wo_bs, d->wo_hs};
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    if (d->head_dim == 128) launch_step<128>(p, m, sw, s);
    else launch_step<64>(p, m, sw, s);
    HK_CHECK_LAUNCH("hk_decode_attn_weights_bf16");
    return HK_OK;
}
