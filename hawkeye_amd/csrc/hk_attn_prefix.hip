// Attention of a batch whose sequences share one prefix, and the decode step that adds its softmax weights to what the keys
// have collected.  Both are bound by reading K and V: the prefix's rows are read once for ALL rows of the batch.
//
//   s_j = q . k_j (+ bias_j log2 e),  p_j = 2^(s_j - M),  o = sum_j p_j v_j / sum_j p_j
//
// over the prefix's keys and the row's own; softmax sums are associative, so the keys are cut into chunks, a chunk leaves
// (m, l, o) = (its maximum, sum_j 2^(s_j - m), sum_j 2^(s_j - m) v_j) in 32 bits, and a second launch joins the chunks of a
// row in index order (bit-reproducible).
//
// hk_prefix_part_kernel: a workgroup = one (head, key chunk, group of query rows).  Prefix chunks take rows of ALL
// sequences (row r = sequence r / Nq, token r % Nq), a sequence's own chunks take its Nq rows.  Its four waves walk 32-key tiles
// of the chunk, each for itself:
//   S^T = K . Q^T  (v_mfma_f32_16x16x32_bf16: 16 keys x 16 rows; lane -> row lane & 15, keys 4 (lane >> 4) + i)
//   O^T += V^T . P^T, where the S^T accumulators of two 16-key blocks ARE the B operand (contraction index 8 q + j <-> key
//   4 q + j of block 0, j < 4, or 4 q + j - 4 of block 1), and V^T comes in that key order from ds_read_b64_tr_b16.
// K goes from memory straight to the A operand's registers, V through 32 keys of LDS that belong to the wave (no barrier in
// the loop).  The next tile's K is requested as soon as this one's scores stand, its V as soon as this one's is in LDS: a
// wave keeps about 16 KB in flight, 8 waves per CU.
#include "hk_common.h"

namespace {

constexpr float REMOVED = -1.0e4f;   // a key whose bias is at or below this does not exist (the framework's mask value)
constexpr float M_NONE = -1.0e30f;   // running maximum of a row that has met no key
constexpr int TK = 32;               // keys per tile
constexpr int NWV = 4;               // waves per workgroup
constexpr int MAX_CHUNK = 1024;      // keys per chunk at most: the chunk's bias lives in LDS

struct PrefixParams {
    const __bf16 *Q, *KP, *VP, *K, *V;
    __bf16* O;
    const float* bias;               // own keys: bias[b * bias_bs + h * bias_hs + j]
    float* part_o;                   // [slot][row][head][HD]
    float* part_ml;                  // [slot][row][head][2]
    float* raw;                      // WEIGHTS: scores [B][H][raw_ld], raw_ld = Nk rounded up to whole tiles
    int B, H, Nq, P, Nk, R;          // R = B * Nq
    int64_t ldq, bsq, ldkp, ldvp, ldk, bsk, ldv, bsv, ldo, bso, bias_bs, bias_hs, raw_ld;
    int pc, npc, nprg;               // prefix: keys per chunk, chunks, row groups
    int oc, noc, norg;               // own keys: the same, per sequence
    int64_t pjobs;                   // workgroups of the prefix: H * npc * nprg (below 2^31 once checked)
};

__device__ __forceinline__ void wave_lds_sync() {   // LDS written by this wave's lanes is read by its other lanes
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

template <int HD, int RT, bool BIAS, bool RAW>
__global__ __launch_bounds__(NWV * 64, 2) void hk_prefix_part_kernel(const PrefixParams p) {
    constexpr int CH = HD / 8;            // 16-byte chunks per key row
    constexpr int KS = HD / 32;           // contraction steps of S^T
    constexpr int DT = HD / 16;           // 16-dim blocks of O^T
    constexpr int RPL = 64 / CH;          // key rows one 64-lane load covers
    constexpr int NL = TK / RPL;          // loads per lane for a tile of V
    constexpr int VB = TK * HD * 2;       // bytes of a wave's V tile
    constexpr int OB = RT * 16 * HD * 4;  // bytes of a wave's O block at the end
    constexpr int WB = VB > OB ? VB : OB;
    __shared__ __attribute__((aligned(16))) char vlds[NWV * WB];
    __shared__ float ml[NWV][RT * 16][2];
    __shared__ __attribute__((aligned(16))) float blds[BIAS ? MAX_CHUNK : 4];

    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int l15 = lane & 15, quad = lane >> 4;

    // ---- which rows, which keys ----
    int head, row0, nrows, k0, k1, slot, lim0 = 0x3fffffff, brow = 0;
    const __bf16 *kb, *vb;
    int64_t ldk, ldv;
    bool shared_keys;
    if (blockIdx.x < p.pjobs) {      // row groups of one (head, chunk) follow each other: the later ones find K and V in L2
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
        int j = (int)(blockIdx.x - p.pjobs);
        const int rg = j % p.norg;
        j /= p.norg;
        head = j % p.H;
        j /= p.H;
        brow = j / p.noc;
        const int c = j - brow * p.noc;
        slot = p.npc + c;
        k0 = c * p.oc;
        k1 = min(k0 + p.oc, p.Nk);
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
    if (has_bias) {
        const float* bp = p.bias + (int64_t)brow * p.bias_bs + (int64_t)head * p.bias_hs;
        for (int i = tid; i < MAX_CHUNK && k0 + i < k1; i += NWV * 64) blds[i] = bp[k0 + i];
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
#pragma unroll
        for (int g = 0; g < 2; ++g) {
            const __bf16* kp = kb + (int64_t)min(k0 + t * TK + 16 * g + l15, k1 - 1) * ldk + 8 * quad;
#pragma unroll
            for (int s = 0; s < KS; ++s) kr[g][s] = *reinterpret_cast<const bf16x8*>(kp + 32 * s);
        }
    };
    auto load_v = [&](int t) {
#pragma unroll
        for (int i = 0; i < NL; ++i)
            vr[i] = *reinterpret_cast<const u32x4*>(vb + (int64_t)min(k0 + t * TK + i * RPL + vrow, k1 - 1) * ldv + vch * 8);
    };
    // 16-byte chunk c of key row r lives at chunk c ^ swz(r): the 16 key rows x 32 bytes of one transposing read then touch every
    // bank twice, the least there is (512 bytes at 128 a cycle)
    auto swz = [](int r) { return HD == 128 ? (r & 7) << 1 : ((r >> 1) & 3) << 1; };
    char* vw = vlds + wave * WB;
    const int trow = 4 * quad + (l15 >> 2);               // transposing read: this lane's key row (and + 16), 8 bytes of it
    int toff[DT];
#pragma unroll
    for (int d = 0; d < DT; ++d) toff[d] = trow * HD * 2 + (((2 * d + ((lane & 3) >> 1)) ^ swz(trow)) << 4) + 8 * (lane & 1);

    const int nt = k1 > k0 ? (k1 - k0 + TK - 1) / TK : 0;
    if (wave < nt) {
        load_k(wave);
        load_v(wave);
    }
    for (int t = wave; t < nt; t += NWV) {
        f32x4 st[RT][2];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
            for (int g = 0; g < 2; ++g) {
                st[rt][g] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int s = 0; s < KS; ++s) st[rt][g] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kr[g][s], qf[rt][s], st[rt][g], 0, 0, 0);
            }
        const bool more = t + NWV < nt;
        if (more) load_k(t + NWV);
        // ---- bias, removed and invisible keys ----
        const int kt = k0 + t * TK;
        uint32_t gone = 0;                                // keys of this tile that no row has: their V rows are made zero
        if (has_bias) {
            const bool rem = lane < TK && (kt + lane >= k1 || blds[t * TK + lane] <= REMOVED);
            gone = (uint32_t)__builtin_amdgcn_ballot_w64(rem);
#pragma unroll
            for (int g = 0; g < 2; ++g) {
                const f32x4 bv = *reinterpret_cast<const f32x4*>(blds + t * TK + 16 * g + 4 * quad);
#pragma unroll
                for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        st[rt][g][i] = (gone >> (16 * g + 4 * quad + i)) & 1 ? -INFINITY : st[rt][g][i] + bv[i] * HK_LOG2E;
            }
        } else if (kt + TK > k1) {
            gone = 0xffffffffu << (k1 - kt);              // k1 - kt is 1 .. 31 here
        }
        if (kt + TK > k1 || kt + TK - 1 > lim0) {
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                const int lim = min(k1 - 1, lim0 + rt * 16 + l15);
#pragma unroll
                for (int g = 0; g < 2; ++g)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (kt + 16 * g + 4 * quad + i > lim) st[rt][g][i] = -INFINITY;
            }
        }
        if (RAW && l15 == 0) {                            // one row: its scores, for the weights
            float* rp = p.raw + ((int64_t)brow * p.H + head) * p.raw_ld + kt;
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
        // P in bf16 (the matrix instruction's operand): half a step of 2^-9 each; the sum l is of the unrounded values
        bf16x8 pf[RT];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            float e[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                e[i] = __builtin_amdgcn_exp2f(st[rt][i >> 2][i & 3] - m[rt]);
                l[rt] += e[i];
            }
            u32x4 w;
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = pack_bf16x2(e[2 * i], e[2 * i + 1]);
            pf[rt] = __builtin_bit_cast(bf16x8, w);
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
        if (more) load_v(t + NWV);
#pragma unroll
        for (int d = 0; d < DT; ++d) {
            const bf16x4 v0 = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((__attribute__((address_space(3))) bf16x4*)(vw + toff[d]));
            const bf16x4 v1 = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((__attribute__((address_space(3))) bf16x4*)(vw + toff[d] + 16 * HD * 2));
            bf16x8 vf;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                vf[i] = v0[i];
                vf[i + 4] = v1[i];
            }
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) ot[rt][d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, pf[rt], ot[rt][d], 0, 0, 0);
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
    for (int r = tid / TPR; r < nrows; r += NWV * 64 / TPR) {
        const int c = tid % TPR;
        float M = ml[0][r][0];
#pragma unroll
        for (int w = 1; w < NWV; ++w) M = fmaxf(M, ml[w][r][0]);
        f32x4 o = {0.f, 0.f, 0.f, 0.f};
        float ls = 0.f;
#pragma unroll
        for (int w = 0; w < NWV; ++w) {
            const float a = __builtin_amdgcn_exp2f(ml[w][r][0] - M);
            const f32x4 x = *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(vlds + w * WB) + r * HD + ((c ^ (r & 7)) << 2));
            ls += a * ml[w][r][1];
#pragma unroll
            for (int i = 0; i < 4; ++i) o[i] += a * x[i];
        }
        const int64_t at = ((int64_t)slot * p.R + row0 + r) * p.H + head;
        *reinterpret_cast<f32x4*>(p.part_o + at * HD + 4 * c) = o;
        if (c == 0) {
            p.part_ml[at * 2] = M;
            p.part_ml[at * 2 + 1] = ls;
        }
    }
}

// Joins the chunks of a row: o = sum_s o_s 2^(m_s - M) / sum_s l_s 2^(m_s - M), slots in index order; no key at all: zeros.
template <int HD>
__global__ __launch_bounds__(256) void hk_prefix_join_kernel(const PrefixParams p) {
    constexpr int TPR = HD / 4;
    const int64_t rh = (int64_t)blockIdx.x * (256 / TPR) + threadIdx.x / TPR;
    if (rh >= (int64_t)p.R * p.H) return;
    const int c = threadIdx.x % TPR;
    const int row = (int)(rh / p.H), head = (int)(rh - (int64_t)row * p.H);
    const int ns = p.npc + p.noc;
    const int64_t step = (int64_t)p.R * p.H;
    const float* mlp = p.part_ml + rh * 2;
    const float* op = p.part_o + rh * HD + 4 * c;
    float M = M_NONE;
    for (int s = 0; s < ns; ++s) M = fmaxf(M, mlp[s * step * 2]);
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    float l = 0.f;
    for (int s = 0; s < ns; ++s) {
        const float a = __builtin_amdgcn_exp2f(mlp[s * step * 2] - M);
        const f32x4 x = *reinterpret_cast<const f32x4*>(op + s * step * HD);
        l += a * mlp[s * step * 2 + 1];
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] += a * x[i];
    }
    const float inv = l > 0.f ? 1.0f / l : (l == 0.f ? 0.f : l);      // l NaN stays NaN
    const int b = row / p.Nq, i = row - b * p.Nq;
    u32x2 w;
    w[0] = pack_bf16x2(o[0] * inv, o[1] * inv);
    w[1] = pack_bf16x2(o[2] * inv, o[3] * inv);
    *reinterpret_cast<u32x2*>(p.O + (int64_t)b * p.bso + (int64_t)i * p.ldo + head * HD + 4 * c) = w;
}

// The same for one decode step, and its weights: w_out[j] = w_in[j] + 2^(s_j - M) / l from the scores the first launch left.
struct StepWeights {
    const float* w_in;               // may be w_out; NULL = zeros
    float* w_out;
    int64_t wi_bs, wi_hs, wo_bs, wo_hs;
};
template <int HD>
__global__ __launch_bounds__(256) void hk_step_join_kernel(const PrefixParams p, const StepWeights sw) {
    constexpr int TPR = HD / 4;
    const int head = blockIdx.x, b = blockIdx.y, tid = threadIdx.x;
    const int64_t rh = (int64_t)b * p.H + head, step = (int64_t)p.R * p.H;
    const float* mlp = p.part_ml + rh * 2;
    float M = M_NONE, l = 0.f;
    for (int s = 0; s < p.noc; ++s) M = fmaxf(M, mlp[s * step * 2]);
    for (int s = 0; s < p.noc; ++s) l += mlp[s * step * 2 + 1] * __builtin_amdgcn_exp2f(mlp[s * step * 2] - M);
    const float inv = l > 0.f ? 1.0f / l : (l == 0.f ? 0.f : l);
    if (blockIdx.z == 0 && tid < TPR) {
        f32x4 o = {0.f, 0.f, 0.f, 0.f};
        for (int s = 0; s < p.noc; ++s) {
            const float a = __builtin_amdgcn_exp2f(mlp[s * step * 2] - M);
            const f32x4 x = *reinterpret_cast<const f32x4*>(p.part_o + (rh + s * step) * HD + 4 * tid);
#pragma unroll
            for (int i = 0; i < 4; ++i) o[i] += a * x[i];
        }
        u32x2 w;
        w[0] = pack_bf16x2(o[0] * inv, o[1] * inv);
        w[1] = pack_bf16x2(o[2] * inv, o[3] * inv);
        *reinterpret_cast<u32x2*>(p.O + (int64_t)b * p.bso + head * HD + 4 * tid) = w;
    }
    const float* rp = p.raw + rh * p.raw_ld;
    const float* wi = sw.w_in ? sw.w_in + (int64_t)b * sw.wi_bs + (int64_t)head * sw.wi_hs : nullptr;
    float* wo = sw.w_out + (int64_t)b * sw.wo_bs + (int64_t)head * sw.wo_hs;
    for (int j = blockIdx.z * 256 + tid; j < p.Nk; j += gridDim.z * 256)
        wo[j] = (wi ? wi[j] : 0.f) + __builtin_amdgcn_exp2f(rp[j] - M) * inv;
}

// How the keys are cut: the whole chip wants about `want` workgroups, a chunk is whole 128-key rounds of the four waves.
int cut(int keys, long rows_x_heads, long want, int* chunk) {
    if (keys <= 0) {
        *chunk = NWV * TK;
        return 0;
    }
    long n = want / (rows_x_heads < 1 ? 1 : rows_x_heads);
    if (n < 1) n = 1;
    long c = (keys + n - 1) / n;
    c = (c + NWV * TK - 1) / (NWV * TK) * (NWV * TK);
    if (c > MAX_CHUNK) c = MAX_CHUNK;
    *chunk = (int)c;
    return (int)((keys + c - 1) / c);
}

int plan(PrefixParams& p, int rt) {
    const long want = 1024;
    p.R = p.B * p.Nq;
    p.nprg = (p.R + rt * 16 - 1) / (rt * 16);
    p.norg = (p.Nq + rt * 16 - 1) / (rt * 16);
    p.npc = cut(p.P, (long)p.H * p.nprg, want, &p.pc);
    p.noc = cut(p.Nk, (long)p.B * p.H * p.norg, want, &p.oc);
    p.pjobs = (int64_t)p.H * p.npc * p.nprg;
    return p.npc + p.noc;
}

int rows_tiles(int B, int Nq) { return B * Nq > 16 && Nq > 1 ? 2 : (B > 16 ? 2 : 1); }

size_t up16(size_t x) { return (x + 15) / 16 * 16; }
size_t part_bytes(const PrefixParams& p, int hd, int slots) {
    return up16((size_t)slots * p.R * p.H * hd * 4) + up16((size_t)slots * p.R * p.H * 8);
}
void set_parts(PrefixParams& p, void* ws, int hd, int slots) {
    p.part_o = reinterpret_cast<float*>(ws);
    p.part_ml = reinterpret_cast<float*>(reinterpret_cast<char*>(ws) + up16((size_t)slots * p.R * p.H * hd * 4));
}

template <int HD, int RT, bool BIAS, bool RAW>
void launch_part(const PrefixParams& p, hipStream_t s) {
    const int64_t grid = p.pjobs + (int64_t)p.B * p.noc * p.H * p.norg;
    hipLaunchKernelGGL((hk_prefix_part_kernel<HD, RT, BIAS, RAW>), dim3((unsigned)grid), dim3(NWV * 64), 0, s, p);
}
template <int HD>
void launch_prefix(const PrefixParams& p, int rt, hipStream_t s) {
    if (rt == 2) {
        if (p.bias) launch_part<HD, 2, true, false>(p, s);
        else launch_part<HD, 2, false, false>(p, s);
    } else {
        if (p.bias) launch_part<HD, 1, true, false>(p, s);
        else launch_part<HD, 1, false, false>(p, s);
    }
    const int64_t rh = (int64_t)p.R * p.H, per = 256 / (HD / 4);
    hipLaunchKernelGGL((hk_prefix_join_kernel<HD>), dim3((unsigned)((rh + per - 1) / per)), dim3(256), 0, s, p);
}
template <int HD>
void launch_step(const PrefixParams& p, const StepWeights& sw, hipStream_t s) {
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
    const int slots = plan(p, rows_tiles(B, Nq));
    return part_bytes(p, head_dim, slots);
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
    HK_REQUIRE(d->ldq >= 0 && d->ldkp >= 0 && d->ldvp >= 0 && d->ldk >= 0 && d->ldv >= 0 && d->bsq >= 0 && d->bsk >= 0 && d->bsv >= 0 &&
                   (d->Nq == 1 || d->ldo >= row) && (d->B == 1 || d->bso >= row) && d->bias_bs >= 0,
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
    const int rt = rows_tiles(p.B, p.Nq);
    const int slots = plan(p, rt);
    HK_REQUIRE(d->ws && d->ws_bytes >= part_bytes(p, d->head_dim, slots),
               "hk_prefix_attn_bf16: workspace of %zu bytes, %zu needed (hk_prefix_attn_ws)", d->ws ? d->ws_bytes : (size_t)0,
               part_bytes(p, d->head_dim, slots));
    HK_REQUIRE(p.pjobs + (int64_t)p.B * p.noc * p.H * p.norg < (1LL << 31), "hk_prefix_attn_bf16: grid too large");
    set_parts(p, d->ws, d->head_dim, slots);
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    if (d->head_dim == 128) launch_prefix<128>(p, rt, s);
    else launch_prefix<64>(p, rt, s);
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
    const int slots = plan(p, 1);
    return part_bytes(p, head_dim, slots) + (size_t)B * H * ((n_keys + TK - 1) / TK * TK) * 4;
}

extern "C" int hk_decode_attn_weights_bf16(const hk_step_weights_desc* d, void* stream) {
    HK_REQUIRE(d && d->q && d->k_cache && d->v_cache && d->out && d->w_out, "hk_decode_attn_weights_bf16: null operand");
    HK_REQUIRE(shape_ok(d->B, d->H, 1, 0, d->n_keys, d->head_dim) && d->n_keys <= d->cache_rows,
               "hk_decode_attn_weights_bf16: bad shape B=%d H=%d head_dim=%d n_keys=%d cache_rows=%ld", d->B, d->H, d->head_dim, d->n_keys,
               (long)d->cache_rows);
    HK_REQUIRE(((uintptr_t)d->q | (uintptr_t)d->k_cache | (uintptr_t)d->v_cache | (uintptr_t)d->ws) % 16 == 0 && (uintptr_t)d->out % 8 == 0 &&
                   ((uintptr_t)d->w_in | (uintptr_t)d->w_out | (uintptr_t)d->key_bias) % 4 == 0,
               "hk_decode_attn_weights_bf16: operands must be 16-byte aligned");
    HK_REQUIRE((d->H == 1 || d->wo_hs >= d->n_keys) && (d->B == 1 || d->wo_bs >= (d->H - 1) * d->wo_hs + d->n_keys) && d->wi_bs >= 0 &&
                   d->wi_hs >= 0 && d->bias_bs >= 0 && d->bias_hs >= 0,
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
    const int slots = plan(p, 1);
    const size_t parts = part_bytes(p, d->head_dim, slots), need = parts + (size_t)p.B * p.H * p.raw_ld * 4;
    HK_REQUIRE(d->ws && d->ws_bytes >= need, "hk_decode_attn_weights_bf16: workspace of %zu bytes, %zu needed (hk_decode_attn_weights_ws)",
               d->ws ? d->ws_bytes : (size_t)0, need);
    HK_REQUIRE((int64_t)p.B * p.noc * p.H < (1LL << 31), "hk_decode_attn_weights_bf16: grid too large");
    set_parts(p, d->ws, d->head_dim, slots);
    p.raw = reinterpret_cast<float*>(reinterpret_cast<char*>(d->ws) + parts);
    StepWeights sw = {d->w_in, d->w_out, d->wi_bs, d->wi_hs, d->wo_bs, d->wo_hs};
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    if (d->head_dim == 128) launch_step<128>(p, sw, s);
    else launch_step<64>(p, sw, s);
    HK_CHECK_LAUNCH("hk_decode_attn_weights_bf16");
    return HK_OK;
}
