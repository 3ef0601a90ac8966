// Attention over packed documents, forward and backward (dim_head 64).
//
// Queries and keys of several documents lie one behind the other on one token axis; document d's queries are rows cu_q[d] .. and its keys
// rows cu_k[d] .. (optionally only the first len_q[d] / len_k[d] of that slot).  Query i of a document with nq queries and nk keys stands at
// position i + nk - nq (the last query on the last key) and sees the keys j < lim(i):
//     full: nk       causal: min(nk, max(position + 1, prefix))
// Per visible pair    z = scale q.k;   c = cap tanh(z / cap)  (cap > 0);   t = c - slope_h |j - position|   or   t = c + table[bucket(j - position), h]
//                     p = softmax(t);  o = p v;   a row that sees nothing has o = 0
// Backward            dS = p (dO.v - dO.o);  dtable[b, h] = sum of dS over the pairs of bucket b;  dz = dS (1 - tanh^2) scale
//                     dq = dz k;  dk = dz^T q;  dv = p^T dO      (grouped heads: dk, dv summed over the query heads of a key head)
//
// Layout: as in attn32.hip a wave owns 32 rows (lane = one query in the forward and dQ kernels, one key in the dK / dV kernel) on 32x32x16
// MFMAs, the scores computed swapped so that a lane's accumulators are the B operand of the next product.  Here the second operands come out
// of the row-major tiles by transposing LDS reads (no V^T copy is needed: packed rows are read as they lie, any token and head stride).
//
// What a wave does per 32-key block beyond the products is a few vector operations per score, and the bias is arranged to cost next to none of
// them: where a block lies wholly on one side of its queries the linear bias splits into a per-lane constant (folded into the running maximum)
// and sixteen wave-uniform addends (the addend of the multiply-add that scales the score anyway); where a block lies beyond the table's reach
// the learned bias is one constant.  Only blocks that cross the diagonal (or lie within reach) take |distance| (an LDS lookup) per score.
//
// Softmax: the reference point of a row is the maximum of the first block it sees, and stays: fp32 sums and bf16 probabilities lose nothing by a
// common factor, so nothing is compared per score.  Only when a row's sum passes 2^60 (or overflows: the first block of a row does) is the block's
// maximum taken, the accumulators rescaled and the block's probabilities taken again -- one compare and a vote per 32-key block.
// The backward works with small differences p (dO.v - dO.o), and the table's gradient is a sum of them over every pair at a distance, in fp32: an
// o that is good to bf16 only (probabilities rounded before the second product, output rounded after it) shows in the gradients of q and k (2.9e-3
// off the exact ones instead of 2.4e-3) and in the third digit of the table's.  A training forward therefore carries the probabilities as two bf16
// terms through the second product, sums them unrounded and keeps what rounding cut off the output (o_lo, bf16; out + o_lo is 3e-6 off, on peaked rows
// too); with a table as three terms and o_lo in fp32 (its gradient is then 8e-7 off, as in plain fp32, instead of 3e-6; 89 -> 101 us on 8397 tokens of
// 11 documents, 16 heads).
//
// Sums are taken in a fixed order throughout: no atomics, the same bits every time.
#include "e2k_device.h"
#include "plan.h"
#include <e2k_asm.h>
#include "../../include/e2k.h"
#include "attn_tile32.h"
#include "attn_score.h"

using namespace e2k;

namespace {

constexpr int STAGE = 16384;          // one ring stage: two [64][64] bf16 tiles
constexpr int NST = 3;                // ring stages: two tiles in flight while one is computed
constexpr float LSE_EMPTY = 1e30f;    // log-sum-exp of a row that sees nothing: exp2(t - it) is 0
constexpr int PADL = 64;              // entries of the distance table beyond its reach on either side (a block's distances spread over 63)
constexpr int REACH_MAX = 512;
constexpr int GAP_PARTS = 8;          // workgroups per gap between documents

struct PAArgs {
    const bf16_t *Q, *K, *V, *dO;
    long sq, hq, sk, hk, sv, hv, so, ho, sg, hg;       // token and head strides (elements) of Q, K, V, O, dO
    const int *cu_q, *cu_k, *len_q, *len_k, *prefix;
    int nd, Tq, Tk, H, Hkv, G;
    float scale, cap;
    int causal, fill;
    const float *slopes, *table; const int* buckets; int nbuckets, R;
    bf16_t* O; void* Olo;                              // O strided; Olo (Tq, H, 64): fp32 with a table, else bf16
    float *lse2, *delta;                               // (H, Tq)
    bf16_t *dQ, *dK, *dV;                              // (Tq, H, 64), (Tk, Hkv, 64)
    float* dist;                                       // [head][row of a (document, tile): dist_row][2 R + 1]: sums of dS by distance
    int nt, nwork, heads, order;                       // row tiles per (document, head) of this grid; workgroups that compute; heads x parts; longest
                                                       // documents first
    int splits; float* part;                           // parts of a tile's sweep; dK / dV: their sums [part][dK | dV][Tk][Hkv][64]; forward: their
                                                       // accumulators [part][Tq][H][64], then reference points and sums [part][2][Tq][H]
};

// rows of document d, kept inside [0, total) whatever the offsets say
struct Span { int at, n; };
__device__ __forceinline__ Span span(const int* cu, const int* len, int d, int total) {
    Span s;
    s.at = clampi(cu[d], 0, total);
    const int end = clampi(cu[d + 1], s.at, total);
    s.n = end - s.at;
    if (len) s.n = clampi(len[d], 0, s.n);
    return s;
}
struct Doc {
    int q0, nq, k0, nk, off, prefix, causal;
    __device__ __forceinline__ int lim(int i) const {           // keys that query i sees: 0 .. lim(i) - 1 (never falls with i)
        if (!causal) return nk;
        const int a = i + off + 1;
        return clampi(a > prefix ? a : prefix, 0, nk);
    }
};
__device__ __forceinline__ Doc doc_of(const PAArgs& p, int d) {
    const Span a = span(p.cu_q, p.len_q, d, p.Tq), b = span(p.cu_k, p.len_k, d, p.Tk);
    Doc r{uniform_i(a.at), uniform_i(a.n), uniform_i(b.at), uniform_i(b.n), 0, 0, p.causal};
    r.off = r.nk - r.nq;
    r.prefix = (p.causal && p.prefix) ? uniform_i(clampi(p.prefix[d], 0, r.nk)) : 0;
    return r;
}

// The document of a given rank by length, longest first (up to 64 documents: a lane each; every wave finds it by itself)
__device__ __forceinline__ int doc_of_rank(const int* cu, const int* len, int nd, int total, int rank) {
    const int lane = threadIdx.x & 63;
    const int n = lane < nd ? span(cu, len, lane, total).n : -1;
    int r = 0;
    for (int j = 0; j < nd; ++j) {
        const int m = __builtin_bit_cast(int, lane_bcast(__builtin_bit_cast(float, n), j));
        r += (m > n || (m == n && j < lane)) ? 1 : 0;
    }
    return uniform_i(__builtin_ctzll(wave_ballot(lane < nd && r == rank)));
}

// Workgroups go to the 8 XCDs round-robin in launch order.  Re-numbered so that an XCD gets a contiguous run of heads with all their documents and
// tiles: the tiles of a (document, head) stream the same K / V through one L2, and with heads in eights every XCD has the same work.  Where there are
// more workgroups than slots the long sweeps go first (cu / len: the axis that a workgroup sweeps, whose length is the workgroup's time) and a
// document's heads side by side: 11 documents of 97 .. 1056 tokens in a mixed order, forward 91 -> 88 us, dQ 118 -> 116, dK / dV 123 -> 119; six of
// 1056 and 2112, causal, forward 89 -> 80, dQ 101 -> 96.  A dK / dV sweep in parts is better off as the documents lie (131 against 141 us there).
struct Work { int h, d, tile; };
__device__ __forceinline__ Work work_of(const PAArgs& p, const int* cu, const int* len, int total) {
    const int q = p.nwork >> 3, r = p.nwork & 7;
    const int xcd = (int)blockIdx.x & 7, in = (int)blockIdx.x >> 3;
    Work w;
    if (p.order && p.heads % 8 == 0) {       // heads xcd hp .. + hp - 1: document by document, the heads inside
        const int hp = p.heads >> 3, rest = in / p.nt;
        w.tile = in % p.nt;
        w.h = xcd * hp + rest % hp;
        w.d = rest / hp;
    } else {
        const int lin = (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + in, hd = lin / p.nt;
        w.tile = lin % p.nt;
        w.d = hd % p.nd;
        w.h = hd / p.nd;
    }
    w.tile = p.nt - 1 - w.tile;              // causal: the long rows first
    if (p.order) w.d = doc_of_rank(cu, len, p.nd, total, w.d);
    return w;
}

// rows that no document covers, between documents d - 1 and d (d = nd: behind the last): zeros
__device__ __forceinline__ void fill_gap(const int* cu, const int* len, int nd, int total, bf16_t* out, long ts, long hs, int nh, int id) {
    const int g = id / GAP_PARTS, part = id % GAP_PARTS;
    int from = 0;
    if (g > 0) {
        const Span s = span(cu, len, g - 1, total);
        from = s.at + s.n;
    }
    const int to = g < nd ? clampi(cu[g], 0, total) : total;
    for (int row = from + part; row < to; row += GAP_PARTS)
        for (int c = threadIdx.x; c < nh * 8; c += blockDim.x)
            st<u32x4>(out + (long)row * ts + (long)(c >> 3) * hs + (c & 7) * 8, u32x4{0u, 0u, 0u, 0u});
}

// ------------------------------------------------------------------------------------------------ scores

// One block of 32 rows x 32 columns of scores, 16 of them in a lane: distance (key - query position) of register r is  rel + SGN reg_off(r).
// The score of register r (log2 domain) is x[r] + c: c = offset() is the part of the bias that a block's registers share.
//   lo: smallest distance of the block's first row to its columns, so that the block spans distances lo - 31 .. lo + 31
template <int BIAS, bool CAP, int SGN, bool FINE, bool KEEP> struct Scorer {
    float sc2; Cap cp;
    float sl2, rc[16];                       // BIAS 1: slope log2(e), and times reg_off(r)
    const float* lut; int R; float far_lo, far_hi;
    __device__ __forceinline__ void init(const PAArgs& p, float slope) {
        sc2 = p.scale * LOG2E;
        if (CAP) cp = cap_of<FINE>(p.scale, p.cap);
        if (BIAS == 1) {
            sl2 = uniform_f(slope * LOG2E);
#pragma unroll
            for (int r = 0; r < 16; ++r) rc[r] = uniform_f(sl2 * (float)reg_off(r));
        }
    }
    __device__ __forceinline__ float offset(int rel, int lo) const {
        if (BIAS == 1) return lo + 31 <= 0 ? sl2 * (float)rel : lo - 31 >= 0 ? -sl2 * (float)rel : 0.f;
        if (BIAS == 2) return lo + 31 <= -R ? far_lo : lo - 31 >= R ? far_hi : 0.f;
        return 0.f;
    }
    // x[r] = score - c - mo(r).  KEEP: z becomes the capped product, which the backward needs again (left as it was without a cap)
    template <class M> __device__ __forceinline__ void args(f32x16& z, float (&x)[16], int rel, int lo, M&& mo) const {
        auto finish = [&](auto&& add) __attribute__((always_inline)) {
            if constexpr (CAP) {
                cap16<FINE, KEEP>(z, x, cp, add);
            } else {
#pragma unroll
                for (int r = 0; r < 16; ++r) x[r] = fmaf(z[r], sc2, add(r));
            }
        };
        if (BIAS == 0) {
            finish([&](int r) { return -mo(r); });
        } else if (BIAS == 1) {
            const float d = (float)rel;
            if (lo + 31 <= 0) finish([&](int r) { return SGN * rc[r] - mo(r); });
            else if (lo - 31 >= 0) finish([&](int r) { return -SGN * rc[r] - mo(r); });
            else finish([&](int r) { return fmaf(-sl2, fabsf(d + (float)(SGN * reg_off(r))), -mo(r)); });
        } else {
            const float* l = lut + PADL + R + rel;
            if (lo + 31 <= -R || lo - 31 >= R) finish([&](int r) { return -mo(r); });
            else finish([&](int r) { return l[SGN * reg_off(r)] - mo(r); });
        }
    }
};

// distance -> learned bias of one head (log2 domain), clamped at the reach; entry PADL + R + distance
__device__ __forceinline__ void load_lut(const PAArgs& p, int h, float* lut) {
    for (int i = threadIdx.x; i < 2 * p.R + 1 + 2 * PADL; i += blockDim.x) {
        const int b = clampi(p.buckets[clampi(i - PADL, 0, 2 * p.R)], 0, p.nbuckets - 1);
        lut[i] = p.table[(long)b * p.H + h] * LOG2E;
    }
}

// one operand row's four fragments (columns 16 ks + 8 hi .. + 7), zeros for a row outside
__device__ __forceinline__ void row_frags(bf16x8 (&f)[4], const bf16_t* row, bool in, int hi) {
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) f[ks] = in ? ld<bf16x8>(row + ks * 16 + hi * 8) : bf16x8{0, 0, 0, 0, 0, 0, 0, 0};
}

// LDS-DMA of 64 rows each of two operands into a ring stage (K-type images: LDS row r holds tile row swap23(r)); rows beyond `last` read row
// `last` (masked by the caller).  Wave-uniform 64-bit bases, 32-bit lane offsets: strides < 2^23 elements keep row * stride inside 24 x 24 bits
struct Stager {
    int row0; unsigned col0, s0, s1;          // byte strides
    int wave;
    __device__ __forceinline__ void init(int wave_, int lane, long st0, long st1) {
        wave = wave_;
        row0 = swap23(wave * 16 + (lane >> 3));
        col0 = (unsigned)(((lane & 7) ^ swz(wave * 16 + (lane >> 3))) * 16);
        s0 = (unsigned)(st0 * 2);
        s1 = (unsigned)(st1 * 2);
    }
    __device__ __forceinline__ void issue(const bf16_t* a, const bf16_t* b, int last, unsigned char* S) const {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const unsigned row = (unsigned)min(row0 + 4 * u, last), col = col0 ^ (64u * u);
            glds16((const char*)a + ((row & 0xffffffu) * (s0 & 0xffffffu) + col), S + (wave * 2 + u) * 1024);
            glds16((const char*)b + ((row & 0xffffffu) * (s1 & 0xffffffu) + col), S + 8192 + (wave * 2 + u) * 1024);
        }
    }
};

// ------------------------------------------------------------------------------------------------ forward

// Few queries over many keys (prompts behind a cache) leave most of the chip empty and are bound by the latency of a block's chain: inference then
// cuts a row's keys into parts and joins them.
// One workgroup = 128 queries of one (document, head): 4 waves x 32; K / V tiles of 64 keys through a three-stage LDS-DMA ring (two tiles in flight
// while one is computed: with one, the copies' latency of about 1 us set the pace; one raw barrier a tile), three workgroups a CU.
// Bound by the vector ALU (85 % of the clocks in which a CU has work, on long rows): 16417 tokens x 16 heads, linear bias, cap: 1.95 .. 2.13 ms by inputs and
// clocks (under this load 1.9 GHz), 518 .. 566 TFLOP/s; 8 x 1056 tokens x 16 heads, no bias: 63 us, 580 TFLOP/s (79 with the training form's second term).
// TRAIN: log-sum-exps, probabilities in two terms (with a table three), o_lo
template <int BIAS, bool CAP, bool TRAIN>
__global__ __launch_bounds__(256, 3) void pa_fwd_kernel(PAArgs p) {
    __shared__ __attribute__((aligned(16))) unsigned char smem[NST * STAGE];
    __shared__ float lut[BIAS == 2 ? 2 * REACH_MAX + 1 + 2 * PADL : 1];
    lds_declare(smem, sizeof(smem));
    if ((int)blockIdx.x >= p.nwork) {
        fill_gap(p.cu_q, p.len_q, p.nd, p.Tq, p.O, p.so, p.ho, p.H, (int)blockIdx.x - p.nwork);
        return;
    }
    const int tid = threadIdx.x, lane = tid & 63, wave = uniform_i(tid >> 6);
    const int l31 = lane & 31, hi = lane >> 5;
    const Work wk = work_of(p, p.cu_k, p.len_k, p.Tk);
    const int h = wk.h / p.splits, part = wk.h % p.splits;
    const Doc D = doc_of(p, wk.d);
    if (wk.tile * 128 >= D.nq) return;
    constexpr bool FINE = TRAIN && BIAS == 2;          // (the table's gradient is returned in fp32)
    Scorer<BIAS, CAP, 1, FINE, false> sc;
    sc.init(p, BIAS == 1 ? p.slopes[h] : 0.f);
    if (BIAS == 2) {
        load_lut(p, h, lut);
        __syncthreads();
        sc.lut = lut;
        sc.R = p.R;
        sc.far_lo = lut[PADL];
        sc.far_hi = lut[PADL + 2 * p.R];
    }
    Stager sg;
    sg.init(wave, lane, p.sk, p.sv);
    unsigned fra[4];
    frag_addr(smem, l31, hi, fra);
    const TrAddr tra = tr_addr(smem, lane);
    const bf16_t* Kb = p.K + (long)D.k0 * p.sk + (long)(h / p.G) * p.hk;
    const bf16_t* Vb = p.V + (long)D.k0 * p.sv + (long)(h / p.G) * p.hv;

    for (int tile = wk.tile; tile * 128 < D.nq; tile += p.nt) {
        const int q0 = tile * 128 + wave * 32, q = q0 + l31;
        const bool live = q0 < D.nq, qin = q < D.nq;
        const int qc = min(q, D.nq - 1);              // (lanes past the end repeat the last query: their sums stay in step with the wave's)
        const int lim = D.lim(qc);
        const int lim_lo = live ? D.lim(q0) : 0, lim_hi = live ? D.lim(min(q0 + 31, D.nq - 1)) : 0;
        const int kend = D.lim(min(tile * 128 + 127, D.nq - 1)), all = (kend + 63) / 64;
        const int kt0 = all * part / p.splits, nt = all * (part + 1) / p.splits;          // this part's key tiles
        bf16x8 qf[4];
        row_frags(qf, p.Q + (long)(D.q0 + qc) * p.sq + (long)h * p.hq, live, hi);
        f32x16 o[2] = {zero16(), zero16()};
        float m = M_INIT, l0 = 0.f, l1 = 0.f;
        // (every ordinary load of the prologue is waited for before the first LDS-DMA: vmcnt is counted in order)
        asm volatile("" ::"v"(qf[0]), "v"(qf[1]), "v"(qf[2]), "v"(qf[3]));
        auto fetch = [&](int kt, unsigned char* S) __attribute__((always_inline)) {
            sg.issue(Kb + (long)(kt * 64) * p.sk, Vb + (long)(kt * 64) * p.sv, D.nk - 1 - kt * 64, S);
        };
        if (kt0 < nt) fetch(kt0, smem);
        if (kt0 + 1 < nt) fetch(kt0 + 1, smem + STAGE);
        const int qp = q0 + D.off;
        // probabilities (arguments of exp2 in x, replaced) packed, and the row's sum with them: of the packed ones in inference, whose second product has
        // no more than them (what rounds a dominating one up rounds the sum up too); of the unrounded ones in training, whose second product has them in
        // two or three terms (with the packed ones' sum a peaked row's output and log-sum-exp were up to 2^-8 off)
        auto probs = [&](float (&x)[16], bf16x8 (&pf)[2], float& la, float& lb) __attribute__((always_inline)) {
            la = l0;
            lb = l1;
#pragma unroll
            for (int r = 0; r < 16; ++r) x[r] = fast_exp2(x[r]);
            pf[0] = pack8f(x);
            pf[1] = pack8f(x + 8);
            if (TRAIN) {
#pragma unroll
                for (int r = 0; r < 16; r += 2) {
                    la += x[r];
                    lb += x[r + 1];
                }
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    la = add_bf16_pair(__builtin_bit_cast(u32x4, pf[0])[i], la);
                    lb = add_bf16_pair(__builtin_bit_cast(u32x4, pf[1])[i], lb);
                }
            }
        };
        auto step = [&](auto stage_, int kt) __attribute__((always_inline)) {
            constexpr int S = decltype(stage_)::value * STAGE;
            const int k0 = kt * 64;
            if (kt + 1 < nt) wait_vmcnt<4>();          // tile kt has landed for this wave (tile kt + 1's four copies may be in flight) ...
            else wait_vmcnt<0>();
            barrier_raw();                             // ... and for every wave; everyone is done with tile kt - 1, whose stage is filled next
            if (kt + 2 < nt) fetch(kt + 2, smem + (decltype(stage_)::value + 2) % NST * STAGE);
            auto block = [&](auto kb_) __attribute__((always_inline)) {
                constexpr int kb = decltype(kb_)::value;
                const int kk = k0 + 32 * kb;
                if (kk >= lim_hi) return;                     // (wave-uniform) nothing of the block is visible
                // (the transposed V fragments are read while the score products run)
                f32x16 s = zero16();
                bf16x8 kf[4], vf[2][2];
                lds_read4<S + kb * 4096>(kf, fra);
#pragma unroll
                for (int ks = 0; ks < 4; ++ks) s = mfma32(kf[ks], qf[ks], s);
                sched_fence();
                tr_frags<S + 8192 + kb * 4096>(vf, tra);
                sched_fence();
                float la, lb, x[16];
                bf16x8 pf[2];
                const int rel = kk + 8 * hi - (qp + l31), lo = kk - qp;
                bool done = false;
                if (kk + 32 <= lim_lo) {                      // every query of the wave sees all of the block
                    f32x16 z = s;
                    const float mo = m - sc.offset(rel, lo);
                    sc.args(z, x, rel, lo, [&](int) { return mo; });
                    probs(x, pf, la, lb);
                    done = wave_all(la + lb < L_MAX);
                }
                if (!done) {                                  // a masked block, or a row whose sum outgrew its reference point
                    cold_path();
                    pin_vgpr(s);                                          // (its arithmetic is not shared with the path above: that would keep 32 registers alive)
                    const float c = sc.offset(rel, lo);
                    sc.args(s, x, rel, lo, [](int) { return 0.f; });
                    const int n = lim - (kk + 8 * hi);
                    float mx = -__builtin_inff();
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        x[r] = reg_off(r) < n ? x[r] : -__builtin_inff();
                        mx = fmaxf(mx, x[r]);
                    }
                    mx += c;
                    const float mn = fmaxf(m, fmaxf(mx, lane32_other(mx))), al = fast_exp2(m - mn);
                    l0 *= al;
                    l1 *= al;
#pragma unroll
                    for (int r = 0; r < 16; ++r) { o[0][r] *= al; o[1][r] *= al; }
                    m = mn;
#pragma unroll
                    for (int r = 0; r < 16; ++r) x[r] -= mn - c;
                    probs(x, pf, la, lb);
                }
                l0 = la;
                l1 = lb;
#pragma unroll
                for (int s2 = 0; s2 < 2; ++s2)
#pragma unroll
                    for (int db = 0; db < 2; ++db) o[db] = mfma32(vf[s2][db], pf[s2], o[db]);
                // what packing cut off, as a second (third) term
#pragma unroll
                for (int term = 1; term < (FINE ? 3 : TRAIN ? 2 : 1); ++term)
#pragma unroll
                    for (int s2 = 0; s2 < 2; ++s2) {
                        float w[8];
                        unpack8(__builtin_bit_cast(u32x4, pf[s2]), w);
#pragma unroll
                        for (int e = 0; e < 8; ++e) x[8 * s2 + e] -= w[e];
                        pf[s2] = pack8f(x + 8 * s2);
#pragma unroll
                        for (int db = 0; db < 2; ++db) o[db] = mfma32(vf[s2][db], pf[s2], o[db]);
                    }
            };
            block(Int<0>{});
            block(Int<1>{});
        };
        for (int kt = kt0; kt < nt; kt += NST) {
            step(Int<0>{}, kt);
            if (kt + 1 < nt) step(Int<1>{}, kt + 1);
            if (kt + 2 < nt) step(Int<2>{}, kt + 2);
        }
        float l = l0 + l1;
        l += lane32_other(l);                                 // a row's keys are split over lanes l and l + 32
        if (!TRAIN && p.splits > 1) {
            if (qin) {
                const long row = (long)part * p.Tq + D.q0 + q;
                float* ws = p.part + (row * p.H + h) * DH;
#pragma unroll
                for (int db = 0; db < 2; ++db)
#pragma unroll
                    for (int g = 0; g < 4; ++g)
                        st<f32x4>(ws + 32 * db + 8 * g + 4 * hi, f32x4{o[db][4 * g], o[db][4 * g + 1], o[db][4 * g + 2], o[db][4 * g + 3]});
                if (hi == 0) {
                    float* ml = p.part + (long)p.splits * p.Tq * p.H * DH + ((long)part * 2 * p.Tq + D.q0 + q) * p.H + h;
                    ml[0] = m;
                    ml[(long)p.Tq * p.H] = l;
                }
            }
        } else if (live) {
            const float inv = l == 0.f ? 0.f : 1.f / l;       // (NaN stays NaN)
            const int row = D.q0 + (qin ? q : 0);
            if (TRAIN && qin && hi == 0) p.lse2[(long)h * p.Tq + row] = l == 0.f ? LSE_EMPTY : m + log2f(l);
            bf16_t* orow = p.O + (long)row * p.so + (long)h * p.ho;
            const long lrow = ((long)row * p.H + h) * DH;
            store_rows32(o, hi, qin, [&](int db, int g, int hi_, bool ok, const float* a, const float* b) __attribute__((always_inline)) {
                float v[8];
#pragma unroll
                for (int e = 0; e < 4; ++e) { v[e] = a[e] * inv; v[4 + e] = b[e] * inv; }
                u32x2 x = pack4(v), y = pack4(v + 4), xl, yl;
                if (TRAIN) {
                    float w[8], lo[8];
                    unpack4(x, w);
                    unpack4(y, w + 4);
#pragma unroll
                    for (int e = 0; e < 8; ++e) lo[e] = v[e] - w[e];
                    if (FINE) {
                        float* lf = (float*)p.Olo + lrow + 32 * db + 8 * g + 4 * hi_;
                        if (ok) {
                            st<f32x4>(lf, f32x4{lo[0], lo[1], lo[2], lo[3]});
                            st<f32x4>(lf + 8, f32x4{lo[4], lo[5], lo[6], lo[7]});
                        }
                    }
                    xl = pack4(lo);
                    yl = pack4(lo + 4);
                    swap_pair(xl, yl);
                }
                swap_pair(x, y);
                const int col = 32 * db + 8 * (g + hi_);
                if (ok) {
                    st<u32x4>(orow + col, u32x4{x[0], x[1], y[0], y[1]});
                    if (TRAIN && !FINE) st<u32x4>((bf16_t*)p.Olo + lrow + col, u32x4{xl[0], xl[1], yl[0], yl[1]});
                }
            });
        }
        if ((tile + p.nt) * 128 < D.nq) __syncthreads();         // (another round: the ring is free again)
    }
}

constexpr int JOIN_ROWS = 4;          // rows of a join workgroup: a thread or two per eight columns (with 32 the few workgroups took 43 us for 890 rows)
// outputs from the parts of their sweeps; eight columns a thread
__global__ __launch_bounds__(256) void pa_fwd_join_kernel(PAArgs p) {
    const int tile = (int)blockIdx.x % p.nt, d = (int)blockIdx.x / p.nt;
    const Span s = span(p.cu_q, p.len_q, d, p.Tq);
    const float* ml = p.part + (long)p.splits * p.Tq * p.H * DH;
    const long step = (long)p.Tq * p.H;
    for (int r0 = tile * JOIN_ROWS; r0 < s.n; r0 += p.nt * JOIN_ROWS) {
        const int rows = min(JOIN_ROWS, s.n - r0);
        for (int i = threadIdx.x; i < rows * p.H * (DH / 8); i += 256) {
            const int c = i & 7, h = (i >> 3) % p.H, row = s.at + r0 + (i >> 3) / p.H;
            const long at = (long)row * p.H + h;
            float M = M_INIT, L = 0.f, a[8];
            for (int q = 0; q < p.splits; ++q) M = fmaxf(M, ml[2 * q * step + at]);
#pragma unroll
            for (int e = 0; e < 8; ++e) a[e] = 0.f;
            for (int q = 0; q < p.splits; ++q) {
                const float w = fast_exp2(ml[2 * q * step + at] - M);
                const float* x = p.part + (q * step + at) * DH + 8 * c;
                const f32x4 u = ld<f32x4>(x), v = ld<f32x4>(x + 4);
                L = fmaf(ml[(2 * q + 1) * step + at], w, L);
#pragma unroll
                for (int e = 0; e < 4; ++e) { a[e] = fmaf(u[e], w, a[e]); a[4 + e] = fmaf(v[e], w, a[4 + e]); }
            }
            const float inv = L == 0.f ? 0.f : 1.f / L;
#pragma unroll
            for (int e = 0; e < 8; ++e) a[e] *= inv;
            st<u32x4>(p.O + (long)row * p.so + (long)h * p.ho + 8 * c, pack8(a));
        }
    }
}

// ------------------------------------------------------------------------------------------------ backward: dQ, dO.o, sums of dS by distance

// sums of one block's dS (16 of them in a lane: query l31, keys reg_off(r) + 8 hi) along its diagonals, added to `dist` (entry = distance +
// an offset folded into `base`).  The block goes through a wave's own LDS scratch ([16 keys][33]) in two halves; lane t (of 32) collects the
// diagonals t and t - 32, whose elements are one per key: the scratch is read without bank conflicts, every distance has one owner, and the
// order of the additions is fixed.
__device__ __forceinline__ void diag_add(const float (&ds)[16], float* scr, float* dist_at_lo, int l31, int hi) {
    float A = 0.f, B = 0.f;
#pragma unroll
    for (int s2 = 0; s2 < 2; ++s2) {
        wave_sync();
#pragma unroll
        for (int e = 0; e < 8; ++e) scr[(8 * hi + e) * 33 + l31] = ds[8 * s2 + e];
        wave_sync();
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int key = 16 * s2 + 8 * hi + j;               // half `hi` of the wave takes its eight keys of the sixteen
            const int i = key - l31;                            // query of diagonal l31, or (wrapped) of diagonal l31 - 32
            const float v = scr[(8 * hi + j) * 33 + (i & 31)];
            A += i >= 0 ? v : 0.f;
            B += i >= 0 ? 0.f : v;
        }
    }
    A += lane32_other(A);
    B += lane32_other(B);
    // diagonals l31 (lower half-wave) and l31 - 32 (upper): 64 entries, each lane its own; dist_at_lo = entry of distance `lo`
    dist_at_lo[hi ? l31 - 32 : l31] += hi ? B : A;
}

// Sums by distance of one head: a row of 2 R + 1 for each tile of each document with rows, however large the grid is (most of its workgroups are empty where
// the longest document is not known).  A document of n rows from row `at` on has tiles at / 128 + min(d, at) .. + ceil(n / 128) - 1: the next one with rows starts
// at least n >= 1 rows further on, so that floor((at + n) / 128) - floor(at / 128) + 1 >= ceil(n / 128) tiles lie between them.
__host__ __device__ __forceinline__ long dist_rows(int nd, int Tq) { return Tq / 128 + (nd < Tq ? nd : Tq); }
__device__ __forceinline__ int dist_row(int d, int at) { return at / 128 + min(d, at); }

constexpr int distn(int reach) { return 2 * reach + 1 + 2 * PADL; }

// Lane layout and ring of the forward; dP beside the scores, dQ^T = K^T dS^T from the same K tile.  8 x 1056 tokens x 16 heads, no bias: 77 us; with a
// table's gradient 113 us at 8397 tokens of 11 documents.
// RG: 0 no table gradient, else the largest reach of this instantiation (its LDS)
template <int BIAS, bool CAP, int RG>
__global__ __launch_bounds__(256, (BIAS || CAP) ? 2 : 3) void pa_dq_kernel(PAArgs p) {
    __shared__ __attribute__((aligned(16))) unsigned char smem[NST * STAGE];
    __shared__ float lut[BIAS == 2 ? distn(RG && RG < REACH_MAX ? RG : REACH_MAX) : 1];
    __shared__ float dist[RG ? 4 * distn(RG) : 1];
    __shared__ float scr[RG ? 4 * 16 * 33 : 1];
    lds_declare(smem, sizeof(smem));
    if ((int)blockIdx.x >= p.nwork) {
        fill_gap(p.cu_q, p.len_q, p.nd, p.Tq, p.dQ, (long)p.H * DH, DH, p.H, (int)blockIdx.x - p.nwork);
        return;
    }
    const int tid = threadIdx.x, lane = tid & 63, wave = uniform_i(tid >> 6);
    const int l31 = lane & 31, hi = lane >> 5;
    const Work wk = work_of(p, p.cu_k, p.len_k, p.Tk);
    const int h = wk.h;
    const Doc D = doc_of(p, wk.d);
    if (wk.tile * 128 >= D.nq) return;
    const int ND = 2 * p.R + 1 + 2 * PADL;
    Scorer<BIAS, CAP, 1, (RG > 0), true> sc;
    sc.init(p, BIAS == 1 ? p.slopes[h] : 0.f);
    if (BIAS == 2) {
        load_lut(p, h, lut);
        if (RG) for (int i = tid; i < 4 * ND; i += 256) dist[i] = 0.f;
        __syncthreads();
        sc.lut = lut;
        sc.R = p.R;
        sc.far_lo = lut[PADL];
        sc.far_hi = lut[PADL + 2 * p.R];
    }
    float* const mydist = dist + (RG ? wave * ND : 0);
    float* const myscr = scr + (RG ? wave * 16 * 33 : 0);
    float far_lo = 0.f, far_hi = 0.f;
    const float icl = CAP ? 1.f / (p.cap * LOG2E) : 0.f;
    Stager sg;
    sg.init(wave, lane, p.sk, p.sv);
    unsigned fra[4];
    frag_addr(smem, l31, hi, fra);
    const TrAddr tra = tr_addr(smem, lane);
    const bf16_t* Kb = p.K + (long)D.k0 * p.sk + (long)(h / p.G) * p.hk;
    const bf16_t* Vb = p.V + (long)D.k0 * p.sv + (long)(h / p.G) * p.hv;

    for (int tile = wk.tile; tile * 128 < D.nq; tile += p.nt) {
        const int q0 = tile * 128 + wave * 32, q = q0 + l31;
        const bool live = q0 < D.nq, qin = q < D.nq;
        const int lim = qin ? D.lim(q) : 0;
        const int lim_lo = live ? D.lim(q0) : 0, lim_hi = live ? D.lim(min(q0 + 31, D.nq - 1)) : 0;
        const int kend = D.lim(min(tile * 128 + 127, D.nq - 1)), nt = (kend + 63) / 64;
        const int row = D.q0 + (qin ? q : 0);
        bf16x8 qf[4], dof[4];
        row_frags(qf, p.Q + (long)row * p.sq + (long)h * p.hq, qin, hi);
        row_frags(dof, p.dO + (long)row * p.sg + (long)h * p.hg, qin, hi);
        float dl = 0.f;
        {
            const bf16_t* orow = p.O + (long)row * p.so + (long)h * p.ho + hi * 8;
            const long lrow = ((long)row * p.H + h) * DH + hi * 8;
#pragma unroll
            for (int ks = 0; ks < 4; ++ks) {
                float a[8], b[8], g[8];
                unpack8(ld<u32x4>(orow + ks * 16), a);
                if (BIAS == 2) {
                    const float* lf = (const float*)p.Olo + lrow + ks * 16;
                    const f32x4 u = ld<f32x4>(lf), w = ld<f32x4>(lf + 4);
#pragma unroll
                    for (int e = 0; e < 4; ++e) { b[e] = u[e]; b[4 + e] = w[e]; }
                } else {
                    unpack8(ld<u32x4>((const bf16_t*)p.Olo + lrow + ks * 16), b);
                }
                unpack8(__builtin_bit_cast(u32x4, dof[ks]), g);
#pragma unroll
                for (int e = 0; e < 8; ++e) dl = fmaf(g[e], a[e] + b[e], dl);
            }
            dl += lane32_other(dl);
            if (qin && hi == 0) p.delta[(long)h * p.Tq + row] = dl;
        }
        const float lse = qin ? p.lse2[(long)h * p.Tq + row] : LSE_EMPTY;
        if (!qin) dl = 0.f;
        f32x16 dq[2] = {zero16(), zero16()};
        asm volatile("" ::"v"(qf[0]), "v"(qf[1]), "v"(qf[2]), "v"(qf[3]), "v"(dof[0]), "v"(dof[1]), "v"(dof[2]), "v"(dof[3]), "v"(lse), "v"(dl));
        auto fetch = [&](int kt, unsigned char* S) __attribute__((always_inline)) {
            sg.issue(Kb + (long)(kt * 64) * p.sk, Vb + (long)(kt * 64) * p.sv, D.nk - 1 - kt * 64, S);
        };
        if (nt > 0) fetch(0, smem);
        if (nt > 1) fetch(1, smem + STAGE);
        auto step = [&](auto stage_, int kt) __attribute__((always_inline)) {
            constexpr int S = decltype(stage_)::value * STAGE;
            const int k0 = kt * 64;
            if (kt + 1 < nt) wait_vmcnt<4>();
            else wait_vmcnt<0>();
            barrier_raw();
            if (kt + 2 < nt) fetch(kt + 2, smem + (decltype(stage_)::value + 2) % NST * STAGE);
            auto block = [&](auto kb_) __attribute__((always_inline)) {
                constexpr int kb = decltype(kb_)::value;
                const int kk = k0 + 32 * kb;
                if (kk >= lim_hi) return;
                f32x16 s = zero16(), dp = zero16();
                bf16x8 kt_[2][2];
                {
                    bf16x8 kf[4], vf[4];
                    lds_read8<S + kb * 4096, S + 8192 + kb * 4096>(kf, vf, fra);
#pragma unroll
                    for (int ks = 0; ks < 4; ++ks) {
                        s = mfma32(kf[ks], qf[ks], s);
                        dp = mfma32(vf[ks], dof[ks], dp);
                    }
                }
                sched_fence();
                tr_frags<S + kb * 4096>(kt_, tra);
                sched_fence();
                float t[16];
                const int qp = q0 + D.off, lo = kk - qp, rel = kk + 8 * hi - (qp + l31);
                const float mo = lse - sc.offset(rel, lo);
                sc.args(s, t, rel, lo, [&](int) { return mo; });
                if (kk + 32 > lim_lo) {
                    cold_path();
                    const int n = lim - (kk + 8 * hi);
#pragma unroll
                    for (int r = 0; r < 16; ++r) t[r] = reg_off(r) < n ? t[r] : -__builtin_inff();
                }
#pragma unroll
                for (int r = 0; r < 16; ++r) t[r] = fast_exp2(t[r]) * (dp[r] - dl);            // dS
                if (RG) {
                    if (lo + 31 <= -p.R || lo - 31 >= p.R) {
                        float a = 0.f;
#pragma unroll
                        for (int r = 0; r < 16; ++r) a += t[r];
                        if (lo < 0) far_lo += a; else far_hi += a;
                    } else {
                        diag_add(t, myscr, mydist + PADL + p.R + lo, l31, hi);
                    }
                }
                if (CAP) {
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        const float th = s[r] * icl;
                        t[r] *= fmaf(-th, th, 1.f);
                    }
                }
                const bf16x8 df[2] = {pack8f(t), pack8f(t + 8)};
#pragma unroll
                for (int s2 = 0; s2 < 2; ++s2)
#pragma unroll
                    for (int db = 0; db < 2; ++db) dq[db] = mfma32(kt_[s2][db], df[s2], dq[db]);
            };
            block(Int<0>{});
            block(Int<1>{});
        };
        for (int kt = 0; kt < nt; kt += NST) {
            step(Int<0>{}, kt);
            if (kt + 1 < nt) step(Int<1>{}, kt + 1);
            if (kt + 2 < nt) step(Int<2>{}, kt + 2);
        }
        if (live) {
            bf16_t* drow = p.dQ + ((long)row * p.H + h) * DH;
            store_rows32(dq, hi, qin, [&](int db, int g, int hi_, bool ok, const float* a, const float* b) __attribute__((always_inline)) {
                float v[8];
#pragma unroll
                for (int e = 0; e < 4; ++e) { v[e] = a[e] * p.scale; v[4 + e] = b[e] * p.scale; }
                u32x2 x = pack4(v), y = pack4(v + 4);
                swap_pair(x, y);
                if (ok) st<u32x4>(drow + 32 * db + 8 * (g + hi_), u32x4{x[0], x[1], y[0], y[1]});
            });
        }
        if ((tile + p.nt) * 128 < D.nq) __syncthreads();
    }
    if (RG) {
        // sums by distance, clamped at the reach: entries beyond it join the ends, with the far blocks' sums; four waves in order
        far_lo = wave_sum_fast(far_lo);
        far_hi = wave_sum_fast(far_hi);
        wave_sync();
        float a = lane < PADL ? mydist[lane] : 0.f, b = lane < PADL ? mydist[PADL + 2 * p.R + 1 + lane] : 0.f;
        a = wave_sum_fast(a);
        b = wave_sum_fast(b);
        wave_sync();
        if (lane == 0) {
            mydist[PADL] += far_lo + a;
            mydist[PADL + 2 * p.R] += far_hi + b;
        }
        __syncthreads();
        float* out = p.dist + (h * dist_rows(p.nd, p.Tq) + dist_row(wk.d, D.q0) + wk.tile) * (2 * p.R + 1);
        for (int i = tid; i < 2 * p.R + 1; i += 256) {
            const float* d = dist + PADL + i;
            out[i] = (d[0] + d[ND]) + (d[2 * ND] + d[3 * ND]);
        }
    }
}

// sums over the tiles of a head -> by_dist[h][2 R + 1]; 64 distances x 16 row groups per workgroup (5 us: latency of its dependent loads).  64 documents at a
// time: their rows are listed (a thread each finds its document by bisection), then added in the list's order
__global__ __launch_bounds__(1024) void pa_dist_reduce_kernel(PAArgs p, float* by_dist) {
    __shared__ float sm[16][64];
    __shared__ int first[64], tiles[64], upto[65], list[1024];
    const int tid = threadIdx.x, lane = tid & 63, grp = tid >> 6, h = blockIdx.y;
    const int N = 2 * p.R + 1, i = blockIdx.x * 64 + lane;
    float a = 0.f;
    const float* q = p.dist + h * dist_rows(p.nd, p.Tq) * N + i;
    for (int d0 = 0; d0 < p.nd; d0 += 64) {
        const int nd = min(64, p.nd - d0);
        if (tid < nd) {
            const Span s = span(p.cu_q, p.len_q, d0 + tid, p.Tq);
            first[tid] = dist_row(d0 + tid, s.at);
            tiles[tid] = min((s.n + 127) / 128, p.nt);            // (a workgroup takes the tiles from nt on into its first one's row)
        }
        __syncthreads();
        if (tid <= nd) {
            int sum = 0;
            for (int j = 0; j < tid; ++j) sum += tiles[j];
            upto[tid] = sum;
        }
        __syncthreads();
        const int total = upto[nd];
        for (int seg = 0; seg < total; seg += 1024) {
            const int f = seg + tid, n = min(1024, total - seg);
            if (f < total) {
                int j = 0, end = nd;                               // upto[j] <= f < upto[end]
                while (end - j > 1) {
                    const int mid = (j + end) / 2;
                    if (upto[mid] <= f) j = mid; else end = mid;
                }
                list[tid] = first[j] + f - upto[j];
            }
            __syncthreads();
            if (i < N) {
#pragma unroll 4
                for (int w = grp; w < n; w += 16) a += q[(long)list[w] * N];
            }
            __syncthreads();
        }
    }
    sm[grp][lane] = a;
    __syncthreads();
    if (grp == 0 && i < N) {
        a = 0.f;
#pragma unroll
        for (int g = 0; g < 16; ++g) a += sm[g][lane];
        by_dist[(long)h * N + i] = a;
    }
}
// sums over the distances of a bucket -> dtable[bucket][h]; one wave each (5 us, a launch)
__global__ __launch_bounds__(256) void pa_table_grad_kernel(const float* by_dist, const int* buckets, int N, int nbuckets, int H, float* dtable, int accumulate) {
    const int lane = threadIdx.x & 63, w = blockIdx.x * 4 + uniform_i(threadIdx.x >> 6);
    if (w >= nbuckets * H) return;
    const int b = w / H, h = w % H;
    float a = 0.f;
    for (int i = lane; i < N; i += 64) a += clampi(buckets[i], 0, nbuckets - 1) == b ? by_dist[(long)h * N + i] : 0.f;
    a = wave_sum_fast(a);
    if (lane == 0) dtable[w] = accumulate ? dtable[w] + a : a;
}

// ------------------------------------------------------------------------------------------------ backward: dK, dV

// One workgroup = 128 keys of one (document, key head); sweep over the 64-query tiles of all its query heads.  The query rows of the Q / dO tiles
// are K-type images, so the accumulators (rows = queries) are the B operands of dV^T = dO^T P and dK^T = Q^T dS; their A operands come out of the
// same tiles by transposing reads.  The 64 lse / delta values of a query tile ride along in the ring stage.  Two workgroups a CU (64 accumulators and
// 32 operand registers a lane); 8 x 1056 tokens x 16 heads, no bias: 111 us (matrix pipe and vector ALU 36 % each of the clocks in which a CU has work); of
// 108 on one box score products 18, output products 24, transposing reads 9, tile copies 5, exp2 3 when each is left out alone: no single resource binds it.
// Few key heads and tokens leave the chip's 512 slots for these workgroups empty: the sweep is then cut into `splits` parts whose fp32 sums a second
// kernel adds in order (7392 tokens, 4 key heads of 16: 271 us whole, see splits_for for the rule).
constexpr int KSTAGE = STAGE + 512;

template <int BIAS, bool CAP>
__global__ __launch_bounds__(256, 2) void pa_dkv_kernel(PAArgs p) {
    __shared__ __attribute__((aligned(16))) unsigned char smem[NST * KSTAGE];
    __shared__ float lut[BIAS == 2 ? 2 * distn(REACH_MAX) : 1];        // two heads' tables in turn
    lds_declare(smem, sizeof(smem));
    if ((int)blockIdx.x >= p.nwork) {
        fill_gap(p.cu_k, p.len_k, p.nd, p.Tk, p.dK, (long)p.Hkv * DH, DH, p.Hkv, (int)blockIdx.x - p.nwork);
        fill_gap(p.cu_k, p.len_k, p.nd, p.Tk, p.dV, (long)p.Hkv * DH, DH, p.Hkv, (int)blockIdx.x - p.nwork);
        return;
    }
    const int tid = threadIdx.x, lane = tid & 63, wave = uniform_i(tid >> 6);
    const int l31 = lane & 31, hi = lane >> 5;
    Work wk = work_of(p, p.cu_q, p.len_q, p.Tq);   // (key head, document, tile) x part
    const int part = wk.h % p.splits;
    wk.h /= p.splits;
    const Doc D = doc_of(p, wk.d);
    const int tile0 = p.nt - 1 - wk.tile;          // (causal: the first keys are seen by the most queries)
    if (tile0 * 128 >= D.nk) return;
    Stager sg;
    sg.init(wave, lane, p.sq, p.sg);
    unsigned fra[4];
    frag_addr(smem, l31, hi, fra);
    const TrAddr tra = tr_addr(smem, lane);
    const float icl = CAP ? 1.f / (p.cap * LOG2E) : 0.f;
    const int nqt = (D.nq + 63) / 64;

    for (int tile = tile0; tile * 128 < D.nk; tile += p.nt) {
        const int kk = tile * 128 + wave * 32, key = kk + l31;
        const bool live = kk < D.nk, kin = key < D.nk;
        bf16x8 kf[4], vf[4];
        row_frags(kf, p.K + (long)(D.k0 + (kin ? key : 0)) * p.sk + (long)wk.h * p.hk, kin, hi);
        row_frags(vf, p.V + (long)(D.k0 + (kin ? key : 0)) * p.sv + (long)wk.h * p.hv, kin, hi);
        f32x16 dk[2] = {zero16(), zero16()}, dv[2] = {zero16(), zero16()};
        // first query that sees this lane's key, and the first query tile that sees any key of the workgroup
        const int qmin = (!D.causal || key < D.prefix) ? -0x40000000 : key - D.off;
        int t0 = 0;
        if (D.causal && tile * 128 >= D.prefix) t0 = max(0, tile * 128 - D.off) / 64;
        const int per = max(0, nqt - t0), all = per * p.G;
        const int it0 = (int)((long)all * part / p.splits), total = (int)((long)all * (part + 1) / p.splits) - it0;
        int ih = per ? it0 / per : 0, iq = it0 - ih * per, ch = ih, cq = iq;          // head and tile that is fetched / computed next
        auto issue = [&](int it) __attribute__((always_inline)) {
            const int h = wk.h * p.G + ih, q0 = (t0 + iq) * 64;
            if (++iq == per) { iq = 0; ++ih; }
            unsigned char* S = smem + it % NST * KSTAGE;
            const long r = D.q0 + q0;
            sg.issue(p.Q + r * p.sq + (long)h * p.hq, p.dO + r * p.sg + (long)h * p.hg, D.nq - 1 - q0, S);
            if (wave < 2) glds4((wave == 0 ? p.lse2 : p.delta) + (long)h * p.Tq + r + min(lane, D.nq - 1 - q0), S + STAGE + wave * 256);
        };
        Scorer<BIAS, CAP, -1, false, true> sc;
        sc.init(p, BIAS == 1 ? p.slopes[wk.h * p.G + min(ch, p.G - 1)] : 0.f);
        if (BIAS == 2) {
            sc.R = p.R;
            if (total > 0) load_lut(p, wk.h * p.G + ch, lut + (ch & 1) * distn(REACH_MAX));
            wait_lgkm0();
        }
        asm volatile("" ::"v"(kf[0]), "v"(kf[1]), "v"(kf[2]), "v"(kf[3]), "v"(vf[0]), "v"(vf[1]), "v"(vf[2]), "v"(vf[3]));
        if (total > 0) issue(0);
        if (total > 1) issue(1);
        auto step = [&](auto stage_, int it) __attribute__((always_inline)) {
            constexpr int S = decltype(stage_)::value * KSTAGE;
            const int hd = ch, j0 = cq, q0 = (t0 + j0) * 64;
            if (++cq == per) { cq = 0; ++ch; }
            // (waves 0 and 1 have five copies a tile, the others four: four may be in flight at most)
            if (it + 1 < total) wait_vmcnt<4>();
            else wait_vmcnt<0>();
            barrier_raw();
            if (it + 2 < total) issue(it + 2);
            if (BIAS == 1 && p.G > 1 && j0 == 0 && it > 0) sc.init(p, p.slopes[wk.h * p.G + hd]);
            if (BIAS == 2) {
                if (j0 == 0 || it == 0) {                     // (its LDS reads wait for every copy in flight: once a head, not once a tile)
                    float* L = lut + (hd & 1) * distn(REACH_MAX);
                    sc.lut = L;
                    sc.far_lo = L[PADL];
                    sc.far_hi = L[PADL + 2 * p.R];
                }
                // the next head's table while this head's last tile is computed (the other buffer: its last reader passed the barrier above)
                if (j0 == per - 1 && hd + 1 < p.G) {
                    load_lut(p, wk.h * p.G + hd + 1, lut + ((hd + 1) & 1) * distn(REACH_MAX));
                    wait_lgkm0();
                }
            }
            if (!live) return;
            const float* lse_s = (const float*)(smem + (S + STAGE));
            auto block = [&](auto qb_) __attribute__((always_inline)) {
                constexpr int qb = decltype(qb_)::value;
                const int qq = q0 + 32 * qb;                  // first query of the block
                if (qq >= D.nq || D.lim(min(qq + 31, D.nq - 1)) <= kk) return;
                f32x16 s = zero16(), dp = zero16();
                bf16x8 dot_[2][2], qt_[2][2];
                {
                    bf16x8 qf[4], gf[4];
                    lds_read8<S + qb * 4096, S + 8192 + qb * 4096>(qf, gf, fra);
#pragma unroll
                    for (int ks = 0; ks < 4; ++ks) {
                        s = mfma32(qf[ks], kf[ks], s);
                        dp = mfma32(gf[ks], vf[ks], dp);
                    }
                }
                sched_fence();
                tr_frags<S + 8192 + qb * 4096>(dot_, tra);
                tr_frags<S + qb * 4096>(qt_, tra);
                sched_fence();
                float t[16], ds[16];
                const int qp = qq + D.off, lo = kk - qp, rel = key - (qp + 8 * hi);
                const float c = sc.offset(rel, lo);
                const float* ls = lse_s + 32 * qb + 8 * hi;
                f32x4 l4[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) l4[i] = ld<f32x4>(ls + reg_off(4 * i));
                sc.args(s, t, rel, lo, [&](int r) { return BIAS == 0 ? l4[r >> 2][r & 3] : l4[r >> 2][r & 3] - c; });
                if (D.lim(qq) < kk + 32 || qq + 32 > D.nq) {
                    cold_path();
                    const int a = qmin - (qq + 8 * hi), b = D.nq - (qq + 8 * hi);
#pragma unroll
                    for (int r = 0; r < 16; ++r) t[r] = (reg_off(r) >= a && reg_off(r) < b) ? t[r] : -__builtin_inff();
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const f32x4 d4 = ld<f32x4>(ls + 64 + reg_off(4 * i));
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int r = 4 * i + j;
                        t[r] = fast_exp2(t[r]);
                        ds[r] = t[r] * (dp[r] - d4[j]);
                        if (CAP) {
                            const float th = s[r] * icl;
                            ds[r] *= fmaf(-th, th, 1.f);
                        }
                    }
                }
                const bf16x8 pf[2] = {pack8f(t), pack8f(t + 8)}, df[2] = {pack8f(ds), pack8f(ds + 8)};
#pragma unroll
                for (int s2 = 0; s2 < 2; ++s2)
#pragma unroll
                    for (int db = 0; db < 2; ++db) {
                        dv[db] = mfma32(dot_[s2][db], pf[s2], dv[db]);
                        dk[db] = mfma32(qt_[s2][db], df[s2], dk[db]);
                    }
            };
            block(Int<0>{});
            block(Int<1>{});
        };
        for (int it = 0; it < total; it += NST) {
            step(Int<0>{}, it);
            if (it + 1 < total) step(Int<1>{}, it + 1);
            if (it + 2 < total) step(Int<2>{}, it + 2);
        }
        if (live) {
            const long orow = ((long)(D.k0 + (kin ? key : 0)) * p.Hkv + wk.h) * DH;
            if (p.splits > 1) {
                float* ws = p.part + (long)part * 2 * p.Tk * p.Hkv * DH + orow;
                if (kin) {
#pragma unroll
                    for (int db = 0; db < 2; ++db)
#pragma unroll
                        for (int g = 0; g < 4; ++g) {
                            const int col = 32 * db + 8 * g + 4 * hi;
                            st<f32x4>(ws + col, f32x4{dk[db][4 * g], dk[db][4 * g + 1], dk[db][4 * g + 2], dk[db][4 * g + 3]});
                            st<f32x4>(ws + (long)p.Tk * p.Hkv * DH + col, f32x4{dv[db][4 * g], dv[db][4 * g + 1], dv[db][4 * g + 2], dv[db][4 * g + 3]});
                        }
                }
            } else {
                auto put = [&](bf16_t* dst, float f, int db, int g, int hi_, bool ok, const float* a, const float* b) __attribute__((always_inline)) {
                    float v[8];
#pragma unroll
                    for (int e = 0; e < 4; ++e) { v[e] = a[e] * f; v[4 + e] = b[e] * f; }
                    u32x2 x = pack4(v), y = pack4(v + 4);
                    swap_pair(x, y);
                    if (ok) st<u32x4>(dst + orow + 32 * db + 8 * (g + hi_), u32x4{x[0], x[1], y[0], y[1]});
                };
                store_rows32(dk, hi, kin, [&](int db, int g, int hi_, bool ok, const float* a, const float* b) __attribute__((always_inline)) { put(p.dK, p.scale, db, g, hi_, ok, a, b); });
                store_rows32(dv, hi, kin, [&](int db, int g, int hi_, bool ok, const float* a, const float* b) __attribute__((always_inline)) { put(p.dV, 1.f, db, g, hi_, ok, a, b); });
            }
        }
        if ((tile + p.nt) * 128 < D.nk) __syncthreads();
    }
}

// dK, dV = sums of the parts; eight columns a thread
__global__ __launch_bounds__(256) void pa_dkv_join_kernel(PAArgs p) {
    const int tile = (int)blockIdx.x % p.nt, d = (int)blockIdx.x / p.nt, w = p.Hkv * DH;
    const Span s = span(p.cu_k, p.len_k, d, p.Tk);
    for (int r0 = tile * JOIN_ROWS; r0 < s.n; r0 += p.nt * JOIN_ROWS) {
        const int rows = min(JOIN_ROWS, s.n - r0);
        const long base = (long)(s.at + r0) * w;
        for (int i = threadIdx.x; i < rows * (w / 8); i += 256) {
            const long at = base + (long)i * 8;
            float a[8], b[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) { a[e] = 0.f; b[e] = 0.f; }
            for (int q = 0; q < p.splits; ++q) {
                const float* x = p.part + (long)q * 2 * p.Tk * w + at;
                const float* y = x + (long)p.Tk * w;
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const f32x4 u = ld<f32x4>(x + 4 * c), v = ld<f32x4>(y + 4 * c);
#pragma unroll
                    for (int e = 0; e < 4; ++e) { a[4 * c + e] += u[e]; b[4 * c + e] += v[e]; }
                }
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) a[e] *= p.scale;
            st<u32x4>(p.dK + at, pack8(a));
            st<u32x4>(p.dV + at, pack8(b));
        }
    }
}

// ------------------------------------------------------------------------------------------------ host side

// Parts of a query row's keys (inference): as many as bring the workgroups to one per CU, each with four key tiles or more; at most eight, sixteen
// where that leaves a part 1024 keys.  Whole / in parts, with the join: 890 queries of 16 heads over up to 4097 keys 62 / 44 us (42 + 7 in twice as
// many parts), 16 queries over 4097 keys 59 / 22 (28 in sixteen), 1 query over 30000 402 / 60 (40 in sixteen), 256 over 1000 20 / 18.
int fwd_splits_for(int Tq, int H, int max_k, int Tk) {
    if (max_k <= 0 || max_k > Tk) max_k = Tk;
    const long wgs = (long)((Tq + 127) / 128) * H;
    if (wgs < 1) return 1;
    long s = 256 / wgs;
    if (s > max_k / 256) s = max_k / 256;
    const long most = max_k >= 16 * 1024 ? 16 : 8;
    return (int)(s < 1 ? 1 : s > most ? most : s);
}
// Parts of a key tile's sweep: as many as bring the workgroups to twice the chip's 512 slots, at most eight, each with four query tiles or more
int splits_for(int Tk, int H, int Hkv, int max_q, int Tq) {
    if (max_q <= 0 || max_q > Tq) max_q = Tq;
    const long wgs = (long)((Tk + 127) / 128) * Hkv, sweep = (long)(H / Hkv) * ((max_q + 63) / 64);
    if (wgs < 1 || wgs >= 384) return 1;
    long s = 1024 / wgs;
    if (s > sweep / 4) s = sweep / 4;
    return (int)(s < 1 ? 1 : s > 8 ? 8 : s);
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }
bool strides_ok(long t, long h) { return t % 8 == 0 && h % 8 == 0 && t >= 0 && h >= 0 && t < (1 << 23); }

// sizes, pointers and layouts that the kernels assume
int check(const PAArgs& a) {
    if (a.nd < 0 || a.Tq < 0 || a.Tk < 0 || a.H < 1 || a.Hkv < 1 || a.H % a.Hkv != 0) return E2K_ERR_SHAPE;
    if (a.nd > 0 && (!a.cu_q || !a.cu_k)) return E2K_ERR_ARG;
    if (!score_range_ok(a.scale, a.cap)) return E2K_ERR_ARG;
    if (a.slopes && a.table) return E2K_ERR_ARG;
    if (a.table && (!a.buckets || a.nbuckets < 1 || a.R < 0 || a.R > REACH_MAX)) return E2K_ERR_SHAPE;
    if ((a.Tq > 0 && !a.Q) || (a.Tk > 0 && (!a.K || !a.V))) return E2K_ERR_ARG;
    if (!strides_ok(a.sq, a.hq) || !strides_ok(a.sk, a.hk) || !strides_ok(a.sv, a.hv) || !strides_ok(a.so, a.ho)) return E2K_ERR_ALIGN;
    if (!aligned16(a.Q) || !aligned16(a.K) || !aligned16(a.V) || !aligned16(a.O)) return E2K_ERR_ALIGN;
    return E2K_OK;
}
// 128-row tiles per (document, head) of a grid: those of the longest document, fewer where documents x heads would make the grid absurd (every
// document gets as many workgroups as the longest is thought to need; a workgroup takes further tiles of its document in turn)
int tiles_for(int longest, int total, int nd, int heads) {
    if (longest <= 0 || longest > total) longest = total;
    const long most = 262144 / ((long)(nd > 0 ? nd : 1) * heads);
    long nt = ((long)longest + 127) / 128;
    if (nt > most) nt = most;
    return (int)(nt < 1 ? 1 : nt);
}
int plan_grid(PAArgs& a, int longest, int total, int heads, long& grid) {
    a.nt = tiles_for(longest, total, a.nd, heads);
    const long work = (long)a.nd * a.nt * heads;
    grid = work + (a.fill ? ((long)a.nd + 1) * GAP_PARTS : 0);
    if (grid > 0x7fffffffL / 256) return E2K_ERR_SHAPE;
    a.nwork = (int)work;
    a.heads = heads;
    a.order = a.nd > 1 && a.nd <= 64 && work > 512;
    return E2K_OK;
}
// the same rows in JOIN_ROWS-row tiles
void plan_join(PAArgs& a) {
    const long most = 65536 / a.nd;
    long nt = (long)a.nt * (128 / JOIN_ROWS);
    if (nt > most) nt = most;
    a.nt = (int)(nt < 1 ? 1 : nt);
}

template <int BIAS, bool CAP> void run_fwd(const PAArgs& a, bool train, long grid, hipStream_t st) {
    if (train) hipLaunchKernelGGL((pa_fwd_kernel<BIAS, CAP, true>), dim3((unsigned)grid), dim3(256), 0, st, a);
    else hipLaunchKernelGGL((pa_fwd_kernel<BIAS, CAP, false>), dim3((unsigned)grid), dim3(256), 0, st, a);
}
template <int BIAS, bool CAP> void run_dq(const PAArgs& a, int rg, long grid, hipStream_t st) {
    if (BIAS == 2 && rg == 1) hipLaunchKernelGGL((pa_dq_kernel<BIAS, CAP, BIAS == 2 ? 128 : 0>), dim3((unsigned)grid), dim3(256), 0, st, a);
    else if (BIAS == 2 && rg == 2) hipLaunchKernelGGL((pa_dq_kernel<BIAS, CAP, BIAS == 2 ? REACH_MAX : 0>), dim3((unsigned)grid), dim3(256), 0, st, a);
    else hipLaunchKernelGGL((pa_dq_kernel<BIAS, CAP, 0>), dim3((unsigned)grid), dim3(256), 0, st, a);
}
template <int BIAS, bool CAP> void run_dkv(const PAArgs& a, int, long grid, hipStream_t st) {
    hipLaunchKernelGGL((pa_dkv_kernel<BIAS, CAP>), dim3((unsigned)grid), dim3(256), 0, st, a);
}
#define PA_PICK(FN, a, ...)                                                                       \
    do {                                                                                          \
        const bool cap_ = (a).cap > 0.f;                                                          \
        if ((a).table) { if (cap_) FN<2, true>(a, __VA_ARGS__); else FN<2, false>(a, __VA_ARGS__); }        \
        else if ((a).slopes) { if (cap_) FN<1, true>(a, __VA_ARGS__); else FN<1, false>(a, __VA_ARGS__); }  \
        else { if (cap_) FN<0, true>(a, __VA_ARGS__); else FN<0, false>(a, __VA_ARGS__); }                  \
    } while (0)

PAArgs common(const void* Q, int64_t sq, int64_t hq, const void* K, int64_t sk, int64_t hk, const void* V, int64_t sv, int64_t hv, const int32_t* cu_q,
              const int32_t* cu_k, const int32_t* len_q, const int32_t* len_k, const int32_t* prefix, int nd, int Tq, int Tk, int H, int Hkv, int causal,
              float scale, float softcap, const float* slopes, const float* table, const int32_t* buckets, int nbuckets, int reach) {
    PAArgs a{};
    a.Q = (const bf16_t*)Q; a.K = (const bf16_t*)K; a.V = (const bf16_t*)V;
    a.sq = sq; a.hq = hq; a.sk = sk; a.hk = hk; a.sv = sv; a.hv = hv;
    a.cu_q = cu_q; a.cu_k = cu_k; a.len_q = len_q; a.len_k = len_k; a.prefix = prefix;
    a.nd = nd; a.Tq = Tq; a.Tk = Tk; a.H = H; a.Hkv = Hkv; a.G = Hkv > 0 ? H / Hkv : 1;
    a.causal = causal; a.scale = scale; a.cap = softcap;
    a.slopes = slopes; a.table = table; a.buckets = buckets; a.nbuckets = nbuckets; a.R = reach;
    return a;
}

int packed_attn_fwd_impl(const void* Q, int64_t sq, int64_t hq, const void* K, int64_t sk, int64_t hk, const void* V, int64_t sv, int64_t hv,
                         const int32_t* cu_q, const int32_t* cu_k, const int32_t* len_q, const int32_t* len_k, const int32_t* prefix, int nd, int Tq,
                         int Tk, int H, int Hkv, int max_q, int max_k, int causal, float scale, float softcap, const float* slopes, const float* table,
                         const int32_t* buckets, int nbuckets, int reach, void* O, int64_t so, int64_t ho, void* Olo, float* lse2, float* ws,
                         int fill_gaps, void* stream) {
    PAArgs a = common(Q, sq, hq, K, sk, hk, V, sv, hv, cu_q, cu_k, len_q, len_k, prefix, nd, Tq, Tk, H, Hkv, causal, scale, softcap, slopes, table,
                      buckets, nbuckets, reach);
    a.O = (bf16_t*)O; a.so = so; a.ho = ho; a.Olo = (void*)Olo; a.lse2 = lse2; a.fill = fill_gaps;
    if (Tq == 0) return E2K_OK;
    const int rc = check(a);
    if (rc) return rc;
    if (!O || (!Olo) != (!lse2)) return E2K_ERR_ARG;
    if (!aligned16(Olo)) return E2K_ERR_ALIGN;
    a.splits = Olo ? 1 : fwd_splits_for(Tq, H, max_k, Tk);
    a.part = ws;
    if (a.splits > 1 && !ws) return E2K_ERR_ARG;
    long grid;
    const int rg = plan_grid(a, max_q, Tq, H * a.splits, grid);
    if (rg) return rg;
    if (grid == 0) return E2K_OK;
    hipStream_t st = (hipStream_t)stream;
    PA_PICK(run_fwd, a, Olo != nullptr, grid, st);
    E2K_CHECK_LAUNCH();
    if (a.splits > 1 && a.nwork > 0) {
        plan_join(a);
        hipLaunchKernelGGL(pa_fwd_join_kernel, dim3((unsigned)(a.nd * a.nt)), dim3(256), 0, st, a);
        E2K_CHECK_LAUNCH();
    }
    return E2K_OK;
}

int packed_attn_bwd_impl(const void* dO, int64_t sg, int64_t hg, const void* Q, int64_t sq, int64_t hq, const void* K, int64_t sk, int64_t hk,
                         const void* V, int64_t sv, int64_t hv, const int32_t* cu_q, const int32_t* cu_k, const int32_t* len_q, const int32_t* len_k,
                         const int32_t* prefix, int nd, int Tq, int Tk, int H, int Hkv, int max_q, int max_k, int causal, float scale, float softcap,
                         const float* slopes, const float* table, const int32_t* buckets, int nbuckets, int reach, const void* O, int64_t so, int64_t ho,
                         const void* Olo, const float* lse2, float* delta, void* dQ, void* dK, void* dV, float* dtable, int accumulate, float* ws,
                         int fill_gaps, void* stream) {
    PAArgs a = common(Q, sq, hq, K, sk, hk, V, sv, hv, cu_q, cu_k, len_q, len_k, prefix, nd, Tq, Tk, H, Hkv, causal, scale, softcap, slopes, table,
                      buckets, nbuckets, reach);
    a.dO = (const bf16_t*)dO; a.sg = sg; a.hg = hg; a.O = (bf16_t*)O; a.so = so; a.ho = ho; a.Olo = (void*)Olo; a.lse2 = (float*)lse2; a.delta = delta;
    a.dQ = (bf16_t*)dQ; a.dK = (bf16_t*)dK; a.dV = (bf16_t*)dV; a.dist = ws; a.fill = fill_gaps;
    hipStream_t st = (hipStream_t)stream;
    long grid;
    const int rc = check(a);                   // (also without queries: keys are read and their gradients written all the same)
    if (rc) return rc;
    if (Tq > 0) {
        if (!dO || !O || !Olo || !lse2 || !delta || !dQ || (dtable && (!table || !ws))) return E2K_ERR_ARG;
        if (!strides_ok(sg, hg) || !aligned16(dO) || !aligned16(Olo) || !aligned16(dQ) || !aligned16(dK) || !aligned16(dV)) return E2K_ERR_ALIGN;
        if (Tk > 0 && (!dK || !dV)) return E2K_ERR_ARG;
        a.splits = 1;
        const int rg = plan_grid(a, max_q, Tq, H, grid);
        if (rg) return rg;
        if (grid > 0) {
            PA_PICK(run_dq, a, dtable ? (reach <= 128 ? 1 : 2) : 0, grid, st);
            E2K_CHECK_LAUNCH();
        }
    }
    float* rest = ws;                          // workspace behind the table's part
    if (dtable) {
        if (!table || !buckets || !ws || nbuckets < 1 || reach < 0 || reach > REACH_MAX) return E2K_ERR_ARG;
        const int N = 2 * reach + 1;
        const long sums = H * dist_rows(nd, Tq) * N;          // (no query rows: none, and no tiles to add)
        float* by_dist = ws + sums;
        hipLaunchKernelGGL(pa_dist_reduce_kernel, dim3((N + 63) / 64, H), dim3(1024), 0, st, a, by_dist);
        E2K_CHECK_LAUNCH();
        hipLaunchKernelGGL(pa_table_grad_kernel, dim3((nbuckets * H + 3) / 4), dim3(256), 0, st, by_dist, buckets, N, nbuckets, H, dtable, accumulate);
        E2K_CHECK_LAUNCH();
        rest = ws + (sums + (long)H * N + 3) / 4 * 4;          // (16-byte rows)
    }
    if (Tk > 0) {
        if (!dK || !dV || !aligned16(dK) || !aligned16(dV)) return E2K_ERR_ARG;
        a.splits = splits_for(Tk, H, Hkv, max_q, Tq);
        a.part = rest;
        if (a.splits > 1 && !ws) return E2K_ERR_ARG;
        const int rg = plan_grid(a, max_k, Tk, Hkv * a.splits, grid);
        if (rg) return rg;
        if (a.splits > 1) a.order = 0;
        if (grid > 0) {
            PA_PICK(run_dkv, a, 0, grid, st);
            E2K_CHECK_LAUNCH();
        }
        if (a.splits > 1 && a.nwork > 0) {
            plan_join(a);
            hipLaunchKernelGGL(pa_dkv_join_kernel, dim3((unsigned)(a.nd * a.nt)), dim3(256), 0, st, a);
            E2K_CHECK_LAUNCH();
        }
    }
    return E2K_OK;
}

}  // namespace

extern "C" {

int64_t e2k_query_packed_attn_fwd_ws_floats(int Tq, int Tk, int H, int max_k) {
    if (Tq < 1 || Tk < 0 || H < 1) return 0;
    const int s = fwd_splits_for(Tq, H, max_k, Tk);
    return s > 1 ? (int64_t)s * Tq * H * (DH + 2) : 0;
}
int e2k_packed_attn_fwd(const void* Q, int64_t sq, int64_t hq, const void* K, int64_t sk, int64_t hk, const void* V, int64_t sv, int64_t hv,
                        const int32_t* cu_q, const int32_t* cu_k, const int32_t* len_q, const int32_t* len_k, const int32_t* prefix, int nd, int Tq,
                        int Tk, int H, int Hkv, int max_q, int max_k, int causal, float scale, float softcap, const float* slopes,
                        const float* table, const int32_t* buckets, int nbuckets, int reach, void* O, int64_t so, int64_t ho, void* Olo, float* lse2,
                        float* ws, int fill_gaps, void* stream) {
    return e2k::dispatch("packed_attn_fwd", packed_attn_fwd_impl, Q, sq, hq, K, sk, hk, V, sv, hv, cu_q, cu_k, len_q, len_k, prefix, nd, Tq, Tk, H, Hkv,
                         max_q, max_k, causal, scale, softcap, slopes, table, buckets, nbuckets, reach, O, so, ho, Olo, lse2, ws, fill_gaps, stream);
}
int64_t e2k_query_packed_attn_bwd_ws_floats(int nd, int Tq, int Tk, int H, int Hkv, int max_q, int reach, int dtable) {
    if (nd < 0 || Tq < 0 || Tk < 0 || H < 1 || Hkv < 1 || H % Hkv != 0 || reach < 0 || reach > REACH_MAX) return 0;
    const int s = splits_for(Tk, H, Hkv, max_q, Tq);
    const int64_t join = s > 1 ? (int64_t)s * 2 * Tk * Hkv * DH : 0;
    if (!dtable) return join;
    const int64_t sums = H * (dist_rows(nd, Tq) + 1) * (2 * (int64_t)reach + 1);
    return (sums + 3) / 4 * 4 + join;
}
int e2k_packed_attn_bwd(const void* dO, int64_t sg, int64_t hg, const void* Q, int64_t sq, int64_t hq, const void* K, int64_t sk, int64_t hk,
                        const void* V, int64_t sv, int64_t hv, const int32_t* cu_q, const int32_t* cu_k, const int32_t* len_q, const int32_t* len_k,
                        const int32_t* prefix, int nd, int Tq, int Tk, int H, int Hkv, int max_q, int max_k, int causal, float scale, float softcap,
                        const float* slopes, const float* table, const int32_t* buckets, int nbuckets, int reach, const void* O, int64_t so, int64_t ho,
                        const void* Olo, const float* lse2, float* delta, void* dQ, void* dK, void* dV, float* dtable, int accumulate, float* ws,
                        int fill_gaps, void* stream) {
    return e2k::dispatch("packed_attn_bwd", packed_attn_bwd_impl, dO, sg, hg, Q, sq, hq, K, sk, hk, V, sv, hv, cu_q, cu_k, len_q, len_k, prefix, nd, Tq,
                         Tk, H, Hkv, max_q, max_k, causal, scale, softcap, slopes, table, buckets, nbuckets, reach, O, so, ho, Olo, lse2, delta, dQ, dK,
                         dV, dtable, accumulate, ws, fill_gaps, stream);
}

}  // extern "C"
