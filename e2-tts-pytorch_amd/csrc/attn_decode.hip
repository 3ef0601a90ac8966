// Attention of ONE query token per sequence over a long key / value cache (dim_head 64): the serving form of packed_attn.hip's scores.
//
//   q stands at position n - 1 of its sequence's n cached keys and sees all of them:  z = scale q.k, c = cap tanh(z / cap),
//   t = c - slope_h |j - (n - 1)|  or  c + table[bucket(j - (n - 1)), h],  o = softmax(t) v;   n = 0: o = 0
//
// What bounds it: HBM, every K and V row of the cache once (410 MB of 32 ragged caches in 79 us: 5.2 TB/s, the rate of a large copy); the
// arithmetic has a factor of two to spare as long as it is not done by shuffles.
// The G query heads of a key head are the columns of a 32 x 32 MFMA (unused columns cost nothing that matters), so a K / V row is read once for
// all of them.  A wave walks its own share of the keys, 32 at a time, through an LDS ring of its own that LDS-DMA fills while the blocks before
// are computed: no barriers, only counted waits.  The keys of a sequence are split evenly over `splits` workgroups of four waves by its actual
// length; waves are joined in LDS, workgroups through a workspace by a second kernel (fixed order: the same bits every time).
#include "e2k_device.h"
#include "plan.h"
#include <e2k_asm.h>
#include "../../include/e2k.h"
#include "attn_tile32.h"
#include "attn_score.h"

using namespace e2k;

namespace {

constexpr int NW = 4;                 // waves per workgroup
constexpr int BLK = 8192;             // one ring stage: 32 keys of K and of V
constexpr int STAGES = 2;
constexpr int PART = 66;              // floats of a partial result: 64 columns, reference point, sum

struct DecodeArgs {
    const bf16_t *Q, *K, *V; long qb, qh, kb, kn, kh, vb, vn, vh, ob, oh;      // strides (elements): batch, key, head
    const int* lens; int B, cap_n, H, Hkv, G, ngrp, splits;
    float scale, cap;
    const float *slopes, *table; const int* buckets; int nbuckets, R;
    bf16_t* O; float* ws;
};

// HEADS: the four waves of a workgroup take the same keys of four neighbouring key heads (512 consecutive bytes of every cache row), else four
// runs of keys of one head, joined here.
template <int BIAS, bool CAP, bool HEADS>
__global__ __launch_bounds__(NW * 64, 2) void attn_decode_kernel(DecodeArgs p) {
    __shared__ __attribute__((aligned(16))) unsigned char smem[NW * STAGES * BLK];
    __shared__ float ml[NW][2][32];
    lds_declare(smem, sizeof(smem));
    const int tid = threadIdx.x, lane = tid & 63, wave = uniform_i(tid >> 6);
    const int l31 = lane & 31, hi = lane >> 5;
    // key heads fastest: neighbouring workgroups read neighbouring parts of the same rows
    int lin = (int)blockIdx.x;
    const int nhk = HEADS ? p.Hkv / NW : p.Hkv;
    const int hk = HEADS ? lin % nhk * NW + wave : lin % nhk; lin /= nhk;
    const int grp = HEADS ? 0 : lin % p.ngrp; lin /= p.ngrp;
    const int split = lin % p.splits, b = lin / p.splits;
    const int cols = min(32, p.G - 32 * grp), h0 = hk * p.G + 32 * grp;        // query heads h0 .. h0 + cols - 1
    const int n = uniform_i(clampi(p.lens[b], 0, p.cap_n));
    const int nblk = (n + 31) / 32;                                            // 32-key blocks of the sequence, shared evenly by splits x waves
    const long parts = HEADS ? p.splits : (long)p.splits * NW, me = HEADS ? split : (long)split * NW + wave;
    const int b0 = (int)(nblk * me / parts), b1 = (int)(nblk * (me + 1) / parts);

    const bool col = l31 < cols;
    const int h = h0 + (col ? l31 : 0);
    bf16x8 qf[4];
#pragma unroll
    for (int ks = 0; ks < 4; ++ks)
        qf[ks] = col ? ld<bf16x8>(p.Q + (long)b * p.qb + (long)h * p.qh + ks * 16 + hi * 8) : bf16x8{0, 0, 0, 0, 0, 0, 0, 0};
    const float sc2 = p.scale * LOG2E;
    Cap cp{};
    if (CAP) cp = cap_of<false>(p.scale, p.cap);
    const float sl2 = BIAS == 1 ? p.slopes[h] * LOG2E : 0.f;
    const float far = BIAS == 2 ? p.table[(long)clampi(p.buckets[0], 0, p.nbuckets - 1) * p.H + h] * LOG2E : 0.f;

    unsigned char* const ring = smem + wave * (STAGES * BLK);
    const bf16_t* Kb = p.K + (long)b * p.kb + (long)hk * p.kh;
    const bf16_t* Vb = p.V + (long)b * p.vb + (long)hk * p.vh;
    const unsigned sk = (unsigned)(p.kn * 2), sv = (unsigned)(p.vn * 2);
    auto issue = [&](int blk) __attribute__((always_inline)) {
        unsigned char* S = ring + (blk - b0) % STAGES * BLK;
        const char* ka = (const char*)(Kb + (long)blk * 32 * p.kn);
        const char* va = (const char*)(Vb + (long)blk * 32 * p.vn);
        const int last = n - 1 - blk * 32;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int r = u * 8 + (lane >> 3);
            const unsigned row = (unsigned)min(swap23(r), last), c = (unsigned)(((lane & 7) ^ swz(r)) * 16);
            glds16(ka + ((row & 0xffffffu) * (sk & 0xffffffu) + c), S + u * 1024);
            glds16(va + ((row & 0xffffffu) * (sv & 0xffffffu) + c), S + 4096 + u * 1024);
        }
    };
    unsigned fra[4];
    frag_addr(ring, l31, hi, fra);
    const TrAddr tra = tr_addr(ring, lane);
    f32x16 o[2] = {zero16(), zero16()};
    float m = M_INIT, l0 = 0.f, l1 = 0.f;
    asm volatile("" ::"v"(qf[0]), "v"(qf[1]), "v"(qf[2]), "v"(qf[3]), "v"(sl2), "v"(far));
#pragma unroll
    for (int s = 0; s < STAGES; ++s)
        if (b0 + s < b1) issue(b0 + s);
    auto step = [&](auto stage_, int blk) __attribute__((always_inline)) {
        constexpr int S = decltype(stage_)::value * BLK;
        // blocks blk + 1 .. blk + STAGES - 1 stay in flight (eight copies each)
        if (blk + STAGES - 1 < b1) wait_vmcnt<8 * (STAGES - 1)>();
        else wait_vmcnt<0>();
        wave_sync();
        f32x16 s = zero16();
        bf16x8 kf[4], vf[2][2];
        lds_read4<S>(kf, fra);
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) s = mfma32(kf[ks], qf[ks], s);
        sched_fence();
        tr_frags<S + 4096>(vf, tra);
        sched_fence();
        const int kk = blk * 32, rel = kk + 8 * hi - (n - 1);
        float t[16], c = 0.f;
        auto finish = [&](auto&& add) __attribute__((always_inline)) {
            if constexpr (CAP) {
                cap16<false, false>(s, t, cp, add);
            } else {
#pragma unroll
                for (int r = 0; r < 16; ++r) t[r] = fmaf(s[r], sc2, add(r));
            }
        };
        if (BIAS == 1) {
            c = sl2 * (float)rel;                              // (every key lies at or before the query)
            finish([&](int r) { return sl2 * (float)reg_off(r); });
        } else if (BIAS == 2 && kk + 31 - (n - 1) > -p.R) {
            cold_path();                                       // the last blocks only: within the table's reach
            finish([&](int r) {
                const int d = clampi(rel + reg_off(r), -p.R, 0) + p.R;
                return p.table[(long)clampi(p.buckets[d], 0, p.nbuckets - 1) * p.H + h] * LOG2E;
            });
        } else {
            c = far;
            finish([](int) { return 0.f; });
        }
        if (kk + 32 > n) {
            cold_path();
            const int left = n - (kk + 8 * hi);
#pragma unroll
            for (int r = 0; r < 16; ++r) t[r] = reg_off(r) < left ? t[r] : -__builtin_inff();
        }
        // probabilities against the reference point m; a sum past 2^60 (the first block's overflows) takes the block's maximum and starts over
        bf16x8 pf[2];
        float la, lb;
        auto probs = [&]() __attribute__((always_inline)) {
            const float mo = m - c;
            float e[16];
#pragma unroll
            for (int r = 0; r < 16; ++r) e[r] = fast_exp2(t[r] - mo);
            pf[0] = pack8f(e);
            pf[1] = pack8f(e + 8);
            la = l0;
            lb = l1;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                la = add_bf16_pair(__builtin_bit_cast(u32x4, pf[0])[i], la);
                lb = add_bf16_pair(__builtin_bit_cast(u32x4, pf[1])[i], lb);
            }
        };
        probs();
        if (!wave_all(la + lb < L_MAX)) {
            cold_path();
            float mx = t[0];
#pragma unroll
            for (int r = 1; r < 16; ++r) mx = fmaxf(mx, t[r]);
            mx += c;
            const float mn = fmaxf(m, fmaxf(mx, lane32_other(mx))), al = fast_exp2(m - mn);
            l0 *= al;
            l1 *= al;
#pragma unroll
            for (int r = 0; r < 16; ++r) { o[0][r] *= al; o[1][r] *= al; }
            m = mn;
            probs();
        }
        l0 = la;
        l1 = lb;
#pragma unroll
        for (int s2 = 0; s2 < 2; ++s2)
#pragma unroll
            for (int db = 0; db < 2; ++db) o[db] = mfma32(vf[s2][db], pf[s2], o[db]);
        wave_sync();                                           // every lane's reads of this stage are done (tr_frags waited): it may be refilled
        if (blk + STAGES < b1) issue(blk + STAGES);
    };
    for (int blk = b0; blk < b1; blk += 2) {
        step(Int<0>{}, blk);
        if (blk + 1 < b1) step(Int<1>{}, blk + 1);
    }
    // join the waves: their accumulators through LDS (the rings are drained), reference points and sums beside them
    float l = l0 + l1;
    l += lane32_other(l);
    __syncthreads();
    float* acc = (float*)smem;                                 // [wave][column][64]
    if (col) {
#pragma unroll
        for (int db = 0; db < 2; ++db)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[(wave * cols + l31) * DH + 32 * db + (r & 3) + 8 * (r >> 2) + 4 * hi] = o[db][r];
        if (hi == 0) { ml[wave][0][l31] = m; ml[wave][1][l31] = l; }
    }
    __syncthreads();
    for (int i = tid; i < (HEADS ? NW : 1) * cols * DH; i += NW * 64) {
        const int cc = i / DH % cols, d = i % DH, w0 = HEADS ? i / DH / cols : 0;
        const int hh = HEADS ? (hk - wave + w0) * p.G + cc : h0 + cc;
        float M = ml[w0][0][cc], L = 0.f, a = 0.f;
        if (!HEADS) {
#pragma unroll
            for (int w = 1; w < NW; ++w) M = fmaxf(M, ml[w][0][cc]);
        }
#pragma unroll
        for (int w = 0; w < (HEADS ? 1 : NW); ++w) {
            const float e = HEADS ? 1.f : fast_exp2(ml[w][0][cc] - M);
            L = fmaf(ml[w0 + w][1][cc], e, L);
            a = fmaf(acc[((w0 + w) * cols + cc) * DH + d], e, a);
        }
        if (p.splits == 1) {
            p.O[(long)b * p.ob + (long)hh * p.oh + d] = f2bf(L == 0.f ? 0.f : a / L);
        } else {
            float* q = p.ws + (((long)b * p.H + hh) * p.splits + split) * PART;
            q[d] = a;
            if (d == 0) { q[DH] = M; q[DH + 1] = L; }
        }
    }
}

// one workgroup per (sequence, query head): lane = output column, the waves take a quarter of the parts each
__global__ __launch_bounds__(256) void attn_decode_join_kernel(DecodeArgs p) {
    __shared__ float sm[4][DH], sl[4];
    const int lane = threadIdx.x & 63, wave = uniform_i(threadIdx.x >> 6);
    const long w = blockIdx.x;
    const float* q = p.ws + w * p.splits * PART;
    float M = M_INIT;
    for (int s = lane; s < p.splits; s += 64) M = fmaxf(M, q[(long)s * PART + DH]);
    M = wave_max(M);
    float L = 0.f, a = 0.f;
#pragma unroll 8
    for (int s = wave; s < p.splits; s += 4) {
        const float* r = q + (long)s * PART;
        const float e = fast_exp2(r[DH] - M);
        L = fmaf(r[DH + 1], e, L);
        a = fmaf(r[lane], e, a);
    }
    sm[wave][lane] = a;
    if (lane == 0) sl[wave] = L;
    __syncthreads();
    if (wave == 0) {
        a = (sm[0][lane] + sm[1][lane]) + (sm[2][lane] + sm[3][lane]);
        L = (sl[0] + sl[1]) + (sl[2] + sl[3]);
        p.O[(w / p.H) * p.ob + (w % p.H) * p.oh + lane] = f2bf(L == 0.f ? 0.f : a / L);
    }
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }
bool ok8(long s) { return s >= 0 && s % 8 == 0; }

// The four waves of a workgroup read four key heads' rows side by side where the heads come in fours (and a pass has all query heads of one)
bool by_heads(int Hkv, int G) { return Hkv % NW == 0 && G <= 32; }
// Parts of a sequence's keys: about 256 keys a wave (eight blocks: the start of a wave is a few blocks' time), fewer where that leaves the chip's
// 512 workgroup slots empty, never less than one block a wave; at most 128 (the join reads them all)
int splits_for(int B, int cap_n, int Hkv, int G) {
    const int run = by_heads(Hkv, G) ? 1 : NW;                      // waves that share a part
    const long wgs = (long)B * (by_heads(Hkv, G) ? Hkv / NW : (long)Hkv * ((G + 31) / 32));
    long s = (cap_n + 128 * run) / (256 * run);
    if (wgs * s < 512) s = (512 + wgs - 1) / wgs;
    const long most = (cap_n + run * 32 - 1) / (run * 32);
    if (s > most) s = most;
    if (s > 128) s = 128;
    return (int)(s < 1 ? 1 : s);
}

template <int BIAS, bool CAP> void run(const DecodeArgs& a, hipStream_t st) {
    if (by_heads(a.Hkv, a.G)) hipLaunchKernelGGL((attn_decode_kernel<BIAS, CAP, true>), dim3((unsigned)((long)a.B * a.splits * (a.Hkv / NW))), dim3(NW * 64), 0, st, a);
    else hipLaunchKernelGGL((attn_decode_kernel<BIAS, CAP, false>), dim3((unsigned)((long)a.B * a.splits * a.ngrp * a.Hkv)), dim3(NW * 64), 0, st, a);
}

int attn_decode_impl(const void* Q, int64_t qb, int64_t qh, const void* K, int64_t kb, int64_t kn, int64_t kh, const void* V, int64_t vb, int64_t vn,
                     int64_t vh, const int32_t* lens, int B, int capacity, int H, int Hkv, float scale, float softcap, const float* slopes,
                     const float* table, const int32_t* buckets, int nbuckets, int reach, void* O, int64_t ob, int64_t oh, float* ws, void* stream) {
    if (B < 0 || capacity < 0 || H < 1 || Hkv < 1 || H % Hkv != 0) return E2K_ERR_SHAPE;
    if (B == 0) return E2K_OK;
    if (!Q || !O || !lens || (capacity > 0 && (!K || !V))) return E2K_ERR_ARG;
    if (!score_range_ok(scale, softcap) || (slopes && table)) return E2K_ERR_ARG;
    if (table && (!buckets || nbuckets < 1 || reach < 0)) return E2K_ERR_SHAPE;
    if (!aligned16(Q) || !aligned16(K) || !aligned16(V) || !ok8(qb) || !ok8(qh) || !ok8(kb) || !ok8(kn) || !ok8(kh) || !ok8(vb) || !ok8(vn) || !ok8(vh))
        return E2K_ERR_ALIGN;
    if (kn >= (1 << 23) || vn >= (1 << 23)) return E2K_ERR_SHAPE;
    DecodeArgs a{};
    a.Q = (const bf16_t*)Q; a.K = (const bf16_t*)K; a.V = (const bf16_t*)V;
    a.qb = qb; a.qh = qh; a.kb = kb; a.kn = kn; a.kh = kh; a.vb = vb; a.vn = vn; a.vh = vh; a.ob = ob; a.oh = oh;
    a.lens = lens; a.B = B; a.cap_n = capacity; a.H = H; a.Hkv = Hkv; a.G = H / Hkv; a.ngrp = (a.G + 31) / 32;
    a.splits = splits_for(B, capacity, Hkv, a.G);
    a.scale = scale; a.cap = softcap; a.slopes = slopes; a.table = table; a.buckets = buckets; a.nbuckets = nbuckets; a.R = reach;
    a.O = (bf16_t*)O; a.ws = ws;
    if (a.splits > 1 && !ws) return E2K_ERR_ARG;
    if ((long)B * a.splits * a.ngrp * Hkv > 0x7fffffffL / (NW * 64) || (long)B * H > 0x7fffffffL / 256) return E2K_ERR_SHAPE;
    hipStream_t st = (hipStream_t)stream;
    const bool c = softcap > 0.f;
    if (table) { if (c) run<2, true>(a, st); else run<2, false>(a, st); }
    else if (slopes) { if (c) run<1, true>(a, st); else run<1, false>(a, st); }
    else { if (c) run<0, true>(a, st); else run<0, false>(a, st); }
    E2K_CHECK_LAUNCH();
    if (a.splits > 1) {
        hipLaunchKernelGGL(attn_decode_join_kernel, dim3((unsigned)((long)B * H)), dim3(256), 0, st, a);
        E2K_CHECK_LAUNCH();
    }
    return E2K_OK;
}

}  // namespace

extern "C" {

int64_t e2k_query_attn_decode_ws_floats(int B, int capacity, int H, int Hkv) {
    if (B < 1 || capacity < 0 || H < 1 || Hkv < 1 || H % Hkv != 0) return 0;
    const int s = splits_for(B, capacity, Hkv, H / Hkv);
    return s > 1 ? (int64_t)B * H * s * PART : 0;
}
int e2k_attn_decode(const void* Q, int64_t qb, int64_t qh, const void* K, int64_t kb, int64_t kn, int64_t kh, const void* V, int64_t vb, int64_t vn,
                    int64_t vh, const int32_t* lens, int B, int capacity, int H, int Hkv, float scale, float softcap, const float* slopes,
                    const float* table, const int32_t* buckets, int nbuckets, int reach, void* O, int64_t ob, int64_t oh, float* ws, void* stream) {
    return e2k::dispatch("attn_decode", attn_decode_impl, Q, qb, qh, K, kb, kn, kh, V, vb, vn, vh, lens, B, capacity, H, Hkv, scale, softcap, slopes,
                         table, buckets, nbuckets, reach, O, ob, oh, ws, stream);
}

}  // extern "C"
