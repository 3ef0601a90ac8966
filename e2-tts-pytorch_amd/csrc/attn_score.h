// Score arithmetic and register layout shared by packed_attn.hip and attn_decode.hip (dim_head 64, log2 domain, 16 scores of a 32 x 32 block in a
// lane).  Internal to those files (anonymous namespace on purpose).
#pragma once
#include "attn_tile32.h"

namespace {

using namespace e2k;

constexpr int DH = 64;
constexpr float LOG2E = 1.4426950408889634f;
constexpr float M_INIT = -1e30f;      // running maximum before any visible key
constexpr float L_MAX = 0x1p60f;      // largest sum of a row (per half-wave) before the accumulators are rescaled

template <int N> struct Int { static constexpr int value = N; };
__device__ __forceinline__ int clampi(int x, int lo, int hi) { return x < lo ? lo : x > hi ? hi : x; }
__device__ __forceinline__ constexpr int reg_off(int r) { return 16 * (r >> 3) + (r & 7); }      // row of accumulator r within its block (+ 8 hi)

// tanh cap:  out tanh(s kx)  with out = cap log2(e).  |s kx| <= 0.3 (a wave vote): minimax of tanh(x) / x in x^2, relative error 1e-8 with four terms
// (FINE: where fp32 results depend on it), 1.2e-6 with three (where probabilities are rounded to bf16: their half step is 4e-3, and the cubed error of
// a score is below 3e-5 at any cap up to 50); beyond: 1 - 2 / (2^(2 x log2 e) + 1), absolute error 2^-22
constexpr float CAP_POLY_MAX = 0.3f;
struct Cap { float a0, a1, a2, a3, k2, out, lim; };
// what the kernels' fp32 arithmetic takes: scale / cap and its products with scores stay finite or saturate
inline bool score_range_ok(float scale, float cap) { return scale > 0.f && scale < 1e30f && (cap == 0.f || (cap >= 1e-30f && cap < 1e30f && scale / cap < 1e30f)); }
template <bool FINE> __device__ __forceinline__ Cap cap_of(float scale, float cap) {
    Cap c;
    const float kx = scale / cap, k2 = kx * kx;
    c.out = cap * LOG2E;
    const float k1 = c.out * kx;
    c.a0 = FINE ? k1 : k1 * 0.99999887f;
    c.a1 = k1 * k2 * (FINE ? -0.33332962f : -0.33310023f);
    c.a2 = k1 * k2 * k2 * (FINE ? 0.13312598f : 0.12633947f);
    c.a3 = FINE ? k1 * k2 * k2 * k2 * -0.050222438f : 0.f;
    c.k2 = 2.f * LOG2E * kx;
    c.lim = k1 * k2 * k2 * k2 < 1e37f ? CAP_POLY_MAX / kx : -1.f;      // (a cap of next to nothing: coefficients that overflow make 0 times infinity of a score of 0)
    return c;
}
// x[r] = capped z[r] + add(r), and with KEEP z[r] capped in place (the backward's 1 - tanh^2)
template <bool FINE, bool KEEP, class A> __device__ __forceinline__ void cap16(f32x16& z, float (&x)[16], const Cap& cp, A&& add) {
    float a = 0.f;
#pragma unroll
    for (int r = 0; r < 16; r += 2) a = fmaxf(fmaxf(fabsf(z[r]), fabsf(z[r + 1])), a);
    if (wave_all(a <= cp.lim)) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const float w = z[r] * z[r];
            const float u = fmaf(FINE ? fmaf(fmaf(w, cp.a3, cp.a2), w, cp.a1) : fmaf(w, cp.a2, cp.a1), w, cp.a0);
            if (KEEP) {
                z[r] *= u;
                x[r] = z[r] + add(r);
            } else {
                x[r] = fmaf(z[r], u, add(r));
            }
        }
    } else {
        cold_path();
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const float c = fmaf(-2.f * cp.out, fast_rcp(fast_exp2(z[r] * cp.k2) + 1.f), cp.out);
            if (KEEP) z[r] = c;
            x[r] = c + add(r);
        }
    }
}

// transposed fragments of a block of 32 tile rows OFF bytes behind the tile image that the addresses were made for:
// f[s2][db] = columns 32 db + l31, rows 16 s2 + 8 hi .. + 7
struct TrAddr { unsigned lo[2], hi_[2]; };
__device__ __forceinline__ TrAddr tr_addr(const unsigned char* tile, int lane) {
    const TrOff t = tr_offsets(lane);
    return TrAddr{{lds_addr(tile + t.lo[0]), lds_addr(tile + t.lo[1])}, {lds_addr(tile + t.hi_[0]), lds_addr(tile + t.hi_[1])}};
}
template <int OFF> __device__ __forceinline__ void tr_frags(bf16x8 (&f)[2][2], const TrAddr& t) {
    s16x4_ d[8];
    lds_tr_read8<OFF, 2048>(d, t.lo[0], t.hi_[0], t.lo[1], t.hi_[1]);
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i >> 1][i & 1] = __builtin_shufflevector(d[2 * i], d[2 * i + 1], 0, 1, 2, 3, 4, 5, 6, 7);
}

// addresses of a lane's row fragments (frag_offsets) in the tile image at `tile`
__device__ __forceinline__ void frag_addr(const unsigned char* tile, int l31, int hi, unsigned (&a)[4]) {
    int off[4];
    frag_offsets(l31, hi, off);
#pragma unroll
    for (int j = 0; j < 4; ++j) a[j] = lds_addr(tile + off[j]);
}

__device__ __forceinline__ f32x16 zero16() {
    f32x16 z;
#pragma unroll
    for (int r = 0; r < 16; ++r) z[r] = 0.f;
    return z;
}

}  // namespace
