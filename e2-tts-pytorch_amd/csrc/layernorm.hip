// Layer norm over rows, forward and backward, with one scale / shift pair for all rows or one per batch element (adaptive layer norm).
//
//   y = (x - m) r w + b,   m = mean(x),  r = 1 / sqrt(mean((x - m)^2) + eps),  w = gamma + gamma_off
//   g = dy w;  dx = r (g - mean(g) - xh mean(g xh)),  xh = (x - m) r;   dgamma = sum_rows dy xh,  dbeta = sum_rows dy
//
// What bounds it: HBM (x and y once; x, dy and dx once): 16399 x 1003 fp32 forward 23 us, backward 34 (5.7 TB/s both); 8448 x 1024 bf16 10 and 13 us.  A row stays in registers between its two reductions (mean first, then the
// centred squares: no cancellation however far the mean lies from 0); the next row of the wave is loaded while the current one is
// reduced.  64 lanes own a row up to 1536 columns, 256 lanes beyond (up to 8192).  Rows whose addresses or width are not multiples of
// 16 bytes take the same accesses unaligned, the last few columns one by one (element-wise rows reached 3.8 TB/s at 16399 x 1003 fp32).
// The sums over rows of the backward stay in registers over all rows of a wave, are joined in LDS in a fixed order, and leave as one
// partial row per workgroup; a second kernel adds the partials in a fixed order: no atomics, the same bits every time.
#include "e2k_device.h"
#include "plan.h"
#include <e2k_asm.h>
#include "../../include/e2k.h"

using namespace e2k;

namespace {

constexpr int LN_MAX = 8192;            // widest row (256 lanes x 32 elements)
constexpr int LN_WAVES = 8;             // waves per workgroup of the backward
constexpr int LN_ROW64 = 1536;          // widest row of 64 lanes: 24 elements a lane (32 of them and the backward's sums do not fit a wave's registers)

struct LNArgs {
    const void* x; long ldx;
    const float *gamma, *beta; long ldg; float gamma_off;
    void* y;                            // forward: y; backward: dx
    float *mean, *rstd;
    const void* dy;
    float* ws;                          // backward: [workgroup][2][D]
    int M, D, rpb, nb; float eps;
    int gpb;                            // backward: workgroups per batch element
};

// vectors at any element's alignment (gfx950 loads and stores 16 bytes at any address; the type keeps the compiler from assuming more)
typedef u32x4 u32x4_u __attribute__((aligned(2)));
typedef f32x4 f32x4_u __attribute__((aligned(4)));

// E elements of a row per lane: chunk c holds columns (c LPR + t) VEC .. + VEC - 1 of the row; columns past the end read 0.
// AL: rows start on 16 bytes and are whole vectors
template <class T, int NCH, int LPR, bool AL> struct Row {
    static constexpr int VEC = 16 / (int)sizeof(T), E = VEC * NCH;
    u32x4 w[NCH];

    __device__ __forceinline__ void load(const T* row, int t, int D) {
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
            const int col = (c * LPR + t) * VEC;
            u32x4 v = {0u, 0u, 0u, 0u};
            if (AL) {
                if (col < D) v = ld<u32x4>(row + col);
            } else if (col + VEC <= D) {
                v = *(const u32x4_u*)(row + col);
            } else {
#pragma unroll
                for (int i = 0; i < VEC; ++i)
                    if (col + i < D) {
                        if (sizeof(T) == 2) v[i >> 1] |= (unsigned)*(const bf16_t*)(row + col + i) << (16 * (i & 1));
                        else v[i] = *(const unsigned*)(row + col + i);
                    }
            }
            w[c] = v;
        }
    }
    __device__ __forceinline__ float get(int e) const {
        if (sizeof(T) == 4) return __uint_as_float(w[e >> 2][e & 3]);
        return (e & 1) ? bfhi(w[e >> 3][(e & 7) >> 1]) : bflo(w[e >> 3][(e & 7) >> 1]);
    }
};
template <class T, int NCH, int LPR, bool AL>
__device__ __forceinline__ void store_elems(T* row, int t, int D, const float (&v)[16 / (int)sizeof(T) * NCH]) {
    constexpr int VEC = 16 / (int)sizeof(T);
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
        const int col = (c * LPR + t) * VEC;
        if (col >= D) continue;
        u32x4 q;
        if (sizeof(T) == 2) q = pack8(&v[VEC * c]);
        else q = __builtin_bit_cast(u32x4, f32x4{v[4 * c], v[4 * c + 1], v[4 * c + 2], v[4 * c + 3]});
        if (AL) {
            st<u32x4>(row + col, q);
        } else if (col + VEC <= D) {
            *(u32x4_u*)(row + col) = q;
        } else {
#pragma unroll
            for (int i = 0; i < VEC; ++i)
                if (col + i < D) {
                    if (sizeof(T) == 2) *(bf16_t*)(row + col + i) = (bf16_t)(q[i >> 1] >> (16 * (i & 1)));
                    else *(unsigned*)(row + col + i) = q[i];
                }
        }
    }
}
// per-column fp32 vector (gamma / beta); `none` where there is none
template <int VEC, int NCH, int LPR, bool AL>
__device__ __forceinline__ void load_cols(const float* p, float off, float none, int t, int D, float (&v)[VEC * NCH]) {
#pragma unroll
    for (int e = 0; e < VEC * NCH; ++e) v[e] = none;
    if (!p) return;
#pragma unroll
    for (int c = 0; c < NCH; ++c)
#pragma unroll
        for (int i = 0; i < VEC; i += 4) {
            const int col = (c * LPR + t) * VEC + i;
            f32x4 w = {0.f, 0.f, 0.f, 0.f};
            if (AL) {
                if (col < D) w = ld<f32x4>(p + col);
            } else if (col + 4 <= D) {
                w = *(const f32x4_u*)(p + col);
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (col + j < D) w[j] = p[col + j];
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) v[c * VEC + i + j] = w[j] + off;
        }
}

// sums over the LPR lanes of a row; with 256 lanes every wave of the workgroup takes part (buf: 2 floats per wave, double-buffered by `ph`)
template <int LPR> __device__ __forceinline__ void row_sum2(float& a, float& b, float* buf, int wave, int ph) {
    a = wave_sum_fast(a);
    b = wave_sum_fast(b);
    if (LPR > 64) {
        float* q = buf + ph * 2 * LN_WAVES;
        if ((threadIdx.x & 63) == 0) { q[2 * wave] = a; q[2 * wave + 1] = b; }
        __syncthreads();
        const int w0 = wave & ~3;
        a = (q[2 * w0] + q[2 * w0 + 2]) + (q[2 * w0 + 4] + q[2 * w0 + 6]);
        b = (q[2 * w0 + 1] + q[2 * w0 + 3]) + (q[2 * w0 + 5] + q[2 * w0 + 7]);
    }
}

// A workgroup of four waves; a row slot (wave, or the whole workgroup) takes rows slot, slot + nslots, ... of its contiguous share.
template <class T, int NCH, int LPR, bool AL>
__global__ __launch_bounds__(256) void ln_fwd_kernel(LNArgs p, int share) {
    constexpr int VEC = 16 / (int)sizeof(T), E = VEC * NCH, RPW = 256 / LPR;
    __shared__ float buf[4 * LN_WAVES];
    const int wave = uniform_i(threadIdx.x >> 6), t = threadIdx.x & (LPR - 1), slot = LPR == 64 ? wave : 0;
    const long r0 = (long)blockIdx.x * share * RPW + slot;
    float w[E], b[E];
    int cur = -1;
    Row<T, NCH, LPR, AL> nx;
    if (r0 < p.M) nx.load((const T*)p.x + r0 * p.ldx, t, p.D);
    const float inv = 1.f / (float)p.D;
    for (int s = 0; s < share; ++s) {
        const long r = r0 + (long)s * RPW;
        if (r >= p.M) break;           // (uniform over the lanes that meet in a reduction: a wave, or the workgroup that is one row slot)
        const Row<T, NCH, LPR, AL> x = nx;
        if (s + 1 < share && r + RPW < p.M) nx.load((const T*)p.x + (r + RPW) * p.ldx, t, p.D);
        const int bi = (int)((unsigned)r / (unsigned)p.rpb);
        if (bi != cur) {
            cur = bi;
            load_cols<VEC, NCH, LPR, AL>(p.gamma ? p.gamma + bi * p.ldg : nullptr, p.gamma_off, 1.f, t, p.D, w);
            load_cols<VEC, NCH, LPR, AL>(p.beta ? p.beta + bi * p.ldg : nullptr, 0.f, 0.f, t, p.D, b);
        }
        float m = 0.f, z = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) m += x.get(e);                // (columns past the end read 0)
        row_sum2<LPR>(m, z, buf, wave, 0);
        m *= inv;
        float v[E], q = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int col = ((e / VEC) * LPR + t) * VEC + e % VEC;
            v[e] = col < p.D ? x.get(e) - m : 0.f;
            q = fmaf(v[e], v[e], q);
        }
        z = 0.f;
        row_sum2<LPR>(q, z, buf, wave, 1);
        const float rs = 1.f / sqrtf(fmaf(q, inv, p.eps));
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = fmaf(v[e] * rs, w[e], b[e]);
        store_elems<T, NCH, LPR, AL>((T*)p.y + r * (long)p.D, t, p.D, v);
        if (t == 0 && p.mean) { p.mean[r] = m; p.rstd[r] = rs; }
    }
}

// Workgroup g of batch element b takes every gpb-th block of eight (two) rows of it; its column sums go to ws[b gpb + g].
template <class T, int NCH, int LPR, bool AL>
__global__ __launch_bounds__(64 * LN_WAVES) void ln_bwd_kernel(LNArgs p) {
    constexpr int VEC = 16 / (int)sizeof(T), E = VEC * NCH, SLOTS = LN_WAVES * 64 / LPR;
    __shared__ float sm[(SLOTS / 2) * 2 * E * LPR];             // [slot][dgamma | dbeta][element][lane]: at most 64 KB
    __shared__ float buf[4 * LN_WAVES];
    const int wave = uniform_i(threadIdx.x >> 6), t = threadIdx.x & (LPR - 1), slot = LPR == 64 ? wave : wave >> 2;
    const int bi = blockIdx.x / p.gpb, g = blockIdx.x % p.gpb;
    const long first = (long)bi * p.rpb, last = first + p.rpb < p.M ? first + p.rpb : p.M;
    float w[E], sg[E], sb[E];
    load_cols<VEC, NCH, LPR, AL>(p.gamma ? p.gamma + bi * p.ldg : nullptr, p.gamma_off, 1.f, t, p.D, w);
#pragma unroll
    for (int e = 0; e < E; ++e) { sg[e] = 0.f; sb[e] = 0.f; }
    const float inv = 1.f / (float)p.D;
    const long step = (long)p.gpb * SLOTS;
    long r = first + (long)g * SLOTS + slot;
    Row<T, NCH, LPR, AL> nx, nd;
    float nm = 0.f, nr = 0.f;
    auto fetch = [&](long row) __attribute__((always_inline)) {
        nx.load((const T*)p.x + row * p.ldx, t, p.D);
        nd.load((const T*)p.dy + row * (long)p.D, t, p.D);
        nm = p.mean[row];
        nr = p.rstd[row];
    };
    if (r < last) fetch(r);
    // (the loop count is the same for every slot of the workgroup: with 256 lanes a row the reductions meet at a barrier)
    for (long base = first + (long)g * SLOTS; base < last; base += step, r += step) {
        const bool in = r < last;
        if (LPR == 64 && !in) break;
        const Row<T, NCH, LPR, AL> x = nx, d = nd;
        const float m = nm, rs = in ? nr : 0.f;
        if (r + step < last) fetch(r + step);
        float xh[E], gy[E], c1 = 0.f, c2 = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const float dy = in ? d.get(e) : 0.f;
            xh[e] = in ? (x.get(e) - m) * rs : 0.f;
            gy[e] = dy * w[e];                       // (columns past the end: dy = 0)
            c1 += gy[e];
            c2 = fmaf(gy[e], xh[e], c2);
            sb[e] += dy;
            sg[e] = fmaf(dy, xh[e], sg[e]);
        }
        row_sum2<LPR>(c1, c2, buf, wave, (int)(((base - first) / step) & 1));
        c1 *= inv;
        c2 *= inv;
        if (in) {
            float v[E];
#pragma unroll
            for (int e = 0; e < E; ++e) v[e] = rs * (gy[e] - c1 - xh[e] * c2);
            store_elems<T, NCH, LPR, AL>((T*)p.y + r * (long)p.D, t, p.D, v);
        }
    }
    if (!p.ws) return;
    // join: the upper half of the row slots hands its sums to the lower half until one is left
#pragma unroll
    for (int half = SLOTS / 2; half >= 1; half >>= 1) {
        __syncthreads();
        if (slot >= half && slot < 2 * half) {
            float* q = sm + (long)(slot - half) * 2 * E * LPR;
#pragma unroll
            for (int e = 0; e < E; ++e) { q[e * LPR + t] = sg[e]; q[(E + e) * LPR + t] = sb[e]; }
        }
        __syncthreads();
        if (slot < half) {
            const float* q = sm + (long)slot * 2 * E * LPR;
#pragma unroll
            for (int e = 0; e < E; ++e) { sg[e] += q[e * LPR + t]; sb[e] += q[(E + e) * LPR + t]; }
        }
    }
    if (slot == 0) {
        float* out = p.ws + (long)blockIdx.x * 2 * p.D;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int col = ((e / VEC) * LPR + t) * VEC + e % VEC;
            if (col < p.D) { out[col] = sg[e]; out[p.D + col] = sb[e]; }
        }
    }
}

// columns c of [dgamma | dbeta] of batch element blockIdx.y: sum over its workgroups' partials; 64 columns x 16 row groups per workgroup
__global__ __launch_bounds__(1024) void ln_bwd_reduce_kernel(const float* ws, int D, int gpb, float* dgamma, float* dbeta, long ldg, int accumulate) {
    __shared__ float sm[16][64];
    const int lane = threadIdx.x & 63, grp = threadIdx.x >> 6;
    const int c = blockIdx.x * 64 + lane, bi = blockIdx.y;
    float a = 0.f;
    if (c < 2 * D) {
        const float* q = ws + (long)bi * gpb * 2 * D + c;
#pragma unroll 8
        for (int g = grp; g < gpb; g += 16) a += q[(long)g * 2 * D];
    }
    sm[grp][lane] = a;
    __syncthreads();
    if (grp == 0 && c < 2 * D) {
        a = 0.f;
#pragma unroll
        for (int g = 0; g < 16; ++g) a += sm[g][lane];
        float* out = c < D ? dgamma : dbeta;
        if (!out) return;
        out += bi * ldg + (c < D ? c : c - D);
        *out = accumulate ? *out + a : a;
    }
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

// rows per slot of the forward: enough workgroups to fill the chip several times over, then longer shares (gamma and beta are read once a share)
int fwd_share(int M, int rpw) {
    const long wgs = 256 * 8;
    long s = (M + wgs * rpw - 1) / (wgs * rpw);
    return (int)(s < 1 ? 1 : s > 16 ? 16 : s);
}

template <class T, int NCH, int LPR, bool AL> int launch_fwd(const LNArgs& a, hipStream_t st) {
    constexpr int RPW = 256 / LPR;
    const int share = fwd_share(a.M, RPW);
    const long per = (long)share * RPW;
    hipLaunchKernelGGL((ln_fwd_kernel<T, NCH, LPR, AL>), dim3((unsigned)((a.M + per - 1) / per)), dim3(256), 0, st, a, share);
    E2K_CHECK_LAUNCH();
    return E2K_OK;
}
template <class T, int NCH, int LPR, bool AL> int launch_bwd(const LNArgs& a, hipStream_t st) {
    hipLaunchKernelGGL((ln_bwd_kernel<T, NCH, LPR, AL>), dim3(a.nb * a.gpb), dim3(64 * LN_WAVES), 0, st, a);
    E2K_CHECK_LAUNCH();
    return E2K_OK;
}

// widths per instantiation: columns a row's lanes cover
#define LN_PICK(FN, T, AL)                                                                        \
    do {                                                                                          \
        constexpr int V_ = 16 / (int)sizeof(T);                                                   \
        const int per = (a.D + V_ - 1) / V_;                                                      \
        if (a.D <= LN_ROW64) {                                                                    \
            const int ch = (per + 63) / 64;                                                       \
            if (ch <= 8 / V_) return FN<T, 8 / V_, 64, AL>(a, st);                                \
            if (ch <= 16 / V_) return FN<T, 16 / V_, 64, AL>(a, st);                              \
            return FN<T, 24 / V_, 64, AL>(a, st);                                                 \
        }                                                                                         \
        const int ch = (per + 255) / 256;                                                         \
        if (ch <= 8 / V_) return FN<T, 8 / V_, 256, AL>(a, st);                                   \
        if (ch <= 16 / V_) return FN<T, 16 / V_, 256, AL>(a, st);                                 \
        return FN<T, 32 / V_, 256, AL>(a, st);                                                    \
    } while (0)

// workgroups per batch element of the backward: at most one (eight waves) per CU over all batch elements -- a 257th workgroup would share a CU and
// finish at half the speed of the others (16399 rows of 1003: 34 us with 256, 44 with 257)
int bwd_gpb(int M, int D, int rpb) {
    const int nb = (M + rpb - 1) / rpb, slots = D <= LN_ROW64 ? LN_WAVES : LN_WAVES / 4;
    const int most = (rpb + slots - 1) / slots;
    int g = 256 / nb;
    if (g > most) g = most;
    return g < 1 ? 1 : g;
}

int check(const void* x, int64_t ldx, int dtype, int64_t ldg, int rows_per_batch, int M, int D, const float* gamma, const float* beta) {
    if (dtype != 0 && dtype != 1) return E2K_ERR_ARG;
    if (M < 0 || D < 1 || D > LN_MAX || rows_per_batch < 1 || ldx < D) return E2K_ERR_SHAPE;
    if (M > 0 && !x) return E2K_ERR_ARG;
    if ((gamma || beta) && ldg < D && M > rows_per_batch) return E2K_ERR_SHAPE;
    return E2K_OK;
}

int layernorm_fwd_impl(const void* x, int64_t ldx, int dtype, const float* gamma, const float* beta, int64_t ldg, float gamma_off, int rows_per_batch,
                       float eps, void* y, float* mean, float* rstd, int M, int D, void* stream) {
    const int rc = check(x, ldx, dtype, ldg, rows_per_batch, M, D, gamma, beta);
    if (rc) return rc;
    if (M == 0) return E2K_OK;
    if (!y || (!mean) != (!rstd)) return E2K_ERR_ARG;
    LNArgs a{};
    a.x = x; a.ldx = ldx; a.gamma = gamma; a.beta = beta; a.ldg = ldg; a.gamma_off = gamma_off; a.y = y; a.mean = mean; a.rstd = rstd;
    a.M = M; a.D = D; a.rpb = rows_per_batch; a.nb = (M + rows_per_batch - 1) / rows_per_batch; a.eps = eps;
    hipStream_t st = (hipStream_t)stream;
    const int vec = dtype == 0 ? 8 : 4;
    const bool cols = aligned16(gamma) && aligned16(beta) && (ldg % 4 == 0 || M <= rows_per_batch);
    const bool wide = cols && D % vec == 0 && ldx % vec == 0 && aligned16(x) && aligned16(y);
    if (dtype == 0) {
        if (wide) LN_PICK(launch_fwd, bf16_t, true);
        LN_PICK(launch_fwd, bf16_t, false);
    }
    if (wide) LN_PICK(launch_fwd, float, true);
    LN_PICK(launch_fwd, float, false);
}

int layernorm_bwd_impl(const void* dy, const void* x, int64_t ldx, int dtype, const float* mean, const float* rstd, const float* gamma, int64_t ldg,
                       float gamma_off, int rows_per_batch, void* dx, float* dgamma, float* dbeta, int64_t ldd, int accumulate, float* ws, int M, int D,
                       void* stream) {
    const int rc = check(x, ldx, dtype, ldg, rows_per_batch, M, D, gamma, nullptr);
    if (rc) return rc;
    if (M == 0) return E2K_OK;
    if (!dy || !mean || !rstd || !dx || ((dgamma || dbeta) && !ws)) return E2K_ERR_ARG;
    if ((dgamma || dbeta) && ldd < D && M > rows_per_batch) return E2K_ERR_SHAPE;
    LNArgs a{};
    a.x = x; a.ldx = ldx; a.gamma = gamma; a.ldg = ldg; a.gamma_off = gamma_off; a.y = dx; a.mean = (float*)mean; a.rstd = (float*)rstd; a.dy = dy;
    a.ws = (dgamma || dbeta) ? ws : nullptr;
    a.M = M; a.D = D; a.rpb = rows_per_batch; a.nb = (M + rows_per_batch - 1) / rows_per_batch; a.gpb = bwd_gpb(M, D, rows_per_batch);
    hipStream_t st = (hipStream_t)stream;
    const int vec = dtype == 0 ? 8 : 4;
    const bool cols = aligned16(gamma) && (ldg % 4 == 0 || M <= rows_per_batch);
    const bool wide = cols && D % vec == 0 && ldx % vec == 0 && aligned16(x) && aligned16(dy) && aligned16(dx);
    const int rl = [&]() -> int {
        if (dtype == 0) {
            if (wide) LN_PICK(launch_bwd, bf16_t, true);
            LN_PICK(launch_bwd, bf16_t, false);
        }
        if (wide) LN_PICK(launch_bwd, float, true);
        LN_PICK(launch_bwd, float, false);
    }();
    if (rl || !a.ws) return rl;
    hipLaunchKernelGGL(ln_bwd_reduce_kernel, dim3((2 * D + 63) / 64, a.nb), dim3(1024), 0, st, ws, D, a.gpb, dgamma, dbeta, (long)ldd, accumulate);
    E2K_CHECK_LAUNCH();
    return E2K_OK;
}

}  // namespace

extern "C" {

int e2k_layernorm_fwd(const void* x, int64_t ldx, int dtype, const float* gamma, const float* beta, int64_t ldg, float gamma_off, int rows_per_batch,
                      float eps, void* y, float* mean, float* rstd, int M, int D, void* stream) {
    return e2k::dispatch("layernorm_fwd", layernorm_fwd_impl, x, ldx, dtype, gamma, beta, ldg, gamma_off, rows_per_batch, eps, y, mean, rstd, M, D, stream);
}
int64_t e2k_query_layernorm_bwd_ws_floats(int M, int D, int rows_per_batch) {
    if (M < 1 || D < 1 || D > LN_MAX || rows_per_batch < 1) return 0;
    return (int64_t)((M + rows_per_batch - 1) / rows_per_batch) * bwd_gpb(M, D, rows_per_batch) * 2 * D;
}
int e2k_layernorm_bwd(const void* dy, const void* x, int64_t ldx, int dtype, const float* mean, const float* rstd, const float* gamma, int64_t ldg,
                      float gamma_off, int rows_per_batch, void* dx, float* dgamma, float* dbeta, int64_t ldd, int accumulate, float* ws, int M, int D,
                      void* stream) {
    return e2k::dispatch("layernorm_bwd", layernorm_bwd_impl, dy, x, ldx, dtype, mean, rstd, gamma, ldg, gamma_off, rows_per_batch, dx, dgamma, dbeta, ldd,
                         accumulate, ws, M, D, stream);
}

}  // extern "C"
