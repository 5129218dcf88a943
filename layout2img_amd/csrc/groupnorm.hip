// Group normalisation with an activation on channels-last maps, forward and backward.
//
//   per image b and group g of C / G consecutive channels, over its n = HW * C / G values:
//     mean, var = biased moments;  xh = (x - mean) * rstd, rstd = 1 / sqrt(var + eps);  z = gamma_c xh + beta_c;  y = act(z)
//   backward, dz = dy act'(z):
//     dbeta_c = sum dz;  dgamma_c = sum dz xh;  dx = rstd (gamma dz - (S1 + xh S2) / n),  S1 = sum gamma dz, S2 = sum gamma dz xh over the group
//
// Bound by bytes. Two forms:
//   resident: a workgroup holds all pixels of a slab of whole groups (at least 64 contiguous bytes a pixel) in registers: one launch, every
//     value read once; used where a slab is at most 4096 values (8192 in bf16: maps up to 16 x 16 of the wide layers). A group's mean is summed around
//     its first value, the squared deviations around the mean.
//   split: the map is cut in NCH chunks of rows (pixels) per image. The first launch leaves every chunk's moments (mean and sum of squared
//     deviations per group, counted from origins that follow the values: neither a mean far from zero nor single values far from the rest cost digits), the
//     second joins them in a fixed order and writes the result, reading the map a second time -- from the chunk that was read last backwards, on the
//     XCD that read it, so that L2 and the Infinity Cache still hold what is read first.
// Measured, B = 32 with silu: 64 x 64 x 128 in bf16 (33.5 MB a map): moments 8.6 us, result 17 (4.0 TB/s), backward sums 19, dx 21 (4.8 TB/s);
// 128 x 128 x 64 in f32 (134 MB): 25, 43 (6.3 TB/s), 51 (5.2), 66 (6.1) -- what a copy of that size reaches. One 4 x 4 x 1024 image, resident: 6 us.
// In the backward pass the sums are S1, S2 per group and rows of (sum dz xh | sum dz) per channel, which the ordered fold adds into dgamma / dbeta (in
// workgroups of their own at the end of the second launch). Statistics are f32; nothing is accumulated by atomics.
#include "vec.h"

struct GnArgs {
    const void* x; const float* gamma; const float* beta; void* y;
    float* mean; float* rstd;             // [B][G]
    const void* dy; void* dx;
    float* part;                          // split: [B][NCH][G] (mean, M2), backward (S1, S2)
    float* cpart;                         // backward: [B][NCH][2 Cp] rows of (sum dz xh | sum dz)
    long long HW; long long rows;         // rows per chunk
    int B, C, Cp, G, cg, nch, act;
    int Cs, slabs, tw, nr;                // resident: channels of a slab, slabs per image, threads along the channels and along the rows
    float eps;
};

// With d = x - mean and A = rstd gamma: z = A d + beta, and every kernel sees a value through d, so that its channel costs three registers.
// silu: s = 1 / (1 + 2^(-z log2 e)) by the hardware's exp2 and reciprocal, silu' = s + z (s - s^2). s is off by about (|z| + 6) 2^-24 of itself: |z| 2^-24 as the
// exponent's argument is rounded to 24 bits, which weighs in where s is small (z far below 0), and a step of each of the others.
#define GN_LOG2E 1.44269504088896340736f
__device__ __forceinline__ float gn_sig(float z) { return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(z * -GN_LOG2E)); }
// A z that is not a number stays one in every activation (not fmaxf: a group with such a value is not a number as a whole and must not come out as zeros).
template <int ACT> __device__ __forceinline__ float gn_act(float z) {
    if (ACT == 1) return z < 0.f ? 0.f : z;
    if (ACT == 2) return z * gn_sig(z);
    return z;
}
template <int ACT> __device__ __forceinline__ float gn_dact(float z, float dy) {
    if (ACT == 1) return z <= 0.f ? 0.f : dy;
    if (ACT == 2) { const float s = gn_sig(z); return dy * fmaf(z, fmaf(-s, s, s), s); }
    return dy;
}

// f(e, channel c + e, its group): one division for the V channels of a thread
template <int V, typename F> __device__ __forceinline__ void gn_each(int c, int cg, F f) {
    int g = c / cg, rem = c - g * cg;
#pragma unroll
    for (int e = 0; e < V; ++e) {
        f(e, c + e, g);
        if (++rem == cg) { rem = 0; ++g; }
    }
}

// ------------------------------------------------------------------------------------------------ split form
// A workgroup covers all C channels of its rows in tiles of tw = min(C / V, 256) vectors; tw threads stand along the channels, 256 / tw along
// the rows. REV: the chunks from the last to the first, each on the XCD (workgroup number modulo 8) that the other order gives it.
#define GN_COLS(V, REV)                                                                                              \
    const int cv = p.C / (V), tw = cv < 256 ? cv : 256, nr = 256 / tw, tx = (int)threadIdx.x % tw, ty = (int)threadIdx.x / tw; \
    int id = blockIdx.x;                                                                                             \
    const int total8 = p.B * p.nch & ~7;                                                                             \
    if ((REV) && id < total8) id = total8 - 8 - (id & ~7) + (id & 7);                                                \
    const int b = id / p.nch, ch = id - b * p.nch;                                                                   \
    const long long r0 = ch * p.rows, r1 = r0 + p.rows < p.HW ? r0 + p.rows : p.HW;                                   \
    const size_t img = (size_t)b * p.HW * p.C;
// rows r0 + ty, + nr, ... of the chunk: LOAD(k, r) puts row r into slot k, four rows in flight, then USE(k, r); FOUR in front of every four
#define GN_ROWS_4(LOAD, FOUR, USE)                                                                                    \
    do {                                                                                                             \
        long long r = r0 + ty;                                                                                       \
        for (; r + 3 * nr < r1; r += 4 * nr) {                                                                       \
            LOAD(0, r) LOAD(1, r + nr) LOAD(2, r + 2 * nr) LOAD(3, r + 3 * nr)                                       \
            FOUR                                                                                                     \
            USE(0, r) USE(1, r + nr) USE(2, r + 2 * nr) USE(3, r + 3 * nr)                                           \
        }                                                                                                            \
        for (; r < r1; r += nr) { LOAD(0, r) USE(0, r) }                                                             \
    } while (0)
#define GN_ROWS(LOAD, USE) GN_ROWS_4(LOAD, , USE)

// Sums around an origin lose the digits of the deviations where the origin lies far from the mean: q - s^2 / n cancels. Every thread therefore moves its
// origin k, at first its first row, to the mean of its rows so far at 4, 16, 64, ... of them. At the end q <= 7 (q - s^2 / N), whatever the values and their
// order: behind the last of the n rows that k is the mean of come at most 6 n, and N (mean - k)^2 is at most (N - n) / n times the deviations that part them
// from the first n. The moments of threads, channels and chunks are joined around one of their means, the squared deviations around the joint one.
// 32 images of 64 x 64 x 128 bf16: 7.4 us, without moving 7.0.
template <int V> __device__ __forceinline__ void gn_recentre(float n, float (&k)[V], float (&s)[V], float (&q)[V]) {
    const float rn = __builtin_amdgcn_rcpf(n);   // (k need not be the mean exactly)
#pragma unroll
    for (int e = 0; e < V; ++e) {
        const float k1 = fmaf(s[e], rn, k[e]), d = k1 - k[e];   // (d: what k really moves by)
        q[e] -= d * (2.f * s[e] - n * d);
        s[e] -= n * d;
        k[e] = k1;
    }
}

template <typename T, int V>
__global__ __launch_bounds__(256) void gn_stats_kernel(GnArgs p) {
    extern __shared__ __attribute__((aligned(16))) float sm[];   // [C] means, [C] squared deviations, [V][2][256] row lanes
    float *cm = sm, *cq = sm + p.Cp, *red = cq + p.Cp;
    GN_COLS(V, false)
    const T* x = reinterpret_cast<const T*>(p.x) + img;
    const int rows = (int)(r1 - r0);
    const float n = (float)rows, rn = 1.f / n;
    for (int t0 = 0; t0 < cv; t0 += tw) {
        const int c = (t0 + tx) * V;
        const bool on = ty < nr && ty < rows && t0 + tx < cv;
        float s[V], q[V], k[V];
#pragma unroll
        for (int e = 0; e < V; ++e) { s[e] = 0.f; q[e] = 0.f; k[e] = 0.f; }
        if (on) {
            Vec<T, V> a[4];
            a[0].load(x + (size_t)(r0 + ty) * p.C + c);
            a[0].get(k);
            int seen = 0, next = 4;
#define GN_L(K, R) a[K].load(x + (size_t)(R) * p.C + c);
#define GN_U(K, R) { float v[V]; a[K].get(v); _Pragma("unroll") for (int e = 0; e < V; ++e) { const float d = v[e] - k[e]; s[e] += d; q[e] = fmaf(d, d, q[e]); } }
#define GN_FOUR if (seen == next) { gn_recentre<V>((float)seen, k, s, q); next *= 4; } seen += 4;
            GN_ROWS_4(GN_L, GN_FOUR, GN_U);
#undef GN_FOUR
#undef GN_U
            const float rl = 1.f / (float)((rows - ty + nr - 1) / nr);
#pragma unroll
            for (int e = 0; e < V; ++e) { const float m = s[e] * rl; q[e] -= s[e] * m; k[e] += m; }
        }
        __syncthreads();
#pragma unroll
        for (int e = 0; e < V; ++e) { red[e * 512 + threadIdx.x] = k[e]; red[e * 512 + 256 + threadIdx.x] = q[e]; }
        __syncthreads();
        // a channel's row lanes: lane j has the rows j, j + nr, ...; P threads of a wave a channel
        const int lanes = rows < nr ? rows : nr, full = rows / nr, more = rows - full * nr;   // the first `more` lanes have full + 1 rows
        int P = 1;
        while (P < 64 && 2 * P * tw * V <= 256) P <<= 1;
        const int sub = (int)threadIdx.x & (P - 1);
        for (int i0 = 0; i0 < tw * V; i0 += 256 / P) {
            const int i = min(i0 + (int)threadIdx.x / P, tw * V - 1), e = i / tw, tt = i - e * tw;   // (threads behind the last channel do it once more)
            const float *ml = red + e * 512 + tt, *ql = ml + 256;
            const float o = ml[0];
            float m = 0.f, m2 = 0.f;
#pragma unroll 4
            for (int j = sub; j < lanes; j += P) m = fmaf((float)(j < more ? full + 1 : full), ml[j * tw] - o, m);
            for (int w = 1; w < P; w <<= 1) m += __shfl_xor(m, w, 64);
            m = fmaf(m, rn, o);
#pragma unroll 4
            for (int j = sub; j < lanes; j += P) { const float d = ml[j * tw] - m; m2 += fmaf((float)(j < more ? full + 1 : full) * d, d, ql[j * tw]); }
            for (int w = 1; w < P; w <<= 1) m2 += __shfl_xor(m2, w, 64);
            if (sub == 0 && t0 + tt < cv) { cm[(t0 + tt) * V + e] = m; cq[(t0 + tt) * V + e] = m2; }
        }
    }
    __syncthreads();
    for (int g = threadIdx.x; g < p.G; g += 256) {   // the group's channels, all over the same rows
        const float *m_ = cm + g * p.cg, *q_ = cq + g * p.cg, o = m_[0];
        float m = 0.f, m2 = 0.f;
        for (int c = 0; c < p.cg; ++c) m += m_[c] - o;
        m = o + m / (float)p.cg;
        for (int c = 0; c < p.cg; ++c) { const float d = m_[c] - m; m2 += fmaf(n * d, d, q_[c]); }
        *reinterpret_cast<float2*>(p.part + (((size_t)b * p.nch + ch) * p.G + g) * 2) = make_float2(m, m2);
    }
}

// L = 256 / (power of two >= G) lanes a group (at least one) walk the chunks; their sums meet in a butterfly of fixed order
#define GN_LANES                                                                                                     \
    int L = 1;                                                                                                       \
    while (L < 64 && 2 * L * p.G <= 256) L <<= 1;                                                                    \
    const int gl = (int)threadIdx.x & (L - 1), gs = 256 / L;

template <typename TI, typename TO, int V, int ACT>
__global__ __launch_bounds__(256) void gn_apply_kernel(GnArgs p) {
    extern __shared__ __attribute__((aligned(16))) float sm[];   // [G] mean, [G] rstd
    float *gm = sm, *gr = sm + p.G;
    GN_COLS(V, true)
    {
        GN_LANES
        const float cgf = (float)p.cg, N = (float)p.HW * cgf, full = (float)p.rows * cgf, last = (float)(p.HW - (p.nch - 1) * p.rows) * cgf;
        for (int g0 = 0; g0 < p.G; g0 += gs) {
            const int g = g0 + (int)threadIdx.x / L;
            // the mean around the first chunk's, then the squared deviations around the mean; four chunks in flight, the first four kept
            const float2* src = reinterpret_cast<const float2*>(p.part) + (size_t)b * p.nch * p.G + (g < p.G ? g : 0);
            const float m0 = src[0].x;
            float2 a[4];
            auto load = [&](int i0) {
#pragma unroll
                for (int k = 0; k < 4; ++k) a[k] = src[(size_t)min(i0 + k * L, p.nch - 1) * p.G];
            };
            auto values = [&](int i) { return i < p.nch - 1 ? full : i == p.nch - 1 ? last : 0.f; };   // in chunk i; one that is not there has none
            float s = 0.f, q = 0.f;
            load(gl);
            float2 first[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) first[k] = a[k];
            for (int i = gl;;) {
#pragma unroll
                for (int k = 0; k < 4; ++k) s = fmaf(values(i + k * L), a[k].x - m0, s);
                if ((i += 4 * L) >= p.nch) break;
                load(i);
            }
            for (int o = 1; o < L; o <<= 1) s += __shfl_xor(s, o, 64);
            const float m = m0 + s / N;
#pragma unroll
            for (int k = 0; k < 4; ++k) a[k] = first[k];
            for (int i = gl;;) {
#pragma unroll
                for (int k = 0; k < 4; ++k) { const float d = a[k].x - m, v = values(i + k * L); q += fmaf(v * d, d, v > 0.f ? a[k].y : 0.f); }
                if ((i += 4 * L) >= p.nch) break;
                load(i);
            }
            for (int o = 1; o < L; o <<= 1) q += __shfl_xor(q, o, 64);
            if (g < p.G && gl == 0) {
                const float rs = 1.f / sqrtf((q < 0.f ? 0.f : q) / N + p.eps);   // (a NaN stays one)
                gm[g] = m; gr[g] = rs;
                if (ch == 0) { p.mean[(size_t)b * p.G + g] = m; p.rstd[(size_t)b * p.G + g] = rs; }
            }
        }
    }
    __syncthreads();
    const TI* x = reinterpret_cast<const TI*>(p.x) + img;
    TO* y = reinterpret_cast<TO*>(p.y) + img;
    if (ty >= nr) return;
    for (int t0 = 0; t0 + tx < cv; t0 += tw) {
        const int c = (t0 + tx) * V;
        float m[V], a_[V], o[V];
        gn_each<V>(c, p.cg, [&](int e, int ce, int g) {
            m[e] = gm[g];
            a_[e] = gr[g] * (p.gamma ? p.gamma[ce] : 1.f);
            o[e] = p.beta ? p.beta[ce] : 0.f;
        });
        Vec<TI, V> a[4];
#define GN_U(K, R) { float v[V]; a[K].get(v); _Pragma("unroll") for (int e = 0; e < V; ++e) v[e] = gn_act<ACT>(fmaf(v[e] - m[e], a_[e], o[e])); \
                     vec_store<TO, V>(y + (size_t)(R) * p.C + c, v); }
        GN_ROWS(GN_L, GN_U);
#undef GN_U
#undef GN_L
    }
}

#define GN_L2(K, R) { a[K].load(x + (size_t)(R) * p.C + c); d[K].load(dy + (size_t)(R) * p.C + c); }
template <typename TI, typename TO, int V, int ACT>
__global__ __launch_bounds__(256) void gn_bwd_sums_kernel(GnArgs p) {
    extern __shared__ __attribute__((aligned(16))) float sm[];   // [C] sum dz xh, [C] sum dz, [V][2][256]
    float *ca = sm, *cb = sm + p.Cp, *red = cb + p.Cp;
    GN_COLS(V, false)
    const TI* x = reinterpret_cast<const TI*>(p.x) + img;
    const TO* dy = reinterpret_cast<const TO*>(p.dy) + img;
    float* o = p.cpart + ((size_t)b * p.nch + ch) * 2 * p.Cp;
    for (int t0 = 0; t0 < cv; t0 += tw) {
        const int c = (t0 + tx) * V;
        float sa[V], sb[V];
#pragma unroll
        for (int e = 0; e < V; ++e) { sa[e] = 0.f; sb[e] = 0.f; }
        if (ty < nr && t0 + tx < cv) {
            float m[V], A[V], be[V];
            gn_each<V>(c, p.cg, [&](int e, int ce, int g) {
                m[e] = p.mean[(size_t)b * p.G + g];
                A[e] = p.rstd[(size_t)b * p.G + g] * (p.gamma ? p.gamma[ce] : 1.f); be[e] = p.beta ? p.beta[ce] : 0.f;
            });
            Vec<TI, V> a[4];
            Vec<TO, V> d[4];
#define GN_U(K, R) { float v[V], w[V]; a[K].get(v); d[K].get(w); _Pragma("unroll") for (int e = 0; e < V; ++e) { \
                     const float dd = v[e] - m[e], dz = gn_dact<ACT>(fmaf(dd, A[e], be[e]), w[e]); sa[e] = fmaf(dz, dd, sa[e]); sb[e] += dz; } }
            GN_ROWS(GN_L2, GN_U);
#undef GN_U
        }
        __syncthreads();
#pragma unroll
        for (int e = 0; e < V; ++e) { red[e * 512 + threadIdx.x] = sa[e]; red[e * 512 + 256 + threadIdx.x] = sb[e]; }
        __syncthreads();
        for (int i = threadIdx.x; i < tw * V; i += 256) {
            const int e = i / tw, tt = i - e * tw;
            if (t0 + tt >= cv) continue;
            float s = 0.f, q = 0.f;
            for (int j = 0; j < nr; ++j) { s += red[e * 512 + j * tw + tt]; q += red[e * 512 + 256 + j * tw + tt]; }
            const int cc = (t0 + tt) * V + e;
            s *= p.rstd[(size_t)b * p.G + cc / p.cg];   // (the sums ran over dz d)
            ca[cc] = s; cb[cc] = q; o[cc] = s; o[p.Cp + cc] = q;
        }
    }
    if (threadIdx.x < p.Cp - p.C) { o[p.C + threadIdx.x] = 0.f; o[p.Cp + p.C + threadIdx.x] = 0.f; }   // (padding columns of the partial rows)
    __syncthreads();
    for (int g = threadIdx.x; g < p.G; g += 256) {
        float s1 = 0.f, s2 = 0.f;
        for (int c = g * p.cg; c < (g + 1) * p.cg; ++c) { const float ga = p.gamma ? p.gamma[c] : 1.f; s1 += ga * cb[c]; s2 += ga * ca[c]; }
        *reinterpret_cast<float2*>(p.part + (((size_t)b * p.nch + ch) * p.G + g) * 2) = make_float2(s1, s2);
    }
}

// workgroups behind the chunks fold the channel rows into dgamma / dbeta (f.src null: none)
template <typename TI, typename TO, int V, int ACT>
__global__ __launch_bounds__(256) void gn_bwd_apply_kernel(GnArgs p, RowsFoldArgs f) {
    extern __shared__ __attribute__((aligned(16))) float sm[];   // [G] S1 / n, [G] S2 / n; the fold's 256 float4
    if ((int)blockIdx.x >= p.B * p.nch) {
        rows_fold2_body(f, (int)blockIdx.x - p.B * p.nch, 0, reinterpret_cast<float4*>(sm));
        return;
    }
    float *g1 = sm, *g2 = sm + p.G;
    GN_COLS(V, true)
    {
        GN_LANES
        const float rn = 1.f / ((float)p.HW * (float)p.cg);
        for (int g0 = 0; g0 < p.G; g0 += gs) {
            const int g = g0 + (int)threadIdx.x / L;
            float s1 = 0.f, s2 = 0.f;
            if (g < p.G) {
                const float2* src = reinterpret_cast<const float2*>(p.part) + (size_t)b * p.nch * p.G + g;
                for (int i = gl; i < p.nch; i += L) { const float2 a = src[(size_t)i * p.G]; s1 += a.x; s2 += a.y; }
            }
            for (int o = 1; o < L; o <<= 1) { s1 += __shfl_xor(s1, o, 64); s2 += __shfl_xor(s2, o, 64); }
            if (g < p.G && gl == 0) { g1[g] = s1 * rn; g2[g] = s2 * rn; }
        }
    }
    __syncthreads();
    const TI* x = reinterpret_cast<const TI*>(p.x) + img;
    const TO* dy = reinterpret_cast<const TO*>(p.dy) + img;
    TI* dx = reinterpret_cast<TI*>(p.dx) + img;
    if (ty >= nr) return;
    for (int t0 = 0; t0 + tx < cv; t0 += tw) {
        const int c = (t0 + tx) * V;
        float m[V], A[V], be[V], s1[V], s2[V];   // dx = A dz - rstd S1 / n - d rstd^2 S2 / n
        gn_each<V>(c, p.cg, [&](int e, int ce, int g) {
            const float rs = p.rstd[(size_t)b * p.G + g];
            m[e] = p.mean[(size_t)b * p.G + g];
            A[e] = rs * (p.gamma ? p.gamma[ce] : 1.f); be[e] = p.beta ? p.beta[ce] : 0.f;
            s1[e] = rs * g1[g]; s2[e] = rs * rs * g2[g];
        });
        Vec<TI, V> a[4];
        Vec<TO, V> d[4];
#define GN_U(K, R) { float v[V], w[V]; a[K].get(v); d[K].get(w); _Pragma("unroll") for (int e = 0; e < V; ++e) { \
                     const float dd = v[e] - m[e], dz = gn_dact<ACT>(fmaf(dd, A[e], be[e]), w[e]); \
                     v[e] = fmaf(A[e], dz, -fmaf(dd, s2[e], s1[e])); } vec_store<TI, V>(dx + (size_t)(R) * p.C + c, v); }
        GN_ROWS(GN_L2, GN_U);
#undef GN_U
    }
}
#undef GN_L2

// ------------------------------------------------------------------------------------------------ resident form
// Thread (ty, tx) holds rows ty, ty + nr, ... (at most R: 4, for maps of two bytes a value up to 8) of V channels of the slab. Sums over the slab's groups: row lanes meet in a tree in
// LDS (fixed order), a wave adds a group's channels.
template <int V>
__device__ __forceinline__ void gn_channel_sums(const GnArgs& p, int cs, int tx, int ty, bool on, const float (&s)[V], float* red /* [nr][cs] */, float* out /* [cs] */) {
    __syncthreads();
    if (on)
#pragma unroll
        for (int e = 0; e < V; ++e) red[ty * cs + tx * V + e] = s[e];
    int st = 1;
    while (2 * st < p.nr) st <<= 1;
    for (; st >= 1; st >>= 1) {
        __syncthreads();
        if (on && ty < st && ty + st < p.nr)
#pragma unroll
            for (int e = 0; e < V; ++e) red[ty * cs + tx * V + e] += red[(ty + st) * cs + tx * V + e];
    }
    if (on && ty == 0)
#pragma unroll
        for (int e = 0; e < V; ++e) out[tx * V + e] = red[tx * V + e];
    __syncthreads();
}
#define GN_RES(V)                                                                                                    \
    const int b = blockIdx.x / p.slabs, slab = blockIdx.x - b * p.slabs, c0 = slab * p.Cs, cs = p.C - c0 < p.Cs ? p.C - c0 : p.Cs; \
    const int tx = (int)threadIdx.x % p.tw, ty = (int)threadIdx.x / p.tw, c = c0 + tx * (V), g0 = c0 / p.cg, ng = cs / p.cg; \
    const bool on = ty < p.nr && tx * (V) < cs;                                                                      \
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, nw = blockDim.x >> 6;                                \
    const size_t base = ((size_t)b * p.HW + ty) * p.C + c, step = (size_t)p.nr * p.C;

template <typename TI, typename TO, int V, int ACT, int R>
__global__ __launch_bounds__(256) void gn_res_kernel(GnArgs p) {
    extern __shared__ __attribute__((aligned(16))) float sm[];   // [nr][Cs], [Cs] channel sums, [2][Cs] per-group results
    float *red = sm, *chan = sm + p.nr * p.Cs, *gres = chan + p.Cs;
    GN_RES(V)
    const TI* x = reinterpret_cast<const TI*>(p.x) + base;
    const TI* origin = reinterpret_cast<const TI*>(p.x) + (size_t)b * p.HW * p.C;   // a group's first value of the first pixel: what its sum is counted from
    Vec<TI, V> a[R];
    float s[V], v[V], k[V];
#pragma unroll
    for (int j = 0; j < R; ++j) if (on && ty + j * p.nr < p.HW) a[j].load(x + j * step);
    gn_each<V>(on ? c : c0, p.cg, [&](int e, int, int g) { k[e] = OpT<TI>::to(origin[g * p.cg]); s[e] = 0.f; });
#pragma unroll
    for (int j = 0; j < R; ++j)
        if (on && ty + j * p.nr < p.HW) {
            a[j].get(v);
#pragma unroll
            for (int e = 0; e < V; ++e) s[e] += v[e] - k[e];
        }
    const float rn = 1.f / ((float)p.HW * (float)p.cg);
    gn_channel_sums<V>(p, cs, tx, ty, on, s, red, chan);
    for (int g = wave; g < ng; g += nw) {
        float t = 0.f;
        for (int i = lane; i < p.cg; i += 64) t += chan[g * p.cg + i];
        t = wave_sum(t);
        if (lane == 0) gres[g] = fmaf(t, rn, OpT<TI>::to(origin[(g0 + g) * p.cg]));
    }
    __syncthreads();
    float m[V], r[V];
    gn_each<V>(on ? c : c0, p.cg, [&](int e, int, int g) { m[e] = gres[g - g0]; s[e] = 0.f; });
#pragma unroll
    for (int k = 0; k < R; ++k)
        if (on && ty + k * p.nr < p.HW) {
            a[k].get(v);
#pragma unroll
            for (int e = 0; e < V; ++e) { const float d = v[e] - m[e]; s[e] = fmaf(d, d, s[e]); }
        }
    gn_channel_sums<V>(p, cs, tx, ty, on, s, red, chan);
    for (int g = wave; g < ng; g += nw) {
        float t = 0.f;
        for (int i = lane; i < p.cg; i += 64) t += chan[g * p.cg + i];
        t = wave_sum(t);
        if (lane == 0) {
            const float rs = 1.f / sqrtf(t * rn + p.eps);
            p.mean[(size_t)b * p.G + g0 + g] = gres[g]; p.rstd[(size_t)b * p.G + g0 + g] = rs;
            gres[p.Cs + g] = rs;
        }
    }
    __syncthreads();
    if (!on) return;
    TO* y = reinterpret_cast<TO*>(p.y) + base;
    gn_each<V>(c, p.cg, [&](int e, int ce, int g) { r[e] = gres[p.Cs + g - g0] * (p.gamma ? p.gamma[ce] : 1.f); s[e] = p.beta ? p.beta[ce] : 0.f; });
#pragma unroll
    for (int k = 0; k < R; ++k)
        if (ty + k * p.nr < p.HW) {
            a[k].get(v);
#pragma unroll
            for (int e = 0; e < V; ++e) v[e] = gn_act<ACT>(fmaf(v[e] - m[e], r[e], s[e]));
            vec_store<TO, V>(y + k * step, v);
        }
}

template <typename TI, typename TO, int V, int ACT, int R>
__global__ __launch_bounds__(256) void gn_res_bwd_kernel(GnArgs p) {
    extern __shared__ __attribute__((aligned(16))) float sm[];   // [nr][Cs], [2][Cs] channel sums, [2][Cs] per-group results
    float *red = sm, *ra = sm + p.nr * p.Cs, *rb = ra + p.Cs, *gres = rb + p.Cs;
    GN_RES(V)
    const TI* x = reinterpret_cast<const TI*>(p.x) + base;
    const TO* dy = reinterpret_cast<const TO*>(p.dy) + base;
    Vec<TI, V> a[R];
    Vec<TO, V> d[R];
#pragma unroll
    for (int k = 0; k < R; ++k) if (on && ty + k * p.nr < p.HW) { a[k].load(x + k * step); d[k].load(dy + k * step); }
    float m[V], rs[V], A[V], be[V], sa[V], sb[V], v[V], w[V];
    gn_each<V>(on ? c : c0, p.cg, [&](int e, int ce, int g) {
        m[e] = p.mean[(size_t)b * p.G + g]; rs[e] = p.rstd[(size_t)b * p.G + g];
        A[e] = rs[e] * (p.gamma ? p.gamma[ce] : 1.f); be[e] = p.beta ? p.beta[ce] : 0.f;
        sa[e] = 0.f; sb[e] = 0.f;
    });
#pragma unroll
    for (int k = 0; k < R; ++k)
        if (on && ty + k * p.nr < p.HW) {
            a[k].get(v); d[k].get(w);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float dd = v[e] - m[e], dz = gn_dact<ACT>(fmaf(dd, A[e], be[e]), w[e]);
                sa[e] = fmaf(dz, dd, sa[e]); sb[e] += dz;
            }
        }
#pragma unroll
    for (int e = 0; e < V; ++e) sa[e] *= rs[e];   // (sum dz d -> sum dz xh)
    gn_channel_sums<V>(p, cs, tx, ty, on, sa, red, ra);
    gn_channel_sums<V>(p, cs, tx, ty, on, sb, red, rb);
    float* o = p.cpart + (size_t)b * 2 * p.Cp;
    for (int i = threadIdx.x; i < cs; i += blockDim.x) { o[c0 + i] = ra[i]; o[p.Cp + c0 + i] = rb[i]; }
    if (c0 + cs == p.C && (int)threadIdx.x < p.Cp - p.C) { o[p.C + threadIdx.x] = 0.f; o[p.Cp + p.C + threadIdx.x] = 0.f; }
    if (!p.dx) return;   // (uniform over the launch)
    const float rn = 1.f / ((float)p.HW * (float)p.cg);
    for (int g = wave; g < ng; g += nw) {
        float t1 = 0.f, t2 = 0.f;
        for (int i = lane; i < p.cg; i += 64) {
            const float gg = p.gamma ? p.gamma[c0 + g * p.cg + i] : 1.f;
            t1 += gg * rb[g * p.cg + i]; t2 += gg * ra[g * p.cg + i];
        }
        t1 = wave_sum(t1); t2 = wave_sum(t2);
        if (lane == 0) { gres[g] = t1 * rn; gres[p.Cs + g] = t2 * rn; }
    }
    __syncthreads();
    if (!on) return;
    TI* dx = reinterpret_cast<TI*>(p.dx) + base;
    gn_each<V>(c, p.cg, [&](int e, int, int g) { sa[e] = rs[e] * gres[g - g0]; sb[e] = rs[e] * rs[e] * gres[p.Cs + g - g0]; });
#pragma unroll
    for (int k = 0; k < R; ++k)
        if (ty + k * p.nr < p.HW) {
            a[k].get(v); d[k].get(w);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float dd = v[e] - m[e], dz = gn_dact<ACT>(fmaf(dd, A[e], be[e]), w[e]);
                v[e] = fmaf(A[e], dz, -fmaf(dd, sb[e], sa[e]));
            }
            vec_store<TI, V>(dx + k * step, v);
        }
}

// ------------------------------------------------------------------------------------------------ entry points
#define GN_MAX_C 4096
// chunks per image: 512 workgroups over the chip (two a CU; 1024 cost 10 us more on four launches over 64 x 64 x 128 x 32 images in bf16, the same in
// f32: what stands in front of a workgroup's loop is paid less often), at least 8192 values each, at most 256 an image, each of whose chunks every
// workgroup of the second launch joins (forward and with backward, at most 256 and at most 512: one 1024 x 1024 x 64 f32 169 and 436 us, 181 and 459; bf16
// 73 and 209, 90 and 225; 256 x 256 x 128 f32 28 and 69, 41 and 90; 128 x 128 x 256 bf16 20 and 45, 35 and 72)
static int gn_chunks(int B, long long HW, int C) {
    long long want = (512 + B - 1) / B, most = (HW * C + 8191) / 8192;
    if (want > most) want = most;
    if (want > HW) want = HW;
    if (want > 256) want = 256;
    return want < 1 ? 1 : (int)want;
}
static bool gn_bad(int B, long long HW, int C, int G, int act, int d0, int d1) {
    return B < 1 || B > 65535 || HW < 1 || C < 1 || C > GN_MAX_C || G < 1 || C % G || act < 0 || act > 2 || ((d0 | d1) & ~1) || HW > (1LL << 40) / C;
}
extern "C" int l2i_group_norm_scratch(int B, long long HW, int C, int G, int bwd, long long* floats) {
    if (!floats || gn_bad(B, HW, C, G, 0, 0, 0)) return L2I_ERR_ARG;
    const long long nch = gn_chunks(B, HW, C), Cp = (C + 3) & ~3;
    const long long rows = (long long)B * nch;
    *floats = ((rows * G * 2 + 3) & ~3LL) + (bwd ? rows * 2 * Cp + (rows > L2I_FOLD_DIRECT ? rows_fold_tmp_floats((int)rows, (int)Cp, 1) : 0) : 0);
    return L2I_OK;
}
// resident form: where a slab of whole groups and vectors of four fits a workgroup's registers, 64 bytes of x a thread. Both forms, forward and
// forward with backward, silu: one bf16 image of 4 x 4 x 1024 7 and 16 us, split 14 and 29; 32 of 16 x 16 x 512 bf16 11 and 28, split 16 and 40; 32 of 12 x 12 x
// 512 f32 11 and 28, split 13 and 30; at 32 of 16 x 16 x 512 f32 they meet (15 and 38, split 14 and 35). Workgroups of 1024 threads for
// 32 x 32 x 256 lose (bf16 26 and 60, split 18 and 45), vectors of eight too (32 of 8 x 8 x 1024: 16 and 35, of four 10 and 22).
static bool gn_resident(GnArgs& a, int v, int in, int out) {
    if (v == 1) return false;
    const int es = in && out ? 2 : 4;
    int cs = a.cg;
    while (cs < a.C && (cs % 4 || cs * es < 64)) cs += a.cg;   // 64 bytes of a pixel
    if (cs > a.C) cs = a.C;
    a.Cs = cs; a.slabs = (a.C + cs - 1) / cs; a.tw = cs / 4;
    if (cs % 4 || a.tw > 256 || (long long)(256 / a.tw) * (in && out ? 8 : 4) < a.HW) return false;
    a.nr = 256 / a.tw < a.HW ? 256 / a.tw : (int)a.HW;
    return true;
}
static void gn_setup(GnArgs& a, int B, long long HW, int C, int G, int act, float eps, float* scratch) {
    a.B = B; a.HW = HW; a.C = C; a.Cp = (C + 3) & ~3; a.G = G; a.cg = C / G; a.act = act; a.eps = eps;
    a.nch = gn_chunks(B, HW, C);
    a.rows = (HW + a.nch - 1) / a.nch;
    a.nch = (int)((HW + a.rows - 1) / a.rows);   // (every chunk has a row)
    a.part = scratch;
    a.cpart = scratch + ((((long long)B * a.nch * G * 2) + 3) & ~3LL);
}
template <typename TI, typename TO, int V, int ACT>
static void gn_fwd_launch(GnArgs& a, bool res, hipStream_t s) {
    if constexpr (V == 4) {
        if (res) {
            const size_t lds = sizeof(float) * ((size_t)a.nr * a.Cs + 3 * a.Cs);
            if (a.HW <= 4 * a.nr) hipLaunchKernelGGL((gn_res_kernel<TI, TO, V, ACT, 4>), dim3(a.B * a.slabs), dim3(256), lds, s, a);
            else if constexpr (sizeof(TI) == 2 && sizeof(TO) == 2) hipLaunchKernelGGL((gn_res_kernel<TI, TO, V, ACT, 8>), dim3(a.B * a.slabs), dim3(256), lds, s, a);
            return;
        }
    }
    const dim3 grid(a.nch * a.B);
    hipLaunchKernelGGL((gn_stats_kernel<TI, V>), grid, dim3(256), sizeof(float) * (2 * a.Cp + 512 * V), s, a);
    hipLaunchKernelGGL((gn_apply_kernel<TI, TO, V, ACT>), grid, dim3(256), sizeof(float) * 2 * a.G, s, a);
}
template <typename TI, typename TO, int V, int ACT>
static void gn_bwd_launch(GnArgs& a, bool res, hipStream_t s, float* dgamma, float* dbeta) {
    int rows = a.B * a.nch;
    bool folded = !dgamma && !dbeta;
    if constexpr (V == 4) {
        if (res) {
            const size_t lds = sizeof(float) * ((size_t)a.nr * a.Cs + 4 * a.Cs);
            if (a.HW <= 4 * a.nr) hipLaunchKernelGGL((gn_res_bwd_kernel<TI, TO, V, ACT, 4>), dim3(a.B * a.slabs), dim3(256), lds, s, a);
            else if constexpr (sizeof(TI) == 2 && sizeof(TO) == 2) hipLaunchKernelGGL((gn_res_bwd_kernel<TI, TO, V, ACT, 8>), dim3(a.B * a.slabs), dim3(256), lds, s, a);
            rows = a.B;
        }
    }
    RowsFoldArgs f = {};
    if (!folded && rows <= L2I_FOLD_DIRECT) f = rows_fold_args4(a.cpart, rows, 2 * a.Cp, 1, dgamma, dbeta, nullptr, nullptr, a.Cp, a.C, 0, 0, nullptr, 2 * a.Cp);
    if (!res) {
        hipLaunchKernelGGL((gn_bwd_sums_kernel<TI, TO, V, ACT>), dim3(rows), dim3(256), sizeof(float) * (2 * a.Cp + 512 * V), s, a);
        if (a.dx) {
            const size_t lds = sizeof(float) * 2 * a.G;
            hipLaunchKernelGGL((gn_bwd_apply_kernel<TI, TO, V, ACT>), dim3(rows + (f.src ? f.nbx : 0)), dim3(256), lds < 4096 ? 4096 : lds, s, a, f);
            folded = folded || f.src;
        }
    }
    if (!folded) {
        if (f.src) hipLaunchKernelGGL(rows_fold2_kernel, dim3(f.nbx), dim3(256), 0, s, f);
        else {
            float* tmp = a.cpart + (size_t)rows * 2 * a.Cp;
            if (dgamma) rows_fold(a.cpart, rows, a.Cp, 1, dgamma, nullptr, a.C, 0, 0, tmp, s, nullptr, 2 * a.Cp);
            if (dbeta) rows_fold(a.cpart + a.Cp, rows, a.Cp, 1, dbeta, nullptr, a.C, 0, 0, tmp, s, nullptr, 2 * a.Cp);
        }
    }
}
#define GN_ACTS(FN, TI, TO, V, ...)                                                                                  \
    do {                                                                                                             \
        if (act == 0) FN<TI, TO, V, 0>(__VA_ARGS__); else if (act == 1) FN<TI, TO, V, 1>(__VA_ARGS__); else FN<TI, TO, V, 2>(__VA_ARGS__); \
    } while (0)
#define GN_VECS(FN, TI, TO, ...)                                                                                     \
    do {                                                                                                             \
        if (vec == 8) GN_ACTS(FN, TI, TO, 8, __VA_ARGS__); else if (vec == 4) GN_ACTS(FN, TI, TO, 4, __VA_ARGS__); else GN_ACTS(FN, TI, TO, 1, __VA_ARGS__); \
    } while (0)
#define GN_DISPATCH(FN, ...)                                                                                         \
    do {                                                                                                             \
        int vec = vec_width(a.C, (const void*)((size_t)a.x | (size_t)a.dx), x_dtype, (const void*)((size_t)a.y | (size_t)a.dy), y_dtype); \
        const bool res = gn_resident(a, vec, x_dtype, y_dtype);                                                      \
        if (res) vec = 4;                                                                                            \
        if (x_dtype == 0 && y_dtype == 0) GN_VECS(FN, float, float, a, res, __VA_ARGS__);                            \
        else if (x_dtype == 0) GN_VECS(FN, float, bf16_t, a, res, __VA_ARGS__);                                      \
        else if (y_dtype == 0) GN_VECS(FN, bf16_t, float, a, res, __VA_ARGS__);                                      \
        else GN_VECS(FN, bf16_t, bf16_t, a, res, __VA_ARGS__);                                                       \
    } while (0)

extern "C" int l2i_group_norm_fwd(const void* x, int x_dtype, const float* gamma, const float* beta, void* y, int y_dtype, float* mean, float* rstd,
                                  int B, long long HW, int C, int G, float eps, int act, float* scratch, long long scratch_floats, void* stream) {
    long long need = 0;
    if (gn_bad(B, HW, C, G, act, x_dtype, y_dtype) || !x || !y || !mean || !rstd || !scratch || ((size_t)scratch & 15)) return L2I_ERR_ARG;
    if (l2i_group_norm_scratch(B, HW, C, G, 0, &need) != L2I_OK || scratch_floats < need) return L2I_ERR_ARG;
    GnArgs a = {};
    a.x = x; a.gamma = gamma; a.beta = beta; a.y = y; a.mean = mean; a.rstd = rstd;
    gn_setup(a, B, HW, C, G, act, eps, scratch);
    hipStream_t s = (hipStream_t)stream;
    GN_DISPATCH(gn_fwd_launch, s);
    return l2i_check_launch();
}
extern "C" int l2i_group_norm_bwd(const void* x, int x_dtype, const float* gamma, const float* beta, const float* mean, const float* rstd, const void* dy,
                                  int y_dtype, void* dx, float* dgamma, float* dbeta, int B, long long HW, int C, int G, int act, float* scratch,
                                  long long scratch_floats, void* stream) {
    long long need = 0;
    if (gn_bad(B, HW, C, G, act, x_dtype, y_dtype) || !x || !dy || !mean || !rstd || !scratch || ((size_t)scratch & 15)) return L2I_ERR_ARG;
    if (l2i_group_norm_scratch(B, HW, C, G, 1, &need) != L2I_OK || scratch_floats < need) return L2I_ERR_ARG;
    GnArgs a = {};
    a.x = x; a.gamma = gamma; a.beta = beta; a.mean = const_cast<float*>(mean); a.rstd = const_cast<float*>(rstd); a.dy = dy; a.dx = dx;
    gn_setup(a, B, HW, C, G, act, 0.f, scratch);
    hipStream_t s = (hipStream_t)stream;
    GN_DISPATCH(gn_bwd_launch, s, dgamma, dbeta);
    return l2i_check_launch();
}
