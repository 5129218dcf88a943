// Group normalisation with an activation on channels-last maps, forward and backward.
//
//   per image b and group g of C / G consecutive channels, over its n = HW * C / G values:
//     mean, var = biased moments;  xh = (x - mean) * rstd, rstd = 1 / sqrt(var + eps);  z = gamma_c xh + beta_c;  y = act(z)
//   backward, dz = dy act'(z):
//     dbeta_c = sum dz;  dgamma_c = sum dz xh;  dx = rstd (gamma dz - (S1 + xh S2) / n),  S1 = sum gamma dz, S2 = sum gamma dz xh over the group
//
// Bound by bytes. The map is cut in NCH chunks of rows (pixels) per image. The first launch leaves every chunk's moments (mean and sum of
// squared deviations per group: sums around a value of the chunk itself, so that a mean far from zero costs no digits), the second joins
// them in chunk order and writes the result; in the backward pass the first leaves the group sums and the channel rows that
// l2i's ordered fold adds into dgamma / dbeta. Statistics are f32; nothing is accumulated by atomics.
#include "common.h"

struct GnArgs {
    const void* x; const float* gamma; const float* beta; void* y;
    float* mean; float* rstd;             // [B][G]
    const void* dy; void* dx;
    float* part;                          // forward: [B][NCH][G] (mean, M2); backward: [B][NCH][G] (S1, S2)
    float* cpart;                         // backward: [B][NCH][2 Cp] rows of (sum dz xh | sum dz)
    long long HW; long long rows;         // rows per chunk
    int B, C, Cp, G, cg, nch, act;
    float eps;
};

// act'(z) * dy, and act(z)
__device__ __forceinline__ float gn_act(float z, int act) {
    if (act == 1) return fmaxf(z, 0.f);
    if (act == 2) return z / (1.f + __expf(-z));
    return z;
}
__device__ __forceinline__ float gn_dact(float z, float dy, int act) {
    if (act == 1) return z > 0.f ? dy : 0.f;
    if (act == 2) { const float s = 1.f / (1.f + __expf(-z)); return dy * s * (1.f + z * (1.f - s)); }
    return dy;
}

template <typename T, int V> __device__ __forceinline__ void gn_load(const T* p, float (&v)[V]) {
    if constexpr (V == 4) Op4<T>::load(p, v);
    else v[0] = OpT<T>::to(p[0]);
}
template <typename T, int V> __device__ __forceinline__ void gn_store(T* p, const float (&v)[V]) {
    if constexpr (V == 4) Op4<T>::store(p, v);
    else p[0] = OpT<T>::from(v[0]);
}

// Column mapping shared by the four kernels: a workgroup covers all C channels of its rows in tiles of tw = min(C / V, 256) vectors; tw threads
// stand along the channels, 256 / tw along the rows.
#define GN_COLS(V)                                                                                                   \
    const int cv = p.C / (V), tw = cv < 256 ? cv : 256, nr = 256 / tw, tx = (int)threadIdx.x % tw, ty = (int)threadIdx.x / tw; \
    const int b = blockIdx.y, ch = blockIdx.x;                                                                       \
    const long long r0 = ch * p.rows, r1 = r0 + p.rows < p.HW ? r0 + p.rows : p.HW;                                   \
    const size_t img = (size_t)b * p.HW * p.C;

template <typename T, int V>
__global__ __launch_bounds__(256) void gn_stats_kernel(GnArgs p) {
    extern __shared__ __attribute__((aligned(16))) float sm[];   // [C] means, [C] squared deviations, [256][2 V] row lanes
    float *cm = sm, *cq = sm + p.Cp, *red = cq + p.Cp;
    GN_COLS(V)
    const T* x = reinterpret_cast<const T*>(p.x) + img;
    const float n = (float)(r1 - r0);
    for (int t0 = 0; t0 < cv; t0 += tw) {
        const int c = (t0 + tx) * V;
        const bool on = ty < nr && t0 + tx < cv;
        float s[V], q[V], k[V];
#pragma unroll
        for (int e = 0; e < V; ++e) { s[e] = 0.f; q[e] = 0.f; k[e] = 0.f; }
        if (on) {
            gn_load<T, V>(x + (size_t)r0 * p.C + c, k);
            for (long long r = r0 + ty; r < r1; r += nr) {
                float v[V];
                gn_load<T, V>(x + (size_t)r * p.C + c, v);
#pragma unroll
                for (int e = 0; e < V; ++e) { const float d = v[e] - k[e]; s[e] += d; q[e] += d * d; }
            }
        }
        __syncthreads();
#pragma unroll
        for (int e = 0; e < V; ++e) { red[threadIdx.x * 2 * V + e] = s[e]; red[threadIdx.x * 2 * V + V + e] = q[e]; }
        __syncthreads();
        if (ty == 0 && t0 + tx < cv) {
            for (int j = 1; j < nr; ++j)
#pragma unroll
                for (int e = 0; e < V; ++e) { s[e] += red[(j * tw + tx) * 2 * V + e]; q[e] += red[(j * tw + tx) * 2 * V + V + e]; }
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float m = s[e] / n;
                cm[c + e] = k[e] + m;
                cq[c + e] = q[e] - s[e] * m;
            }
        }
    }
    __syncthreads();
    for (int g = threadIdx.x; g < p.G; g += 256) {   // the group's channels, all over the same n rows
        float m = 0.f, m2 = 0.f;
        for (int c = g * p.cg; c < (g + 1) * p.cg; ++c) m += cm[c];
        m /= (float)p.cg;
        for (int c = g * p.cg; c < (g + 1) * p.cg; ++c) { const float d = cm[c] - m; m2 += cq[c] + n * d * d; }
        float* o = p.part + (((size_t)b * p.nch + ch) * p.G + g) * 2;
        o[0] = m; o[1] = m2;
    }
}

template <typename TI, typename TO, int V>
__global__ __launch_bounds__(256) void gn_apply_kernel(GnArgs p) {
    extern __shared__ __attribute__((aligned(16))) float sm[];   // [G] mean, [G] rstd
    float *gm = sm, *gr = sm + p.G;
    GN_COLS(V)
    for (int g = threadIdx.x; g < p.G; g += 256) {
        const float* q = p.part + ((size_t)b * p.nch * p.G + g) * 2;
        float m = 0.f, m2 = 0.f;
        for (int i = 0; i < p.nch; ++i) {
            const long long ra = i * p.rows, rb = ra + p.rows < p.HW ? ra + p.rows : p.HW;
            m += q[(size_t)i * p.G * 2] * ((float)(rb - ra) / (float)p.HW);
        }
        for (int i = 0; i < p.nch; ++i) {
            const long long ra = i * p.rows, rb = ra + p.rows < p.HW ? ra + p.rows : p.HW;
            const float d = q[(size_t)i * p.G * 2] - m;
            m2 += q[(size_t)i * p.G * 2 + 1] + d * d * (float)(rb - ra) * (float)p.cg;
        }
        const float rs = 1.f / sqrtf(fmaxf(m2, 0.f) / ((float)p.HW * (float)p.cg) + p.eps);
        gm[g] = m; gr[g] = rs;
        if (ch == 0) { p.mean[(size_t)b * p.G + g] = m; p.rstd[(size_t)b * p.G + g] = rs; }
    }
    __syncthreads();
    const TI* x = reinterpret_cast<const TI*>(p.x) + img;
    TO* y = reinterpret_cast<TO*>(p.y) + img;
    if (ty >= nr) return;
    for (int t0 = 0; t0 + tx < cv; t0 += tw) {
        const int c = (t0 + tx) * V;
        float m[V], a[V], o[V];
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const int g = (c + e) / p.cg;
            m[e] = gm[g];
            a[e] = gr[g] * (p.gamma ? p.gamma[c + e] : 1.f);
            o[e] = p.beta ? p.beta[c + e] : 0.f;
        }
        for (long long r = r0 + ty; r < r1; r += nr) {
            float v[V];
            gn_load<TI, V>(x + (size_t)r * p.C + c, v);
#pragma unroll
            for (int e = 0; e < V; ++e) v[e] = gn_act((v[e] - m[e]) * a[e] + o[e], p.act);
            gn_store<TO, V>(y + (size_t)r * p.C + c, v);
        }
    }
}

template <typename TI, typename TO, int V>
__global__ __launch_bounds__(256) void gn_bwd_sums_kernel(GnArgs p) {
    extern __shared__ __attribute__((aligned(16))) float sm[];   // [C] sum dz xh, [C] sum dz, [256][2 V]
    float *ca = sm, *cb = sm + p.Cp, *red = cb + p.Cp;
    GN_COLS(V)
    const TI* x = reinterpret_cast<const TI*>(p.x) + img;
    const TO* dy = reinterpret_cast<const TO*>(p.dy) + img;
    for (int t0 = 0; t0 < cv; t0 += tw) {
        const int c = (t0 + tx) * V;
        const bool on = ty < nr && t0 + tx < cv;
        float sa[V], sb[V];
#pragma unroll
        for (int e = 0; e < V; ++e) { sa[e] = 0.f; sb[e] = 0.f; }
        if (on) {
            float m[V], rs[V], ga[V], be[V];
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const int g = (c + e) / p.cg;
                m[e] = p.mean[(size_t)b * p.G + g]; rs[e] = p.rstd[(size_t)b * p.G + g];
                ga[e] = p.gamma ? p.gamma[c + e] : 1.f; be[e] = p.beta ? p.beta[c + e] : 0.f;
            }
            for (long long r = r0 + ty; r < r1; r += nr) {
                float v[V], d[V];
                gn_load<TI, V>(x + (size_t)r * p.C + c, v);
                gn_load<TO, V>(dy + (size_t)r * p.C + c, d);
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    const float xh = (v[e] - m[e]) * rs[e], dz = gn_dact(xh * ga[e] + be[e], d[e], p.act);
                    sa[e] += dz * xh; sb[e] += dz;
                }
            }
        }
        __syncthreads();
#pragma unroll
        for (int e = 0; e < V; ++e) { red[threadIdx.x * 2 * V + e] = sa[e]; red[threadIdx.x * 2 * V + V + e] = sb[e]; }
        __syncthreads();
        if (ty == 0 && t0 + tx < cv) {
            for (int j = 1; j < nr; ++j)
#pragma unroll
                for (int e = 0; e < V; ++e) { sa[e] += red[(j * tw + tx) * 2 * V + e]; sb[e] += red[(j * tw + tx) * 2 * V + V + e]; }
            float* o = p.cpart + ((size_t)b * p.nch + ch) * 2 * p.Cp;
#pragma unroll
            for (int e = 0; e < V; ++e) { ca[c + e] = sa[e]; cb[c + e] = sb[e]; o[c + e] = sa[e]; o[p.Cp + c + e] = sb[e]; }
        }
    }
    if (threadIdx.x < p.Cp - p.C) {   // (padding columns of the partial rows)
        float* o = p.cpart + ((size_t)b * p.nch + ch) * 2 * p.Cp + p.C + threadIdx.x;
        o[0] = 0.f; o[p.Cp] = 0.f;
    }
    __syncthreads();
    for (int g = threadIdx.x; g < p.G; g += 256) {
        float s1 = 0.f, s2 = 0.f;
        for (int c = g * p.cg; c < (g + 1) * p.cg; ++c) { const float ga = p.gamma ? p.gamma[c] : 1.f; s1 += ga * cb[c]; s2 += ga * ca[c]; }
        float* o = p.part + (((size_t)b * p.nch + ch) * p.G + g) * 2;
        o[0] = s1; o[1] = s2;
    }
}

template <typename TI, typename TO, int V>
__global__ __launch_bounds__(256) void gn_bwd_apply_kernel(GnArgs p) {
    extern __shared__ __attribute__((aligned(16))) float sm[];   // [G] S1 / n, [G] S2 / n
    float *g1 = sm, *g2 = sm + p.G;
    GN_COLS(V)
    const float rn = 1.f / ((float)p.HW * (float)p.cg);
    for (int g = threadIdx.x; g < p.G; g += 256) {
        const float* q = p.part + ((size_t)b * p.nch * p.G + g) * 2;
        float s1 = 0.f, s2 = 0.f;
        for (int i = 0; i < p.nch; ++i) { s1 += q[(size_t)i * p.G * 2]; s2 += q[(size_t)i * p.G * 2 + 1]; }
        g1[g] = s1 * rn; g2[g] = s2 * rn;
    }
    __syncthreads();
    const TI* x = reinterpret_cast<const TI*>(p.x) + img;
    const TO* dy = reinterpret_cast<const TO*>(p.dy) + img;
    TI* dx = reinterpret_cast<TI*>(p.dx) + img;
    if (ty >= nr) return;
    for (int t0 = 0; t0 + tx < cv; t0 += tw) {
        const int c = (t0 + tx) * V;
        float m[V], rs[V], ga[V], be[V], s1[V], s2[V];
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const int g = (c + e) / p.cg;
            m[e] = p.mean[(size_t)b * p.G + g]; rs[e] = p.rstd[(size_t)b * p.G + g];
            ga[e] = p.gamma ? p.gamma[c + e] : 1.f; be[e] = p.beta ? p.beta[c + e] : 0.f;
            s1[e] = g1[g]; s2[e] = g2[g];
        }
        for (long long r = r0 + ty; r < r1; r += nr) {
            float v[V], d[V];
            gn_load<TI, V>(x + (size_t)r * p.C + c, v);
            gn_load<TO, V>(dy + (size_t)r * p.C + c, d);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float xh = (v[e] - m[e]) * rs[e], dz = gn_dact(xh * ga[e] + be[e], d[e], p.act);
                v[e] = rs[e] * (ga[e] * dz - (s1[e] + xh * s2[e]));
            }
            gn_store<TI, V>(dx + (size_t)r * p.C + c, v);
        }
    }
}

// ------------------------------------------------------------------------------------------------ entry points
#define GN_MAX_C 4096
// chunks per image: 1024 workgroups over the chip, at least 8 rows of 256 vectors each
static int gn_chunks(int B, long long HW, int C) {
    long long want = (1024 + B - 1) / B, most = (HW * C + 8191) / 8192;
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
    *floats = ((rows * G * 2 + 3) & ~3LL) + (bwd ? rows * 2 * Cp + (rows > L2I_FOLD_DIRECT ? rows_fold_tmp_floats((int)rows, 2 * (int)Cp, 1) : 0) : 0);
    return L2I_OK;
}
static void gn_setup(GnArgs& a, int B, long long HW, int C, int G, int act, float eps, float* scratch) {
    a.B = B; a.HW = HW; a.C = C; a.Cp = (C + 3) & ~3; a.G = G; a.cg = C / G; a.act = act; a.eps = eps;
    a.nch = gn_chunks(B, HW, C);
    a.rows = (HW + a.nch - 1) / a.nch;
    a.nch = (int)((HW + a.rows - 1) / a.rows);   // (every chunk has a row)
    a.part = scratch;
    a.cpart = scratch + ((((long long)B * a.nch * G * 2) + 3) & ~3LL);
}
template <typename TI, typename TO, int V>
static void gn_fwd_launch(const GnArgs& a, hipStream_t s) {
    const dim3 grid(a.nch, a.B);
    hipLaunchKernelGGL((gn_stats_kernel<TI, V>), grid, dim3(256), sizeof(float) * (2 * a.Cp + 512 * V), s, a);
    hipLaunchKernelGGL((gn_apply_kernel<TI, TO, V>), grid, dim3(256), sizeof(float) * 2 * a.G, s, a);
}
template <typename TI, typename TO, int V>
static void gn_bwd_launch(const GnArgs& a, hipStream_t s) {
    const dim3 grid(a.nch, a.B);
    hipLaunchKernelGGL((gn_bwd_sums_kernel<TI, TO, V>), grid, dim3(256), sizeof(float) * (2 * a.Cp + 512 * V), s, a);
    if (a.dx) hipLaunchKernelGGL((gn_bwd_apply_kernel<TI, TO, V>), grid, dim3(256), sizeof(float) * 2 * a.G, s, a);
}
static bool gn_vec(const GnArgs& a, int in, int out) {
    const size_t mi = in ? 7 : 15, mo = out ? 7 : 15;
    return a.C % 4 == 0 && !(((size_t)a.x | (size_t)a.dx) & mi) && !(((size_t)a.y | (size_t)a.dy) & mo);
}
#define GN_DISPATCH(FN)                                                                                              \
    do {                                                                                                             \
        const bool vec = gn_vec(a, x_dtype, y_dtype);                                                                \
        if (x_dtype == 0 && y_dtype == 0) { if (vec) FN<float, float, 4>(a, s); else FN<float, float, 1>(a, s); }     \
        else if (x_dtype == 0) { if (vec) FN<float, bf16_t, 4>(a, s); else FN<float, bf16_t, 1>(a, s); }              \
        else if (y_dtype == 0) { if (vec) FN<bf16_t, float, 4>(a, s); else FN<bf16_t, float, 1>(a, s); }              \
        else { if (vec) FN<bf16_t, bf16_t, 4>(a, s); else FN<bf16_t, bf16_t, 1>(a, s); }                              \
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
    GN_DISPATCH(gn_fwd_launch);
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
    GN_DISPATCH(gn_bwd_launch);
    if (dgamma || dbeta) {
        const int rows = a.B * a.nch;
        float* tmp = a.cpart + (size_t)rows * 2 * a.Cp;
        if (dgamma) rows_fold(a.cpart, rows, a.Cp, 1, dgamma, nullptr, C, 0, 0, tmp, s, nullptr, 2 * a.Cp);
        if (dbeta) rows_fold(a.cpart + a.Cp, rows, a.Cp, 1, dbeta, nullptr, C, 0, 0, tmp, s, nullptr, 2 * a.Cp);
    }
    return l2i_check_launch();
}
