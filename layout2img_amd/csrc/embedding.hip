// Embedding lookup with scaling, and its gradient by sorted tokens.
//
//   out[i] = scale * W[t_i]           dW[v] = scale * sum over the i with t_i = v of dy[i]
// A token outside [0, V), or equal to the padding index, gives a row of zeros and has no gradient.
//
// Lookup: bound by bytes (a row read, a row written). Gradient: V rows of D values are written, most of them zeros for a large
// vocabulary, and n rows of dy are read once in the order of their tokens: (token, position) pairs are sorted stably, so that the rows
// of a token are added in the order of their positions, by ONE writer -- no float atomics, the same bits on every run.
#include "common.h"

// ------------------------------------------------------------------------------------------------ lookup
struct EmbArgs {
    const void* w; const long long* tok; void* out;
    long long n; int V, D, pad; float scale;
    int tx;   // lanes along a row: a power of two
};

template <typename TI, typename TO, bool VEC>
__global__ __launch_bounds__(256) void embedding_fwd_kernel(EmbArgs p) {
    const int tx = threadIdx.x & (p.tx - 1), ty = threadIdx.x / p.tx, rows = 256 / p.tx;
    const long long i = (long long)blockIdx.x * rows + ty;
    if (i >= p.n) return;
    const long long t = p.tok[i];
    const bool there = t >= 0 && t < p.V && t != p.pad;
    const TI* src = reinterpret_cast<const TI*>(p.w) + (size_t)(there ? t : 0) * p.D;
    TO* dst = reinterpret_cast<TO*>(p.out) + (size_t)i * p.D;
    constexpr int E = VEC ? 4 : 1;
    for (int c = tx * E; c < p.D; c += p.tx * E) {
        if (VEC) {
            float v[4] = {0.f, 0.f, 0.f, 0.f};
            if (there) Op4<TI>::load(src + c, v);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = there ? v[e] * p.scale : 0.f;
            Op4<TO>::store(dst + c, v);
        } else {
            dst[c] = OpT<TO>::from(there ? OpT<TI>::to(src[c]) * p.scale : 0.f);
        }
    }
}

// ------------------------------------------------------------------------------------------------ sort
// The rank of pair i is the number of pairs in front of it: those with a smaller key, and those with the same key at a smaller position.
// Counting it directly is n^2 comparisons and one launch. A workgroup ranks 64 pairs: each of its four waves counts over a quarter of
// every tile of 1024 keys that the workgroup stages in LDS.
__device__ __forceinline__ int emb_key(long long t, int V, int pad) { return (t >= 0 && t < V && t != pad) ? (int)t : V; }

__global__ __launch_bounds__(256) void embedding_rank_kernel(const long long* __restrict__ tok, int n, int V, int pad, int* __restrict__ skey, int* __restrict__ spos) {
    __shared__ __attribute__((aligned(16))) int keys[1024];
    __shared__ int cnt[4][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = blockIdx.x * 64 + lane;
    const int me = i < n ? emb_key(tok[i], V, pad) : 0x7fffffff;
    int rank = 0;
    for (int base = 0; base < n; base += 1024) {
        __syncthreads();
        for (int k = threadIdx.x; k < 1024; k += 256) keys[k] = base + k < n ? emb_key(tok[base + k], V, pad) : 0x7fffffff;
        __syncthreads();
        const int b0 = base + wave * 256;
        const int4* q = reinterpret_cast<const int4*>(keys + wave * 256);
        if (b0 + 256 <= i - lane) {          // all in front of this workgroup's pairs: equal keys count
            for (int k = 0; k < 64; ++k) { const int4 a = q[k]; rank += (a.x <= me) + (a.y <= me) + (a.z <= me) + (a.w <= me); }
        } else if (b0 >= i - lane + 64) {    // all behind them
            for (int k = 0; k < 64; ++k) { const int4 a = q[k]; rank += (a.x < me) + (a.y < me) + (a.z < me) + (a.w < me); }
        } else {
            for (int k = 0; k < 64; ++k) {
                const int4 a = q[k];
                const int j = b0 + 4 * k;
                rank += (a.x < me || (a.x == me && j < i)) + (a.y < me || (a.y == me && j + 1 < i)) + (a.z < me || (a.z == me && j + 2 < i)) +
                        (a.w < me || (a.w == me && j + 3 < i));
            }
        }
    }
    cnt[wave][lane] = rank;
    __syncthreads();
    if (wave == 0 && i < n) {
        const int r = cnt[0][lane] + cnt[1][lane] + cnt[2][lane] + cnt[3][lane];
        skey[r] = me;
        spos[r] = i;
    }
}

// Above EMB_RANK_MAX pairs: a stable radix sort, eight bits a pass from the lowest, three launches a pass. A workgroup owns 2048
// consecutive pairs, a wave 512 of them; hist[digit][workgroup] counts, its exclusive scan is where each workgroup's pairs of a digit go.
#define EMB_RANK_MAX 8192
#define EMB_TILE 2048
struct EmbSortArgs {
    const long long* tok; const int* kin; const int* pin; int* kout; int* pout; int* hist;
    int n, V, pad, shift, nblk;
};
__device__ __forceinline__ int emb_sort_key(const EmbSortArgs& p, int i) { return p.tok ? emb_key(p.tok[i], p.V, p.pad) : p.kin[i]; }

__global__ __launch_bounds__(256) void embedding_hist_kernel(EmbSortArgs p) {
    __shared__ int h[256];
    h[threadIdx.x] = 0;
    __syncthreads();
    for (int k = threadIdx.x; k < EMB_TILE; k += 256) {
        const int i = blockIdx.x * EMB_TILE + k;
        if (i < p.n) atomicAdd(&h[(emb_sort_key(p, i) >> p.shift) & 255], 1);   // (integers: the order does not matter)
    }
    __syncthreads();
    p.hist[(size_t)threadIdx.x * p.nblk + blockIdx.x] = h[threadIdx.x];
}
// exclusive scan of m integers in place by one workgroup of 1024
__global__ __launch_bounds__(1024) void embedding_scan_kernel(int* __restrict__ a, int m) {
    __shared__ int wtot[16];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int carry = 0;
    for (int base = 0; base < m; base += 1024) {
        const int i = base + (int)threadIdx.x;
        const int v = i < m ? a[i] : 0;
        int s = v;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) { const int t = __shfl_up(s, o, 64); if (lane >= o) s += t; }
        if (lane == 63) wtot[wave] = s;
        __syncthreads();
        int off = carry, tot = 0;
        for (int w = 0; w < 16; ++w) { const int t = wtot[w]; if (w < wave) off += t; tot += t; }
        if (i < m) a[i] = off + s - v;
        carry += tot;
        __syncthreads();
    }
}
__global__ __launch_bounds__(256) void embedding_scatter_kernel(EmbSortArgs p) {
    __shared__ int at[4][256];   // where the wave's next pair of a digit goes
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int k = threadIdx.x; k < 1024; k += 256) (&at[0][0])[k] = 0;
    __syncthreads();
    const int base = blockIdx.x * EMB_TILE + wave * 512;
    int key[8];
#pragma unroll
    for (int r = 0; r < 8; ++r) {
        const int i = base + r * 64 + lane;
        key[r] = i < p.n ? emb_sort_key(p, i) : -1;
        if (i < p.n) atomicAdd(&at[wave][(key[r] >> p.shift) & 255], 1);
    }
    __syncthreads();
    {
        int s = p.hist[(size_t)threadIdx.x * p.nblk + blockIdx.x];
        for (int w = 0; w < 4; ++w) { const int t = at[w][threadIdx.x]; at[w][threadIdx.x] = s; s += t; }
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < 8; ++r) {
        const int i = base + r * 64 + lane;
        const bool on = i < p.n;
        const int d = on ? (key[r] >> p.shift) & 255 : 0;
        unsigned long long same = __ballot(on);
#pragma unroll
        for (int b = 0; b < 8; ++b) {
            const bool bit = (d >> b) & 1;
            const unsigned long long m = __ballot(on && bit);
            same &= bit ? m : ~m;
        }
        const int before = __popcll(same & ((1ull << lane) - 1ull));
        int dst = 0;
        if (on) dst = at[wave][d] + before;
        __builtin_amdgcn_wave_barrier();
        if (on && before == 0) at[wave][d] += __popcll(same);   // (the first lane of a digit; the wave runs in step, its LDS accesses in order)
        __builtin_amdgcn_wave_barrier();
        if (on) { p.kout[dst] = key[r]; p.pout[dst] = p.pin ? p.pin[i] : i; }
    }
}

// ------------------------------------------------------------------------------------------------ gradient rows
// The sorted pairs are cut in chunks of EMB_CHUNK. A chunk whose pairs all carry one token is added up by embedding_part_kernel (so that
// a token which half of the batch carries is summed by many workgroups); embedding_rows_kernel owns the rows of dW, adds the partial rows
// of the chunks inside a token's range and the single rows at its two ends, and writes the row -- zeros where the range is empty.
#define EMB_CHUNK 32
#define EMB_VROWS 16   // rows of dW per workgroup
struct EmbBwdArgs {
    const int* skey; const int* spos; const void* dy; float* part; void* dw;
    int n, V, D; float scale;
    int tx;
};

template <typename T, bool VEC>
__device__ __forceinline__ void emb_add(const T* __restrict__ src, float (&s)[4]) {
    if (VEC) {
        float v[4];
        Op4<T>::load(src, v);
#pragma unroll
        for (int e = 0; e < 4; ++e) s[e] += v[e];
    } else {
        s[0] += OpT<T>::to(src[0]);
    }
}

template <typename TO, bool VEC>
__global__ __launch_bounds__(256) void embedding_part_kernel(EmbBwdArgs p) {
    const int c0 = blockIdx.x, base = c0 * EMB_CHUNK;   // (whole chunks only)
    const int k = p.skey[base];
    if (k >= p.V || k != p.skey[base + EMB_CHUNK - 1]) return;
    constexpr int E = VEC ? 4 : 1;
    for (int c = threadIdx.x * E; c < p.D; c += 256 * E) {
        float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
        for (int j = 0; j < EMB_CHUNK; ++j) emb_add<TO, VEC>(reinterpret_cast<const TO*>(p.dy) + (size_t)p.spos[base + j] * p.D + c, s);
        float* d = p.part + (size_t)c0 * p.D + c;
        if (VEC) *reinterpret_cast<float4*>(d) = make_float4(s[0], s[1], s[2], s[3]);
        else *d = s[0];
    }
}

// the first sorted pair whose key is >= v: every lane of the wave probes, 64 places a step
__device__ __forceinline__ int emb_lower_bound(const int* __restrict__ skey, int n, int v) {
    const int lane = threadIdx.x & 63;
    int lo = 0, hi = n;   // the answer lies in [lo, hi]
    while (lo < hi) {
        const int step = (hi - lo + 63) / 64;
        const long long at = (long long)lo + (long long)step * (lane + 1) - 1;   // the last pair of the lane's piece
        const bool below = at < hi && skey[at] < v;
        const int full = __popcll(__ballot(below));                              // pieces that lie below v as a whole
        lo = lo + full * step < hi ? lo + full * step : hi;
        hi = lo + step - 1 < hi ? lo + step - 1 : hi;
    }
    return lo;
}

template <typename TO, typename TW, bool VEC>
__global__ __launch_bounds__(256) void embedding_rows_kernel(EmbBwdArgs p) {
    __shared__ int first[EMB_VROWS + 1];
    const int v0 = blockIdx.x * EMB_VROWS, wave = threadIdx.x >> 6;
    for (int r = wave; r <= EMB_VROWS; r += 4) {
        const int a = emb_lower_bound(p.skey, p.n, min(v0 + r, p.V));
        if ((threadIdx.x & 63) == 0) first[r] = a;
    }
    __syncthreads();
    const int tx = threadIdx.x & (p.tx - 1), ty = threadIdx.x / p.tx, nr = 256 / p.tx;
    constexpr int E = VEC ? 4 : 1;
    const TO* dy = reinterpret_cast<const TO*>(p.dy);
    for (int r = ty; r < EMB_VROWS && v0 + r < p.V; r += nr) {
        const int a = first[r], b = first[r + 1];
        const int ca = (a + EMB_CHUNK - 1) / EMB_CHUNK, cb = b / EMB_CHUNK;   // whole chunks inside [a, b): [ca, cb)
        TW* dst = reinterpret_cast<TW*>(p.dw) + (size_t)(v0 + r) * p.D;
        for (int c = tx * E; c < p.D; c += p.tx * E) {
            float s[4] = {0.f, 0.f, 0.f, 0.f};
            if (ca < cb) {
                for (int j = a; j < ca * EMB_CHUNK; ++j) emb_add<TO, VEC>(dy + (size_t)p.spos[j] * p.D + c, s);
                for (int j = ca; j < cb; ++j) emb_add<float, VEC>(p.part + (size_t)j * p.D + c, s);
                for (int j = cb * EMB_CHUNK; j < b; ++j) emb_add<TO, VEC>(dy + (size_t)p.spos[j] * p.D + c, s);
            } else {
                for (int j = a; j < b; ++j) emb_add<TO, VEC>(dy + (size_t)p.spos[j] * p.D + c, s);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) s[e] *= p.scale;
            if (VEC) Op4<TW>::store(dst + c, s);
            else dst[c] = OpT<TW>::from(s[0]);
        }
    }
}

// ------------------------------------------------------------------------------------------------ entry points
static int emb_lanes(int D, int E) {
    int tx = 1;
    while (tx < 256 && tx * E < D) tx <<= 1;
    return tx;
}
template <typename TI, typename TO>
static void emb_fwd_launch(EmbArgs a, hipStream_t s) {
    const bool vec = a.D % 4 == 0 && !((size_t)a.w & (4 * sizeof(TI) - 1)) && !((size_t)a.out & (4 * sizeof(TO) - 1));
    a.tx = emb_lanes(a.D, vec ? 4 : 1);
    const unsigned grid = (unsigned)((a.n + 256 / a.tx - 1) / (256 / a.tx));
    if (vec) hipLaunchKernelGGL((embedding_fwd_kernel<TI, TO, true>), dim3(grid), dim3(256), 0, s, a);
    else hipLaunchKernelGGL((embedding_fwd_kernel<TI, TO, false>), dim3(grid), dim3(256), 0, s, a);
}
extern "C" int l2i_embedding_fwd(const void* weight, int w_dtype, const long long* tokens, void* out, int out_dtype, long long n, int V, int D,
                                 float scale, int padding_idx, void* stream) {
    if (n < 0 || n > 0x7fffffffLL || V < 1 || V > 0x7fffff00 || D < 1 || D > 65536 || (w_dtype | out_dtype) & ~1) return L2I_ERR_ARG;
    if (n == 0) return L2I_OK;
    if (!weight || !tokens || !out) return L2I_ERR_ARG;
    EmbArgs a;
    a.w = weight; a.tok = tokens; a.out = out; a.n = n; a.V = V; a.D = D; a.pad = padding_idx; a.scale = scale; a.tx = 0;
    hipStream_t s = (hipStream_t)stream;
    if (w_dtype == 0) { if (out_dtype == 0) emb_fwd_launch<float, float>(a, s); else emb_fwd_launch<float, bf16_t>(a, s); }
    else { if (out_dtype == 0) emb_fwd_launch<bf16_t, float>(a, s); else emb_fwd_launch<bf16_t, bf16_t>(a, s); }
    return l2i_check_launch();
}

// scratch, in ints: sorted keys and positions [n] each, a second pair of them and the histogram when the radix sort runs, then the partial rows
static long long emb_al(long long ints) { return (ints + 3) & ~3LL; }
static long long emb_hist_ints(long long n) { return 256 * ((n + EMB_TILE - 1) / EMB_TILE); }
extern "C" int l2i_embedding_bwd_scratch(long long n, int D, long long* floats) {
    if (!floats || n < 0 || n > 0x7fffffffLL || D < 1) return L2I_ERR_ARG;
    *floats = emb_al(n) * (n > EMB_RANK_MAX ? 4 : 2) + (n > EMB_RANK_MAX ? emb_al(emb_hist_ints(n)) : 0) + (n / EMB_CHUNK) * (long long)D;
    return L2I_OK;
}

template <typename TO, typename TW>
static void emb_bwd_launch(EmbBwdArgs a, hipStream_t s) {
    const bool vec = a.D % 4 == 0 && !((size_t)a.dy & (4 * sizeof(TO) - 1)) && !((size_t)a.dw & (4 * sizeof(TW) - 1));
    a.tx = emb_lanes(a.D, vec ? 4 : 1);
    const unsigned grid = (unsigned)((a.V + EMB_VROWS - 1) / EMB_VROWS), nch = (unsigned)(a.n / EMB_CHUNK);
    if (vec) {
        if (nch) hipLaunchKernelGGL((embedding_part_kernel<TO, true>), dim3(nch), dim3(256), 0, s, a);
        hipLaunchKernelGGL((embedding_rows_kernel<TO, TW, true>), dim3(grid), dim3(256), 0, s, a);
    } else {
        if (nch) hipLaunchKernelGGL((embedding_part_kernel<TO, false>), dim3(nch), dim3(256), 0, s, a);
        hipLaunchKernelGGL((embedding_rows_kernel<TO, TW, false>), dim3(grid), dim3(256), 0, s, a);
    }
}
extern "C" int l2i_embedding_bwd(const long long* tokens, const void* dy, int dy_dtype, void* dw, int dw_dtype, long long n, int V, int D, float scale,
                                 int padding_idx, float* scratch, long long scratch_floats, void* stream) {
    if (n < 0 || n > 0x7fffffffLL - EMB_TILE || V < 1 || V > 0x7fffff00 || D < 1 || D > 65536 || (dy_dtype | dw_dtype) & ~1) return L2I_ERR_ARG;
    if (!dw || (n && (!tokens || !dy || !scratch || ((size_t)scratch & 15)))) return L2I_ERR_ARG;
    long long need = 0;
    if (l2i_embedding_bwd_scratch(n, D, &need) != L2I_OK || (n && scratch_floats < need)) return L2I_ERR_ARG;
    hipStream_t s = (hipStream_t)stream;
    int* skey = reinterpret_cast<int*>(scratch);
    int* spos = skey + emb_al(n);
    int* end = spos + emb_al(n);
    if (n > EMB_RANK_MAX) {
        int *k2 = end, *p2 = k2 + emb_al(n), *hist = p2 + emb_al(n);
        end = hist + emb_al(emb_hist_ints(n));
        int bits = 1;
        while (bits < 31 && (V >> bits)) ++bits;   // keys 0 .. V
        const int passes = (bits + 7) / 8;
        EmbSortArgs a;
        a.n = (int)n; a.V = V; a.pad = padding_idx; a.hist = hist; a.nblk = (int)((n + EMB_TILE - 1) / EMB_TILE);
        for (int q = 0; q < passes; ++q) {   // the last pass writes skey / spos
            const bool to_first = (passes - 1 - q) % 2 == 0;
            a.tok = q == 0 ? tokens : nullptr;
            a.kin = to_first ? k2 : skey; a.pin = q == 0 ? nullptr : (to_first ? p2 : spos);
            a.kout = to_first ? skey : k2; a.pout = to_first ? spos : p2;
            a.shift = 8 * q;
            hipLaunchKernelGGL(embedding_hist_kernel, dim3(a.nblk), dim3(256), 0, s, a);
            hipLaunchKernelGGL(embedding_scan_kernel, dim3(1), dim3(1024), 0, s, hist, 256 * a.nblk);
            hipLaunchKernelGGL(embedding_scatter_kernel, dim3(a.nblk), dim3(256), 0, s, a);
        }
    } else if (n) {
        hipLaunchKernelGGL(embedding_rank_kernel, dim3((unsigned)((n + 63) / 64)), dim3(256), 0, s, tokens, (int)n, V, padding_idx, skey, spos);
    }
    EmbBwdArgs b;
    b.skey = skey; b.spos = spos; b.dy = dy; b.part = reinterpret_cast<float*>(end); b.dw = dw; b.n = (int)n; b.V = V; b.D = D; b.scale = scale; b.tx = 0;
    if (dy_dtype == 0) { if (dw_dtype == 0) emb_bwd_launch<float, float>(b, s); else emb_bwd_launch<float, bf16_t>(b, s); }
    else { if (dw_dtype == 0) emb_bwd_launch<bf16_t, float>(b, s); else emb_bwd_launch<bf16_t, bf16_t>(b, s); }
    return l2i_check_launch();
}
