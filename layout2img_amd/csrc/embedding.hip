// Embedding lookup with scaling, and its gradient by sorted tokens.
//
//   out[i] = scale * W[t_i]           dW[v] = scale * sum over the i with t_i = v of dy[i]
// A token outside [0, V), or equal to the padding index, gives a row of zeros and has no gradient.
//
// Lookup: bound by bytes (a row read, a row written). Gradient: V rows of D values are written, most of them zeros for a large
// vocabulary, and n rows of dy are read once in the order of their tokens: (token, position) pairs are sorted stably, so that the rows
// of a token are added in the order of their positions, by ONE writer -- no float atomics, the same bits on every run.
// Measured, 16384 skewed tokens of a 32000 x 1024 table in bf16: lookup 11 us (6.0 TB/s), sort 16, rows in the order of their tokens 15, the rest of
// dW 19 (65 MB written).
#include "vec.h"

// ------------------------------------------------------------------------------------------------ lookup
struct EmbArgs {
    const void* w; const long long* tok; void* out;
    long long n; int V, D, pad; float scale;
    int tx;   // lanes along a row: a power of two
};

template <typename TI, typename TO, int V>
__global__ __launch_bounds__(256) void embedding_fwd_kernel(EmbArgs p) {
    const int tx = threadIdx.x & (p.tx - 1), ty = threadIdx.x / p.tx, rows = 256 / p.tx;
    const long long i = (long long)blockIdx.x * rows + ty;
    if (i >= p.n) return;
    const long long t = p.tok[i];
    const bool there = t >= 0 && t < p.V && t != p.pad;
    const TI* src = reinterpret_cast<const TI*>(p.w) + (size_t)(there ? t : 0) * p.D;
    TO* dst = reinterpret_cast<TO*>(p.out) + (size_t)i * p.D;
    for (int c = tx * V; c < p.D; c += p.tx * V) {
        Vec<TI, V> a;
        float v[V];
        a.load(src + c);
        a.get(v);
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] = there ? v[e] * p.scale : 0.f;
        vec_store<TO, V>(dst + c, v);
    }
}

// ------------------------------------------------------------------------------------------------ gradient of a few rows
// Up to EMB_DIRECT pairs (the labels of a batch of layouts) need no sort: a workgroup owns a row of dW, its four waves look through a quarter of the
// pairs each, in order, add the rows they find and are joined in order. One launch and no scratch (the sorted form takes three and 13 us at 256
// labels of a 184 x 180 table; this one 4).
#define EMB_DIRECT 1024
struct EmbDirectArgs { const long long* tok; const void* dy; void* dw; int n, V, D, pad; float scale; };

template <typename TO, typename TW, int V>
__global__ __launch_bounds__(256) void embedding_direct_kernel(EmbDirectArgs p) {
    __shared__ float red[3][64 * V];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, quarter = (p.n + 3) / 4;
    const int j0 = wave * quarter, j1 = min(p.n, j0 + quarter);
    const long long v = blockIdx.x;
    const TO* dy = reinterpret_cast<const TO*>(p.dy);
    unsigned long long hit[EMB_DIRECT / 4 / 64];
    int any = 0;
#pragma unroll
    for (int k = 0; k < EMB_DIRECT / 4 / 64; ++k) {
        const int j = j0 + 64 * k + lane;
        hit[k] = __ballot(j < j1 && p.tok[j] == v && v != p.pad);
        any |= hit[k] != 0;
    }
    const bool found = __syncthreads_or(any);
    for (int c0 = 0; c0 < p.D; c0 += 64 * V) {
        const int c = c0 + lane * V;
        const bool on = c < p.D;
        float s[V];
#pragma unroll
        for (int e = 0; e < V; ++e) s[e] = 0.f;
        if (found) {
#pragma unroll
            for (int k = 0; k < EMB_DIRECT / 4 / 64; ++k) {
                unsigned long long m = hit[k];
                while (m) {   // four rows in flight, added in order
                    Vec<TO, V> a[4];
                    int got = 0;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        if (!m) break;
                        const int j = j0 + 64 * k + __ffsll((unsigned long long)m) - 1;
                        m &= m - 1;
                        if (on) a[i].load(dy + (size_t)j * p.D + c);
                        ++got;
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        if (i >= got) break;
                        float x[V];
                        if (on) a[i].get(x);
#pragma unroll
                        for (int e = 0; e < V; ++e) s[e] += on ? x[e] : 0.f;
                    }
                }
            }
            __syncthreads();
            if (wave > 0)
#pragma unroll
                for (int e = 0; e < V; ++e) red[wave - 1][e * 64 + lane] = s[e];
            __syncthreads();
        }
        if (wave == 0 && on) {
#pragma unroll
            for (int e = 0; e < V; ++e) {
                if (found) s[e] = ((s[e] + red[0][e * 64 + lane]) + red[1][e * 64 + lane]) + red[2][e * 64 + lane];
                s[e] *= p.scale;
            }
            vec_store<TW, V>(reinterpret_cast<TW*>(p.dw) + (size_t)v * p.D + c, s);
        }
    }
}

// ------------------------------------------------------------------------------------------------ sort
// The rank of pair i is the number of pairs in front of it: those with a smaller key, and those with the same key at a smaller position.
// Counting it directly is n^2 comparisons and one launch: what up to EMB_RANK_MAX pairs take (lookup and gradient of 4096 rows of 512 in a table of
// 32000: 43 us, with the radix sort 46; even at 6000 pairs; 49 and 45 at 8192). A workgroup ranks 64 pairs: each of its NW waves counts over its share of
// every tile of 256 NW keys that the workgroup stages in LDS (four waves up to 2048 pairs, sixteen above: four a SIMD hide the LDS reads).
// The sort's first launch also marks every row of dW as absent (range[v] = (-1, 0)); the next kernel fills in the tokens that occur.
__device__ __forceinline__ int emb_key(long long t, int V, int pad) { return (t >= 0 && t < V && t != pad) ? (int)t : V; }
__device__ __forceinline__ void emb_clear(int2* range, int V) {
    for (long long v = (long long)blockIdx.x * blockDim.x + threadIdx.x; v < V; v += (long long)gridDim.x * blockDim.x) range[v] = make_int2(-1, 0);
}

template <int NW>
__global__ __launch_bounds__(NW * 64) void embedding_rank_kernel(const long long* __restrict__ tok, int n, int V, int pad, int* __restrict__ skey,
                                                                 int* __restrict__ spos, int2* __restrict__ range) {
    __shared__ __attribute__((aligned(16))) int keys[256 * NW];
    __shared__ int cnt[NW][64];
    emb_clear(range, V);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i0 = blockIdx.x * 64, i = i0 + lane;
    if (i0 >= n) return;   // (a workgroup that only clears)
    const int me = i < n ? emb_key(tok[i], V, pad) : 0x7fffffff;
    int c0 = 0, c1 = 0, c2 = 0, c3 = 0;
    for (int base = 0; base < n; base += 256 * NW) {
        const int m = min(256 * NW, n - base), q4 = (m + 4 * NW - 1) / (4 * NW);   // groups of four keys a wave
        __syncthreads();
        for (int k = threadIdx.x; k < 4 * NW * q4; k += 64 * NW) keys[k] = k < m ? emb_key(tok[base + k], V, pad) : 0x7fffffff;
        __syncthreads();
        const int b0 = base + wave * 4 * q4;
        const int4* q = reinterpret_cast<const int4*>(keys + wave * 4 * q4);
        if (b0 + 4 * q4 <= i0) {          // all in front of this workgroup's pairs: equal keys count
#pragma unroll 8
            for (int k = 0; k < q4; ++k) { const int4 a = q[k]; c0 += a.x <= me; c1 += a.y <= me; c2 += a.z <= me; c3 += a.w <= me; }
        } else if (b0 >= i0 + 64) {       // all behind them
#pragma unroll 8
            for (int k = 0; k < q4; ++k) { const int4 a = q[k]; c0 += a.x < me; c1 += a.y < me; c2 += a.z < me; c3 += a.w < me; }
        } else {
#pragma unroll 4
            for (int k = 0; k < q4; ++k) {
                const int4 a = q[k];
                const int j = b0 + 4 * k;
                c0 += a.x < me || (a.x == me && j < i); c1 += a.y < me || (a.y == me && j + 1 < i);
                c2 += a.z < me || (a.z == me && j + 2 < i); c3 += a.w < me || (a.w == me && j + 3 < i);
            }
        }
    }
    cnt[wave][lane] = (c0 + c1) + (c2 + c3);
    __syncthreads();
    if (wave == 0 && i < n) {
        int r = 0;
#pragma unroll
        for (int w = 0; w < NW; ++w) r += cnt[w][lane];
        skey[r] = me;
        spos[r] = i;
    }
}

// Above EMB_RANK_MAX pairs: a stable radix sort, eight bits a pass from the lowest. A workgroup owns 256 R consecutive pairs (R: 2, or 8 above
// EMB_FEW pairs), a wave a quarter of them; hist[digit][workgroup] counts, its exclusive scan is where each workgroup's pairs of a digit go. Up to
// EMB_SCAN workgroups each of them scans the counts by itself, above that a launch of its own does (262144 rows of 512, lookup and gradient: 291 us with
// that launch, 237 without). Sizes: 16384 pairs are sorted by the four launches of two passes in 16 us (a rank by n^2 comparisons: 29), 8192 the same.
#define EMB_RANK_MAX 6144
#define EMB_FEW 32768
#define EMB_SCAN 256
struct EmbSortArgs {
    const long long* tok; const int* kin; const int* pin; int* kout; int* pout; int* hist; int2* range;   // range: first pass only
    int n, V, pad, shift, nblk, scanned;
};
__device__ __forceinline__ int emb_sort_key(const EmbSortArgs& p, int i) { return p.tok ? emb_key(p.tok[i], p.V, p.pad) : p.kin[i]; }

template <int R>
__global__ __launch_bounds__(256) void embedding_hist_kernel(EmbSortArgs p) {
    __shared__ int h[256];
    if (p.range) emb_clear(p.range, p.V);
    h[threadIdx.x] = 0;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < R; ++k) {
        const int i = (blockIdx.x * R + k) * 256 + threadIdx.x;
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
template <int R>
__global__ __launch_bounds__(256) void embedding_scatter_kernel(EmbSortArgs p) {
    __shared__ int at[4][256];   // where the wave's next pair of a digit goes
    __shared__ int wtot[4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int w = 0; w < 4; ++w) at[w][threadIdx.x] = 0;
    __syncthreads();
    const int base = blockIdx.x * 256 * R + wave * 64 * R;
    int key[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int i = base + r * 64 + lane;
        key[r] = i < p.n ? emb_sort_key(p, i) : -1;
        if (i < p.n) atomicAdd(&at[wave][(key[r] >> p.shift) & 255], 1);
    }
    int s;
    if (p.scanned) {
        s = p.hist[(size_t)threadIdx.x * p.nblk + blockIdx.x];
        __syncthreads();
    } else {   // thread d: this digit's pairs in the workgroups in front of this one, and the pairs of all smaller digits
        const int* row = p.hist + (size_t)threadIdx.x * p.nblk;
        int tot = 0;
        s = 0;
#pragma unroll 16
        for (int k = 0; k < p.nblk; ++k) { const int t = row[k]; tot += t; s += k < (int)blockIdx.x ? t : 0; }
        int run = tot;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) { const int t = __shfl_up(run, o, 64); if (lane >= o) run += t; }
        if (lane == 63) wtot[wave] = run;
        __syncthreads();
        s += run - tot;
        for (int w = 0; w < wave; ++w) s += wtot[w];
    }
#pragma unroll
    for (int w = 0; w < 4; ++w) { const int t = at[w][threadIdx.x]; at[w][threadIdx.x] = s; s += t; }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < R; ++r) {
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
// The sorted pairs are cut in chunks. embedding_part_kernel walks a chunk: the tokens that lie in it as a whole are finished there (their
// row of dW is written), the run that came in from the chunk before and the run that goes on in the next are left as partial rows, so that
// every chunk costs the same however skewed the tokens are. embedding_rows_kernel owns the other rows of dW: it adds a token's partial
// rows in chunk order, or writes zeros where the token does not occur.
#define EMB_VROWS 8   // rows of dW per workgroup
struct EmbBwdArgs {
    const int* skey; const int* spos; int2* range /* [V]: a token's pairs [x, y); x = -1: none */; const void* dy;
    float* part /* [chunks][2][D]: come in, go on */; void* dw;
    int n, V, D, chunk, nch; float scale;
    int tx;   // lanes along a row: a power of two
    int v0;   // first row of the launch (embedding_rows_kernel)
};

template <typename TO, typename TW, int V>
__global__ __launch_bounds__(256) void embedding_part_kernel(EmbBwdArgs p) {
    const int tx = threadIdx.x & (p.tx - 1), c = blockIdx.x * (256 / p.tx) + threadIdx.x / p.tx;
    if (c >= p.nch) return;
    const int base = c * p.chunk, m = min(p.chunk, p.n - base);
    const int before = base > 0 ? p.skey[base - 1] : -1, behind = base + m < p.n ? p.skey[base + m] : -1;
    const TO* dy = reinterpret_cast<const TO*>(p.dy);
    for (int col = tx * V; col < p.D; col += p.tx * V) {
        float s[V];
#pragma unroll
        for (int e = 0; e < V; ++e) s[e] = 0.f;
        bool in = p.skey[base] == before;
        int prev = before;
        for (int j0 = 0; j0 < m; j0 += 8) {
            Vec<TO, V> a[8];
            int key[9];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int at = base + min(j0 + j, m - 1);
                key[j] = p.skey[at];
                a[j].load(dy + (size_t)p.spos[at] * p.D + col);
            }
            key[8] = j0 + 8 < m ? p.skey[base + j0 + 8] : -1;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                if (j0 + j >= m) break;
                float v[V];
                a[j].get(v);
#pragma unroll
                for (int e = 0; e < V; ++e) s[e] += v[e];
                const bool last = j0 + j == m - 1;
                const int next = last ? behind : key[j + 1];
                if (tx == 0 && col == 0 && key[j] < p.V) {
                    if (prev != key[j]) p.range[key[j]].x = base + j0 + j;
                    if (next != key[j]) p.range[key[j]].y = base + j0 + j + 1;
                }
                prev = key[j];
                if (next == key[j] && !last) continue;
                // the run ends here, or the chunk does
                if (key[j] < p.V) {
                    if (in || next == key[j]) {
                        vec_store<float, V>(p.part + ((size_t)c * 2 + (in ? 0 : 1)) * p.D + col, s);
                    } else {
#pragma unroll
                        for (int e = 0; e < V; ++e) s[e] *= p.scale;
                        vec_store<TW, V>(reinterpret_cast<TW*>(p.dw) + (size_t)key[j] * p.D + col, s);
                    }
                }
                in = false;
#pragma unroll
                for (int e = 0; e < V; ++e) s[e] = 0.f;
            }
        }
    }
}

template <typename TW, int V>
__global__ __launch_bounds__(256) void embedding_rows_kernel(EmbBwdArgs p) {
    __shared__ int ra[EMB_VROWS], rk[EMB_VROWS];   // first chunk of a row and chunks it runs through; 0: absent, 1: finished
    __shared__ float red[256 * V];
    const int v0 = p.v0 + blockIdx.x * EMB_VROWS, nv = min(EMB_VROWS, p.V - v0);
    if ((int)threadIdx.x < nv) {
        const int2 a = p.n ? p.range[v0 + threadIdx.x] : make_int2(-1, 0);
        ra[threadIdx.x] = a.x / p.chunk;
        rk[threadIdx.x] = a.x < 0 ? 0 : (a.y - 1) / p.chunk - a.x / p.chunk + 1;
    }
    __syncthreads();
    const int tx = threadIdx.x & (p.tx - 1), ty = threadIdx.x / p.tx, nr = 256 / p.tx;
    TW* dw = reinterpret_cast<TW*>(p.dw) + (size_t)v0 * p.D;
    float s[V];
    auto add = [&](int ca, int c, int j0, int k, int step) {   // partial rows j0, j0 + step, ... of k from chunk ca on: the first went on from its chunk, the others came in
#pragma unroll
        for (int e = 0; e < V; ++e) s[e] = 0.f;
#pragma unroll 8
        for (int j = j0; j < k; j += step) {
            Vec<float, V> t;
            float v[V];
            t.load(p.part + ((size_t)(ca + j) * 2 + (j == 0 ? 1 : 0)) * p.D + c);
            t.get(v);
#pragma unroll
            for (int e = 0; e < V; ++e) s[e] += v[e];
        }
    };
    auto put = [&](int r, int c) {
#pragma unroll
        for (int e = 0; e < V; ++e) s[e] *= p.scale;
        vec_store<TW, V>(dw + (size_t)r * p.D + c, s);
    };
    bool many = false;
    for (int r = 0; r < nv; ++r) many = many || rk[r] > 32;
    for (int r = ty; r < nv; r += nr) {
        const int k = rk[r];
        if (k == 1 || k > 32) continue;
        for (int c = tx * V; c < p.D; c += p.tx * V) { add(ra[r], c, 0, k, 1); put(r, c); }
    }
    if (!many) return;
    for (int r = 0; r < nv; ++r) {   // a token of many chunks: the whole workgroup, every nr-th partial row a lane, joined in lane order
        const int k = rk[r];
        if (k <= 32) continue;
        for (int c0 = 0; c0 < p.D; c0 += p.tx * V) {
            const int c = c0 + tx * V;
            if (c < p.D) add(ra[r], c, ty, k, nr);
            __syncthreads();
            if (c < p.D)
#pragma unroll
                for (int e = 0; e < V; ++e) red[e * 256 + threadIdx.x] = s[e];
            __syncthreads();
            if (ty == 0 && c < p.D) {
                for (int j = 1; j < nr && j < k; ++j)
#pragma unroll
                    for (int e = 0; e < V; ++e) s[e] += red[e * 256 + j * p.tx + tx];
                put(r, c);
            }
        }
    }
}

// ------------------------------------------------------------------------------------------------ entry points
#define EMB_GRID (1LL << 23)   // workgroups of a launch, which has less than 2^32 threads: what takes more is cut
static int emb_lanes(int D, int E) {
    int tx = 1;
    while (tx < 256 && tx * E < D) tx <<= 1;
    return tx;
}
template <typename TI, typename TO>
static void emb_fwd_launch(EmbArgs a, hipStream_t s) {
    const int v = vec_width(a.D, a.w, sizeof(TI) == 2, a.out, sizeof(TO) == 2);
    a.tx = emb_lanes(a.D, v);
    const long long n = a.n, per = 256 / a.tx;
    for (long long i = 0; i < n; i += per * EMB_GRID) {
        a.n = n - i < per * EMB_GRID ? n - i : per * EMB_GRID;
        const dim3 grid((unsigned)((a.n + per - 1) / per));
        if (v == 8) hipLaunchKernelGGL((embedding_fwd_kernel<TI, TO, 8>), grid, dim3(256), 0, s, a);
        else if (v == 4) hipLaunchKernelGGL((embedding_fwd_kernel<TI, TO, 4>), grid, dim3(256), 0, s, a);
        else hipLaunchKernelGGL((embedding_fwd_kernel<TI, TO, 1>), grid, dim3(256), 0, s, a);
        a.tok += per * EMB_GRID;
        a.out = reinterpret_cast<TO*>(a.out) + (size_t)per * EMB_GRID * a.D;
    }
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

// scratch, in ints: sorted keys and positions [n] each, the tokens' ranges [V][2], a second pair of them and the histogram when the radix sort runs, then the partial rows
static int emb_chunk(long long n) { return n <= 2048 ? 8 : n <= 8192 ? 16 : n <= 65536 ? 32 : 128; }   // few pairs: more workgroups; many: fewer partial rows
// every row of dW looks through all pairs: few pairs, and not millions of rows
static bool emb_direct(long long n, int V) { return n <= EMB_DIRECT && n * V <= (1 << 24) && V <= EMB_GRID; }
static long long emb_al(long long ints) { return (ints + 3) & ~3LL; }
static int emb_rounds(long long n) { return n <= EMB_FEW ? 2 : 8; }
static long long emb_blocks(long long n) { return (n + 256 * emb_rounds(n) - 1) / (256 * emb_rounds(n)); }
static long long emb_hist_ints(long long n) { return 256 * emb_blocks(n); }
extern "C" int l2i_embedding_bwd_scratch(long long n, int V, int D, long long* floats) {
    if (!floats || n < 0 || n > 0x7fffffffLL || V < 1 || V > 0x7fffff00 || D < 1 || D > 65536) return L2I_ERR_ARG;
    if (emb_direct(n, V)) { *floats = 0; return L2I_OK; }
    *floats = emb_al(2LL * V) + emb_al(n) * (n > EMB_RANK_MAX ? 4 : 2) + (n > EMB_RANK_MAX ? emb_al(emb_hist_ints(n)) : 0) + (n + emb_chunk(n) - 1) / emb_chunk(n) * 2 * (long long)D;
    return L2I_OK;
}

template <typename TO, typename TW>
static void emb_direct_launch(const EmbDirectArgs& a, hipStream_t s) {
    const int v = vec_width(a.D, a.dy, sizeof(TO) == 2, a.dw, sizeof(TW) == 2);
    if (v == 8) hipLaunchKernelGGL((embedding_direct_kernel<TO, TW, 8>), dim3(a.V), dim3(256), 0, s, a);
    else if (v == 4) hipLaunchKernelGGL((embedding_direct_kernel<TO, TW, 4>), dim3(a.V), dim3(256), 0, s, a);
    else hipLaunchKernelGGL((embedding_direct_kernel<TO, TW, 1>), dim3(a.V), dim3(256), 0, s, a);
}
template <typename TO, typename TW, int V>
static void emb_bwd_kernels(EmbBwdArgs a, hipStream_t s) {
    a.tx = emb_lanes(a.D, V);
    const long long groups = ((long long)a.V + EMB_VROWS - 1) / EMB_VROWS;
    const unsigned per = 256 / a.tx;
    if (a.n) hipLaunchKernelGGL((embedding_part_kernel<TO, TW, V>), dim3((a.nch + per - 1) / per), dim3(256), 0, s, a);
    for (long long i = 0; i < groups; i += EMB_GRID) {
        a.v0 = (int)(i * EMB_VROWS);
        hipLaunchKernelGGL((embedding_rows_kernel<TW, V>), dim3((unsigned)(groups - i < EMB_GRID ? groups - i : EMB_GRID)), dim3(256), 0, s, a);
    }
}
template <typename TO, typename TW>
static void emb_bwd_launch(const EmbBwdArgs& a, hipStream_t s) {
    const int v = vec_width(a.D, a.dy, sizeof(TO) == 2, a.dw, sizeof(TW) == 2);
    if (v == 8) emb_bwd_kernels<TO, TW, 8>(a, s);
    else if (v == 4) emb_bwd_kernels<TO, TW, 4>(a, s);
    else emb_bwd_kernels<TO, TW, 1>(a, s);
}
extern "C" int l2i_embedding_bwd(const long long* tokens, const void* dy, int dy_dtype, void* dw, int dw_dtype, long long n, int V, int D, float scale,
                                 int padding_idx, float* scratch, long long scratch_floats, void* stream) {
    if (n < 0 || n > 0x7fffffffLL - 2048 || V < 1 || V > 0x7fffff00 || D < 1 || D > 65536 || (dy_dtype | dw_dtype) & ~1) return L2I_ERR_ARG;
    if (!dw || (n && (!tokens || !dy))) return L2I_ERR_ARG;
    long long need = 0;
    if (l2i_embedding_bwd_scratch(n, V, D, &need) != L2I_OK) return L2I_ERR_ARG;
    if (need && (!scratch || ((size_t)scratch & 15) || scratch_floats < need)) return L2I_ERR_ARG;
    hipStream_t s = (hipStream_t)stream;
    if (emb_direct(n, V)) {
        EmbDirectArgs a;
        a.tok = tokens; a.dy = dy; a.dw = dw; a.n = (int)n; a.V = V; a.D = D; a.pad = padding_idx; a.scale = scale;
        if (dy_dtype == 0) { if (dw_dtype == 0) emb_direct_launch<float, float>(a, s); else emb_direct_launch<float, bf16_t>(a, s); }
        else { if (dw_dtype == 0) emb_direct_launch<bf16_t, float>(a, s); else emb_direct_launch<bf16_t, bf16_t>(a, s); }
        return l2i_check_launch();
    }
    int* skey = reinterpret_cast<int*>(scratch);
    int* spos = skey + emb_al(n);
    int2* range = reinterpret_cast<int2*>(spos + emb_al(n));
    int* end = reinterpret_cast<int*>(range) + emb_al(2LL * V);
    if (n > EMB_RANK_MAX) {
        int *k2 = end, *p2 = k2 + emb_al(n), *hist = p2 + emb_al(n);
        end = hist + emb_al(emb_hist_ints(n));
        int bits = 1;
        while (bits < 31 && (V >> bits)) ++bits;   // keys 0 .. V
        const int passes = (bits + 7) / 8;
        EmbSortArgs a;
        a.n = (int)n; a.V = V; a.pad = padding_idx; a.hist = hist; a.nblk = (int)emb_blocks(n); a.scanned = a.nblk > EMB_SCAN;
        for (int q = 0; q < passes; ++q) {   // the last pass writes skey / spos
            const bool to_first = (passes - 1 - q) % 2 == 0;
            a.tok = q == 0 ? tokens : nullptr;
            a.kin = to_first ? k2 : skey; a.pin = q == 0 ? nullptr : (to_first ? p2 : spos);
            a.kout = to_first ? skey : k2; a.pout = to_first ? spos : p2;
            a.shift = 8 * q; a.range = q == 0 ? range : nullptr;
            if (emb_rounds(n) == 2) {
                hipLaunchKernelGGL((embedding_hist_kernel<2>), dim3(a.nblk), dim3(256), 0, s, a);
                hipLaunchKernelGGL((embedding_scatter_kernel<2>), dim3(a.nblk), dim3(256), 0, s, a);
            } else {
                hipLaunchKernelGGL((embedding_hist_kernel<8>), dim3(a.nblk), dim3(256), 0, s, a);
                if (a.scanned) hipLaunchKernelGGL(embedding_scan_kernel, dim3(1), dim3(1024), 0, s, hist, 256 * a.nblk);
                hipLaunchKernelGGL((embedding_scatter_kernel<8>), dim3(a.nblk), dim3(256), 0, s, a);
            }
        }
    } else if (n) {
        int grid = (int)((n + 63) / 64);
        const int clear = V / 8192 < 256 ? V / 8192 : 256;
        if (grid < clear) grid = clear;
        if (n <= 2048) hipLaunchKernelGGL((embedding_rank_kernel<4>), dim3(grid), dim3(256), 0, s, tokens, (int)n, V, padding_idx, skey, spos, range);
        else hipLaunchKernelGGL((embedding_rank_kernel<16>), dim3(grid), dim3(1024), 0, s, tokens, (int)n, V, padding_idx, skey, spos, range);
    }
    EmbBwdArgs b;
    b.skey = skey; b.spos = spos; b.range = range; b.dy = dy; b.part = reinterpret_cast<float*>(end); b.dw = dw; b.n = (int)n; b.V = V; b.D = D; b.scale = scale; b.tx = 0; b.v0 = 0;
    b.chunk = emb_chunk(n); b.nch = (int)((n + b.chunk - 1) / b.chunk);
    if (dy_dtype == 0) { if (dw_dtype == 0) emb_bwd_launch<float, float>(b, s); else emb_bwd_launch<float, bf16_t>(b, s); }
    else { if (dw_dtype == 0) emb_bwd_launch<bf16_t, float>(b, s); else emb_bwd_launch<bf16_t, bf16_t>(b, s); }
    return l2i_check_launch();
}
