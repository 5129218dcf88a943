// Attention of a map's (or a sequence's) queries to the states of another sequence, forward and backward.
//
//   S_ij = scale q_i . k_j over the live keys j of query i;  P = softmax_j(S);  out_i = sum_j P_ij v_j   (no live key: out_i = 0)
//   backward, g = dL/dout:  D_i = g_i . out_i;  dS_ij = P_ij (g_i . v_j - D_i);
//   dq_i = scale sum_j dS_ij k_j;  dk_j = scale sum_i dS_ij q_i;  dv_j = sum_i P_ij g_i
// A key is live when it lies below its image's length and its mask byte is not zero. Hq = Hk G query heads: head h reads state head h / G;
// the G heads of a group are G further ROWS of the same problem (row r = (query r / G, head r % G)), so that a tile of states is read
// once for the whole group and dk / dv sum over the group without a further pass.
//
// Products run on MFMA 32x32 tiles (bf16: 32x32x16; f32: 32x32x2, exact), one pass over the states with the running maximum and sum of the
// softmax. S is computed transposed (keys along the accumulator's rows, queries along its lanes): a lane then owns one query, the maximum
// and sum are in-lane plus one exchange between the wave's halves, and the accumulator's registers ARE the B operand of P V with no
// movement, because the sum over keys may run in any order as long as V is read in the same one: bf16 V^T comes from LDS by
// the transposing read (ds_read_b64_tr_b16), f32 V by plain reads. Probabilities enter P V (and dS the gradient products) rounded to bf16 in
// the bf16 kernels (relative 2^-8, as small as the rounding of the inputs); maxima, sums, S, D and all accumulators are f32.
//
// What bounds it: with 64 values a head, a wave's 32 x 64 scores cost 16 MFMAs (512 cycles) and 32 exponentials a lane with what surrounds
// them (about 900 cycles), so the vector unit; tiles therefore come to LDS by LDS-DMA (no registers, no instructions of the waves), two
// buffers deep, and the rescaling of the accumulators waits until the maximum has grown by 2^8. Measured in bf16: 4096 queries of 16 x 128 over 2048 states
// of 4 x 128, four images, 261 to 281 us from card to card (980 to 1050 TFLOP/s); 4096 queries over up to 512 states of 8 x 64, 16 images, 97 us (530 TFLOP/s; 42 of them for q, out and
// what rounding left of it). One query of 16 x 128 over up to 4096 states of 4 x 128, 32 images: 35 us (5.8 TB/s) and 4 for the join.
#include "igemm.h"
#include <algorithm>
#include <type_traits>

typedef __attribute__((ext_vector_type(8))) __bf16 b16x8_t;
typedef __attribute__((ext_vector_type(4))) short s16x4_t;

struct XaArgs {
    const void *q, *k, *v; void* o;          // o, g, dq: [B][Lq][H][D]; dk, dv: [B][Lk][Hk][D]
    bf16_t* lo;                               // what rounding o to bf16 left, or null: D = g . (o + lo) is off by 2^-16 of |g| |o| then (o alone: by 2^-8,
                                              // which where few keys share the weight is more than the rounding of dS itself)
    const void* g; void *dq, *dk, *dv;
    float* lse;                               // [B Hk][R] log2 of the softmax's denominator; +inf for a row without a live key
    float* delta;                             // [B Hk][R] D
    float* part; float* ml;                   // splits: [ns][B Hk][R][D] sums, [ns][B Hk][R] (max, sum); backward [2][ns][B Hk][Lk][D]
    const int* len; const unsigned char* mask;
    long long qb, ql, qh, kb, kl, kh, vb, vl, vh, mb, mq;   // strides in elements (mask: bytes; mq = 0: one mask row for all queries)
    int B, Lq, Lk, Hk, G, D, R, ns;
    float scale, c;                           // c = |scale| log2(e); a negative scale turns the sign of one operand of S
};

// ---- LDS tiles: rows of CH 16-byte chunks, chunk c of row r at place c ^ f(r): 16 rows at one chunk (row reads) and 4 rows x 4 chunks
// (transposing reads) each fall on 16 different 16-byte bank groups
template <int CH> __device__ __forceinline__ int xa_swz(int row) {
    if constexpr (CH == 4) return (row >> 2) & 3;
    else if constexpr (CH == 8) return (((row >> 1) & 1) << 2) | ((row >> 2) & 3);
    else return ((row & 3) << 2) | ((row >> 2) & 3);
}
template <int CH> __device__ __forceinline__ int xa_at(int row, int chunk) { return (row * CH + (chunk ^ xa_swz<CH>(row))) * 16; }

// ---- acc[a's row][b's row] += a . b over one step of dims (bf16: 16, f32: 8): a, b = the lane's 16-byte chunk 2 s + lane / 32 of its row
__device__ __forceinline__ void xa_dot(f32x16_t& acc, const uint4& a, const uint4& b, bf16_t) {
    acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(b16x8_t, a), __builtin_bit_cast(b16x8_t, b), acc, 0, 0, 0);
}
__device__ __forceinline__ void xa_dot(f32x16_t& acc, const uint4& a, const uint4& b, float) {
    acc = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a.x), __uint_as_float(b.x), acc, 0, 0, 0);
    acc = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a.y), __uint_as_float(b.y), acc, 0, 0, 0);
    acc = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a.z), __uint_as_float(b.z), acc, 0, 0, 0);
    acc = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a.w), __uint_as_float(b.w), acc, 0, 0, 0);
}
// The lane's places in a tile, as byte offsets: what differs by rows of 16 or 32, by tile or by buffer is a constant behind them, so that a read costs
// no address arithmetic. row[s]: its chunk of step s of row lane % 32; tr[db][..]: see xa_tr; el: where a f32 value is counted from.
template <typename T, int CH> struct XaAddr {
    static constexpr int S = CH / 2, ND = CH * 16 / (int)sizeof(T) / 32;
    int row[S], tr[sizeof(T) == 2 ? ND : 1][2], el = 0;
    __device__ __forceinline__ XaAddr() {
        const int lane = threadIdx.x & 63, h = lane >> 5, i = lane & 15, d16 = (lane >> 4) & 1;
#pragma unroll
        for (int s = 0; s < S; ++s) row[s] = xa_at<CH>(lane & 31, 2 * s + h);
        if constexpr (sizeof(T) == 2) {
            const int ra = 4 * h + (i >> 2);
#pragma unroll
            for (int db = 0; db < ND; ++db) {
                const int chunk = db * 4 + d16 * 2 + ((i & 3) >> 1), sub = (i & 1) * 8;
                tr[db][0] = xa_at<CH>(ra, chunk) + sub;
                tr[db][1] = xa_at<CH>(ra + 8, chunk) + sub;
            }
        }
    }
    __device__ __forceinline__ void move(int bytes) {
#pragma unroll
        for (int s = 0; s < S; ++s) row[s] += bytes;
#pragma unroll
        for (int db = 0; db < (sizeof(T) == 2 ? ND : 1); ++db) { tr[db][0] += bytes; tr[db][1] += bytes; }
        el += bytes;
    }
};
template <int NA> __device__ __forceinline__ void xa_zero(f32x16_t (&acc)[NA]) {
#pragma unroll
    for (int k = 0; k < NA; ++k)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[k][e] = 0.f;
}
__device__ __forceinline__ void xa_zero1(f32x16_t& acc) {
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[e] = 0.f;
}
// x = tile a . fa, y = tile b . fb (32 rows each; y on top of what it holds if not from0): two chains of products, one behind the other in turn
template <typename T, int CH>
__device__ __forceinline__ void xa_rows_dot2(f32x16_t& x, f32x16_t& y, const char* a, const char* b, const XaAddr<T, CH>& ad, const uint4 (&fa)[CH / 2],
                                             const uint4 (&fb)[CH / 2], bool from0 = true) {
    xa_zero1(x);
    if (from0) xa_zero1(y);
#pragma unroll
    for (int s = 0; s < CH / 2; ++s) {
        xa_dot(x, *reinterpret_cast<const uint4*>(a + ad.row[s]), fa[s], T());
        xa_dot(y, *reinterpret_cast<const uint4*>(b + ad.row[s]), fb[s], T());
    }
}
template <typename T, int CH> __device__ __forceinline__ void xa_rows_dot(f32x16_t& x, const char* a, const XaAddr<T, CH>& ad, const uint4 (&fa)[CH / 2]) {
    xa_zero1(x);
#pragma unroll
    for (int s = 0; s < CH / 2; ++s) xa_dot(x, *reinterpret_cast<const uint4*>(a + ad.row[s]), fa[s], T());
}

// ---- bf16: the lane's column of 8 tile rows as a product operand: column 32 db + lane % 32, rows 4 h + {0 .. 3} and 8 further on (and 16 t behind
// the tile pointer) -- the order in which an accumulator's registers 8 t .. 8 t + 7 hold its rows
__device__ __forceinline__ b16x8_t xa_tr(const char* tile, const int (&at)[2]) {
    typedef __attribute__((address_space(3))) s16x4_t lds4_t;
    const s16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4_t*)(tile + at[0]));
    const s16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4_t*)(tile + at[1]));
    bf16x8_t a;
#pragma unroll
    for (int e = 0; e < 4; ++e) { a[e] = lo[e]; a[4 + e] = hi[e]; }
    return __builtin_bit_cast(b16x8_t, a);
}
template <int CH> __device__ __forceinline__ float xa_el(const char* tile, int row, int col) {   // f32: one value
    return *reinterpret_cast<const float*>(tile + xa_at<CH>(row, col >> 2) + (col & 3) * 4);
}

// ---- acc[d][lane] += sum over 32 tile rows i of tile[i][d] p_i(lane); p: an accumulator (register r of a lane = row 8 (r / 4) + 4 (lane / 32) + r % 4)
template <int CH, int ND>
__device__ __forceinline__ void xa_tdot(f32x16_t (&acc)[ND], const char* tile, const XaAddr<bf16_t, CH>& ad, const f32x16_t& p) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        uint4 pb;
        pb.x = f2bf2(p[8 * t], p[8 * t + 1]); pb.y = f2bf2(p[8 * t + 2], p[8 * t + 3]);
        pb.z = f2bf2(p[8 * t + 4], p[8 * t + 5]); pb.w = f2bf2(p[8 * t + 6], p[8 * t + 7]);
#pragma unroll
        for (int db = 0; db < ND; ++db) acc[db] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(xa_tr(tile + 16 * t * CH * 16, ad.tr[db]), __builtin_bit_cast(b16x8_t, pb), acc[db], 0, 0, 0);
    }
}
template <int CH, int ND>
__device__ __forceinline__ void xa_tdot(f32x16_t (&acc)[ND], const char* tile, const XaAddr<float, CH>& ad, const f32x16_t& p) {
    const int lane = threadIdx.x & 63, h = lane >> 5;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        const int row = 8 * (r >> 2) + 4 * h + (r & 3);
#pragma unroll
        for (int db = 0; db < ND; ++db) acc[db] = __builtin_amdgcn_mfma_f32_32x32x2f32(xa_el<CH>(tile + ad.el, row, db * 32 + (lane & 31)), p[r], acc[db], 0, 0, 0);
    }
}
// ---- the same with p from a second tile of 32 rows x 32 columns (row i, column = lane): what an accumulator's transpose is, through LDS
template <typename T> struct XaSquare {
    static constexpr int CH = 32 * (int)sizeof(T) / 16, BYTES = 32 * CH * 16;
    __device__ __forceinline__ static void store(char* tile, const f32x16_t& p) {   // column i of the lane's accumulator -> row `lane`
        const int lane = threadIdx.x & 63, h = lane >> 5;
#pragma unroll
        for (int a = 0; a < 4; ++a) {
            const float v[4] = {p[4 * a], p[4 * a + 1], p[4 * a + 2], p[4 * a + 3]};
            if constexpr (sizeof(T) == 2) Op4<bf16_t>::store(reinterpret_cast<bf16_t*>(tile + xa_at<CH>(lane & 31, a) + 8 * h), v);
            else Op4<float>::store(reinterpret_cast<float*>(tile + xa_at<CH>(lane & 31, 2 * a + h)), v);
        }
        asm volatile("" ::: "memory");   // (the wave's own LDS accesses run in order; the compiler keeps them so)
    }
};
template <int CH, int ND>
__device__ __forceinline__ void xa_tdot(f32x16_t (&acc)[ND], const char* tile, const XaAddr<bf16_t, CH>& ad, const char* sq, const XaAddr<bf16_t, 4>& as) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        const b16x8_t pb = xa_tr(sq + 16 * t * 4 * 16, as.tr[0]);
#pragma unroll
        for (int db = 0; db < ND; ++db) acc[db] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(xa_tr(tile + 16 * t * CH * 16, ad.tr[db]), pb, acc[db], 0, 0, 0);
    }
}
template <int CH, int ND>
__device__ __forceinline__ void xa_tdot(f32x16_t (&acc)[ND], const char* tile, const XaAddr<float, CH>&, const char* sq, const XaAddr<float, 8>&) {
    const int lane = threadIdx.x & 63, h = lane >> 5;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        const int row = 8 * (r >> 2) + 4 * h + (r & 3);
        const float pb = xa_el<XaSquare<float>::CH>(sq, row, lane & 31);
#pragma unroll
        for (int db = 0; db < ND; ++db) acc[db] = __builtin_amdgcn_mfma_f32_32x32x2f32(xa_el<CH>(tile, row, db * 32 + (lane & 31)), pb, acc[db], 0, 0, 0);
    }
}

// workgroups go to the eight XCDs in turn: give each XCD a contiguous range of tiles, so that the tiles which read the same states share its L2.
// Pair j of an image and a state head is head j / B of image j % B: an XCD has many images' states, not a few images' heads, and no XCD is left
// with the long ones where lengths differ.
__device__ __forceinline__ int xa_tile_id(int n) {
    const int per = (n + 7) >> 3;
    return (blockIdx.x & 7) * per + (blockIdx.x >> 3);
}
__device__ __forceinline__ int xa_row_query(const XaArgs& p, int r) { return p.G == 1 ? r : (int)((unsigned)r / (unsigned)p.G); }
__device__ __forceinline__ int xa_len(const XaArgs& p, int b) {
    if (!p.len) return p.Lk;
    const int n = p.len[b];
    return n < 0 ? 0 : (n < p.Lk ? n : p.Lk);
}

// ---- tiles of NR rows x CH chunks to LDS by LDS-DMA. Thread i of TH fills places i, i + TH, ...: place (row, pos) takes chunk pos ^ f(row) of
// its row; what does not exist (rows that `rows` refuses, chunks behind D) is read out of range, which writes zeros.
#define XA_OOB 0x80000000u
#define XA_SPAN 0x7fffffffu   // bytes a tile's rows may span: checked on the host
template <typename T, int CH, int NR, int TH> struct XaDma {
    static constexpr int N = NR * CH / TH;
    unsigned off[N];   // byte offset of the place's chunk from the tile's first row
    __device__ __forceinline__ static int row(int i) { return (int)((threadIdx.x % TH + TH * i) / CH); }
    __device__ __forceinline__ static int chunk(int i) { return (int)((threadIdx.x % TH + TH * i) % CH) ^ xa_swz<CH>(row(i)); }
    __device__ __forceinline__ void init(long long stride, int D) {
#pragma unroll
        for (int i = 0; i < N; ++i) off[i] = chunk(i) * 16 < D * (int)sizeof(T) ? (unsigned)(row(i) * stride * (int)sizeof(T)) + chunk(i) * 16 : XA_OOB;
    }
    template <typename F> __device__ __forceinline__ void issue(const T* base, unsigned lds, F rows) const {   // base, lds: the same for all lanes
        if constexpr (TH == 64) asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // a wave refills a tile of its own behind no barrier: its reads of it are done
        const u32x4_t r = make_rsrc(base, XA_SPAN);
        const unsigned at = lds + (TH == 64 ? 0 : (__builtin_amdgcn_readfirstlane(threadIdx.x >> 6) * 1024));
#pragma unroll
        for (int i = 0; i < N; ++i) buf_load_lds16(r, rows(row(i)) ? off[i] : XA_OOB, at + i * TH * 16);
    }
    __device__ __forceinline__ void issue(const T* base, unsigned lds) const { issue(base, lds, [](int) { return true; }); }
};
template <int N> __device__ __forceinline__ void xa_wait_dma() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }

// the lane's chunks of a row as a product operand; neg: with the other sign
template <typename T, int CH> __device__ __forceinline__ void xa_row_frag(uint4 (&f)[CH / 2], const T* src, int D, bool neg = false) {
    const int h = (threadIdx.x & 63) >> 5;
    const unsigned flip = neg ? (sizeof(T) == 2 ? 0x80008000u : 0x80000000u) : 0u;
#pragma unroll
    for (int s = 0; s < CH / 2; ++s) {
        const int e = (2 * s + h) * (16 / (int)sizeof(T));
        f[s] = make_uint4(0, 0, 0, 0);
        if (src && e < D) f[s] = *reinterpret_cast<const uint4*>(src + e);
        f[s].x ^= flip; f[s].y ^= flip; f[s].z ^= flip; f[s].w ^= flip;
    }
}
// live bits of four consecutive keys j .. j + 3 of a mask row of Lk bytes (none is read outside the row)
__device__ __forceinline__ unsigned xa_mask4(const unsigned char* row, int j, int Lk) {
    unsigned w = 0;
    if (Lk >= 4) {
        const int jj = min(j, Lk - 4), sh = min(8 * (j - jj), 31);   // (bytes behind the row's end fall out of the word; j - jj > 3: nothing is left that counts)
        __builtin_memcpy(&w, row + jj, 4);
        w = j - jj > 3 ? 0u : w >> sh;
    } else {
        for (int e = 0; e < 3; ++e) if (j + e < Lk && row[j + e]) w |= 1u << (8 * e);
    }
    w = ((((w & 0x7f7f7f7fu) + 0x7f7f7f7fu) | w) >> 7) & 0x01010101u;   // one bit a byte: byte != 0
    return (w * 0x01020408u) >> 24 & 15u;
}
// live bits of the lane's 16 scores of 32 keys from j0 on: bit r = key j0 + 8 (r / 4) + 4 h + r % 4. kbits: the keys' own 32 bits
// (length, mask row of all queries), row: the query's own mask row or null
__device__ __forceinline__ unsigned xa_live(unsigned kbits, const unsigned char* row, int j0, int Lk) {
    const int h = (threadIdx.x & 63) >> 5;
    unsigned m = 0;
#pragma unroll
    for (int a = 0; a < 4; ++a) m |= ((kbits >> (8 * a + 4 * h)) & 15u) << (4 * a);
    if (row) {
        unsigned q = 0;
#pragma unroll
        for (int a = 0; a < 4; ++a) q |= xa_mask4(row, j0 + 8 * a + 4 * h, Lk) << (4 * a);
        m &= q;
    }
    return m;
}
typedef __bf16 xa_bf2_t __attribute__((ext_vector_type(2)));
__device__ __forceinline__ float xa_exp2(float x) { return __builtin_amdgcn_exp2f(x); }   // (below 2^-126: 0)
// x where bit e of live is set, else `other` (both by bits: two instructions)
__device__ __forceinline__ float xa_pick(unsigned live, int e, float x, unsigned other) {
    const unsigned m = (unsigned)__builtin_amdgcn_sbfe((int)live, e, 1);
    return __uint_as_float((__float_as_uint(x) & m) | (other & ~m));
}
// d + the dot product of two chunks, summed in 32 bits
template <typename T> __device__ __forceinline__ float xa_chunk_dot(const uint4& a, const uint4& b, float d) {
    const unsigned x[4] = {a.x, a.y, a.z, a.w}, y[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (sizeof(T) == 4) d = fmaf(__uint_as_float(x[i]), __uint_as_float(y[i]), d);
        else d = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(xa_bf2_t, x[i]), __builtin_bit_cast(xa_bf2_t, y[i]), d, false);
    }
    return d;
}
// One 32-row block of an accumulator (times f) to the D values of the lane's row from `row` on; lo: what rounding left, if wanted. bf16: the wave's halves
// trade registers (their rows are the same) so that each lane stores eight consecutive values at once.
template <typename T> __device__ __forceinline__ void xa_put(T* row, const f32x16_t& acc, float f, int d0, int D, bf16_t* lo = nullptr) {
    const int h = (threadIdx.x & 63) >> 5;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int a = 0; a < 4; ++a) {
            const int dd = d0 + 8 * a + 4 * h;
            const float v[4] = {acc[4 * a] * f, acc[4 * a + 1] * f, acc[4 * a + 2] * f, acc[4 * a + 3] * f};
            if (dd < D) Op4<float>::store(row + dd, v);
        }
    } else {
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            unsigned u[4], w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float x = acc[8 * q + 2 * i] * f, y = acc[8 * q + 2 * i + 1] * f;
                u[i] = f2bf2(x, y);
                w[i] = f2bf2(x - __uint_as_float(u[i] << 16), y - __uint_as_float(u[i] & 0xffff0000u));
            }
            const int dd = d0 + 16 * q + 8 * h;
            auto trade = [&](unsigned (&z)[4], bf16_t* to) {   // halves hold 4 h + 0 .. 3 and 8 + 4 h + 0 .. 3: -> 8 h + 0 .. 7
                const auto a = __builtin_amdgcn_permlane32_swap(z[0], z[2], false, false), b = __builtin_amdgcn_permlane32_swap(z[1], z[3], false, false);
                if (dd < D) *reinterpret_cast<uint4*>(to + dd) = make_uint4(a[0], b[0], a[1], b[1]);
            };
            trade(u, row);
            if (lo) trade(w, lo);
        }
    }
}
#define XA_NINF 0xff800000u
// log2 of a row's denominator l over the reference m, and 1 / l: +inf and 0 for a row without a live key (l = 0 and no maximum). Any other denominator that is no
// use shows: one that is not a number (a key or a query is not) stays so, so that the backward pass does not take the row for one that sees nothing, and
// one that vanished or overflowed beside a finite maximum (scores beyond 2^30, whose roundings in f32 pass the exponent's range) gives NaN, not zeros.
__device__ __forceinline__ bool xa_no_key(float m, float l) { return l == 0.f && m == -INFINITY; }
__device__ __forceinline__ float xa_lse(float m, float l) { return xa_no_key(m, l) ? INFINITY : l > 0.f && l < INFINITY ? m + log2f(l) : NAN; }
__device__ __forceinline__ float xa_inv(float m, float l) { return xa_no_key(m, l) ? 0.f : 1.f / l; }
// Between a matrix instruction and the first read of its result no branch may join: the compiler's wait count there follows one of the joining
// paths only. Live bits are therefore made in front of the products, masked and unmasked tiles are separate straight bodies, and behind a
// loop of products this wait stands.
__device__ __forceinline__ void xa_settle() { asm volatile("s_nop 15\n\ts_nop 7" ::: "memory"); }

// the states of one (image, state head): where they are and which of them live
template <typename T> struct XaStates {
    const T *k, *v;
    const unsigned char* mb;   // the image's mask or null
    int len; bool kmask;       // kmask: one mask row for all queries
    __device__ __forceinline__ XaStates(const XaArgs& p, int b, int hk) {
        k = reinterpret_cast<const T*>(p.k) + b * p.kb + hk * p.kh;
        v = reinterpret_cast<const T*>(p.v) + b * p.vb + hk * p.vh;
        mb = p.mask ? p.mask + b * p.mb : nullptr;
        len = xa_len(p, b);
        kmask = mb && p.mq == 0;
    }
    __device__ __forceinline__ bool live(int j) const { return j < len && (!kmask || mb[j]); }
};

// NR rows from r0 on of the queries and of g, for groups of several heads: row r0 + i = head (g0 + i) % G of query iq0 + (g0 + i) / G
template <typename T, int CH, int NR, int TH>
__device__ __forceinline__ void xa_issue_heads(const XaArgs& p, const T* qp, const T* gp, long long gl, int r0, float rG, unsigned qat, unsigned gat) {
    const int iq0 = (int)((unsigned)r0 / (unsigned)p.G), g0 = r0 - iq0 * p.G, left = p.R - r0;
    XaDma<T, CH, NR, TH> a, c;
#pragma unroll
    for (int i = 0; i < a.N; ++i) {
        const int rr = g0 + a.row(i), di = (int)(((float)rr + 0.5f) * rG), gg = rr - di * p.G, ck = a.chunk(i) * 16;
        const bool ok = ck < p.D * (int)sizeof(T) && a.row(i) < left;
        a.off[i] = ok ? (unsigned)((di * p.ql + gg * p.qh) * (int)sizeof(T)) + ck : XA_OOB;
        c.off[i] = ok ? (unsigned)((di * gl + gg * p.D) * (int)sizeof(T)) + ck : XA_OOB;
    }
    a.issue(qp + (long long)iq0 * p.ql, qat);
    c.issue(gp + (long long)iq0 * gl, gat);
}

// ------------------------------------------------------------------------------------------------ forward
// WQ = 4: four waves x 32 rows share tiles of 64 keys (one barrier a tile). WQ = 1: 32 rows (a single token, a few), every wave has tiles of 32
// keys of its own in its own part of LDS, no barrier in the loop, and a softmax of its own; the four are joined at the end. ns > 1: the tiles of states
// are cut in ns ranges, joined by xa_join_kernel.
template <typename T, int DP, int WQ> struct XaFwdTile {
    static constexpr int CH = DP * (int)sizeof(T) / 16, KT = WQ == 4 ? 64 : 32, TH = WQ == 4 ? 256 : 64;
    static constexpr int BYTES = KT * CH * 16;                                    // of K; V behind it
    static constexpr int NBUF = 4 * BYTES * (WQ == 4 ? 1 : 4) <= 128 * 1024 ? 2 : 1;
    static constexpr int LDS = 2 * BYTES * NBUF * (WQ == 4 ? 1 : 4);
    static constexpr int TOTAL = WQ == 4 ? LDS : (LDS > 512 * DP ? LDS : 512 * DP) + 1024;
};
template <typename T, int DP, int WQ>
__global__ __launch_bounds__(256, DP == 128 ? (sizeof(T) == 4 ? 1 : 2) : (sizeof(T) == 4 ? 2 : 3)) void xa_fwd_kernel(XaArgs p, int nqt, int total) {
    using Tile = XaFwdTile<T, DP, WQ>;
    constexpr int CH = Tile::CH, ND = DP / 32, S = CH / 2, KT = Tile::KT, TH = Tile::TH, QT = 32 * WQ, NBUF = Tile::NBUF, STEP = WQ == 4 ? 1 : 4;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int id = xa_tile_id(total);
    if (id >= total) return;
    const int j = id / (nqt * p.ns), rest = id - j * nqt * p.ns, split = rest / nqt, qt = rest - split * nqt;
    const int hk = j / p.B, b = j - hk * p.B, bh = b * p.Hk + hk;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5;
    const int r = qt * QT + (WQ == 4 ? wave * 32 : 0) + (lane & 31);
    const int iq = r < p.R ? xa_row_query(p, r) : 0, head = hk * p.G + (r < p.R ? r - iq * p.G : 0);
    const XaStates<T> st(p, b, hk);
    const int nt = (st.len + KT - 1) / KT, per = (nt + p.ns - 1) / p.ns;
    const int t0 = split * per + (WQ == 4 ? 0 : wave), t1 = min(nt, split * per + per);
    const unsigned char* mrow = st.mb && !st.kmask ? st.mb + (long long)iq * p.mq : nullptr;   // (null or not: the same for the whole launch)
    const unsigned lds = lds_addr_of(smem) + (WQ == 4 ? 0 : wave * 2 * Tile::BYTES * NBUF);
    XaDma<T, CH, KT, TH> dk, dv;
    dk.init(p.kl, p.D);
    dv.init(p.vl, p.D);
    auto issue = [&](int t, int buf) {
        const T *kp = st.k + (long long)t * KT * p.kl, *vp = st.v + (long long)t * KT * p.vl;
        const unsigned at = lds + buf * 2 * Tile::BYTES;
        if (st.kmask || (t + 1) * KT > st.len) {
            auto rows = [&](int i) { return st.live(t * KT + i); };
            dk.issue(kp, at, rows);
            dv.issue(vp, at + Tile::BYTES, rows);
        } else {
            dk.issue(kp, at);
            dv.issue(vp, at + Tile::BYTES);
        }
    };
    if (t0 < t1) issue(t0, 0);
    uint4 qf[S];
    xa_row_frag<T, CH>(qf, r < p.R ? reinterpret_cast<const T*>(p.q) + b * p.qb + (long long)iq * p.ql + head * p.qh : nullptr, p.D, p.scale < 0.f);
    XaAddr<T, CH> ad;
    if (WQ == 1) ad.move(wave * 2 * Tile::BYTES * NBUF);
    f32x16_t oacc[ND];
    xa_zero(oacc);
    float m = -INFINITY, l = 0.f;
    // one tile from the buffer at ks; live: its bits where `masked`
    auto work = [&](auto masked, const char* ks, const unsigned (&live)[KT / 32]) {
        constexpr bool M = decltype(masked)::value;
        const char* vs = ks + Tile::BYTES;
        f32x16_t sc[KT / 32];
        if constexpr (KT == 64) xa_rows_dot2<T, CH>(sc[0], sc[1], ks, ks + 32 * CH * 16, ad, qf, qf);
        else xa_rows_dot<T, CH>(sc[0], ks, ad, qf);
        float tm = -INFINITY;
#pragma unroll
        for (int kb = 0; kb < KT / 32; ++kb)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                if constexpr (M) sc[kb][e] = xa_pick(live[kb], e, sc[kb][e], XA_NINF);
                tm = fmaxf(tm, sc[kb][e]);
            }
        tm = fmaxf(tm, __shfl_xor(tm, 32, 64));
        tm *= p.c;   // (c > 0: -inf stays)
        if (__any(tm > m + 8.f)) {   // the reference moves only when it has to: what is summed stays below 2^8
            const float mn = fmaxf(m, tm), al = xa_exp2(m - (mn == -INFINITY ? 0.f : mn));
            m = mn;
            l *= al;
#pragma unroll
            for (int d = 0; d < ND; ++d)
#pragma unroll
                for (int e = 0; e < 16; ++e) oacc[d][e] *= al;
        }
        const float ref = M && m == -INFINITY ? 0.f : m;
#pragma unroll
        for (int kb = 0; kb < KT / 32; ++kb) {
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                sc[kb][e] = xa_exp2(fmaf(sc[kb][e], p.c, -ref));
                l += sc[kb][e];
            }
            xa_tdot<CH, ND>(oacc, vs + kb * 32 * CH * 16, ad, sc[kb]);
        }
    };
    // the tile's data has come; the next one's is sent for
    auto turn = [&](int t, int buf) {
        if (WQ == 4) {
            xa_wait_dma<0>();
            __syncthreads();
            if (NBUF == 2 && t + STEP < t1) issue(t + STEP, buf ^ 1);
        } else if (NBUF == 2 && t + STEP < t1) {
            issue(t + STEP, buf ^ 1);
            xa_wait_dma<2 * XaDma<T, CH, KT, TH>::N>();
        } else {
            xa_wait_dma<0>();
        }
    };
    const unsigned none[KT / 32] = {};
    const int tf = st.mb ? t0 : min(t1, st.len / KT);   // tiles below tf have no dead key
    int t = t0;
    if (NBUF == 2)
        for (; t + STEP < tf; t += 2 * STEP) {   // two tiles a round: the buffers' addresses are constants
            turn(t, 0);
            work(std::false_type(), smem, none);
            turn(t + STEP, 1);
            work(std::false_type(), smem + 2 * Tile::BYTES, none);
        }
    int buf = 0;
    for (; t < t1; t += STEP) {
        const int jl = t * KT + lane;
        const unsigned long long kbits = __ballot(lane < KT && st.live(jl));
        unsigned live[KT / 32];
#pragma unroll
        for (int kb = 0; kb < KT / 32; ++kb) live[kb] = xa_live((unsigned)(kbits >> (32 * kb)), mrow, t * KT + 32 * kb, p.Lk);
        turn(t, buf);
        work(std::true_type(), smem + buf * 2 * Tile::BYTES, live);
        if (NBUF == 2) buf ^= 1;
        else if (t + STEP < t1) {
            if (WQ == 4) __syncthreads();
            issue(t + STEP, 0);
        }
    }
    xa_settle();
    l += __shfl_xor(l, 32, 64);
    if constexpr (WQ == 1) {   // the four waves' softmaxes, in wave order
        float* ob = reinterpret_cast<float*>(smem);                                  // [4][DP][32]
        float* stt = reinterpret_cast<float*>(smem + Tile::TOTAL - 1024);            // [4][32] max, [4][32] sum
        __syncthreads();
        if (lane < 32) { stt[wave * 32 + lane] = m; stt[128 + wave * 32 + lane] = l; }
        __syncthreads();
        const int n = lane & 31;
        const float mn = fmaxf(fmaxf(stt[n], stt[32 + n]), fmaxf(stt[64 + n], stt[96 + n])), ref = mn == -INFINITY ? 0.f : mn;
        const float al = xa_exp2(m - ref);
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int e = 0; e < 16; ++e) ob[(wave * DP + d * 32 + 8 * (e >> 2) + 4 * h + (e & 3)) * 32 + n] = oacc[d][e] * al;
        l = 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w) l += stt[128 + w * 32 + n] * xa_exp2(stt[w * 32 + n] - ref);
        m = mn;
        __syncthreads();
        if (wave >= ND) return;   // wave d joins block d of the dims
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const int dd = wave * 32 + 8 * (e >> 2) + 4 * h + (e & 3);
            oacc[0][e] = (ob[dd * 32 + n] + ob[(DP + dd) * 32 + n]) + (ob[(2 * DP + dd) * 32 + n] + ob[(3 * DP + dd) * 32 + n]);
        }
    }
    if (r >= p.R) return;
    const size_t row = (size_t)bh * p.R + r;
    if (p.ns > 1) {
        float* o = p.part + ((size_t)split * p.B * p.Hk * p.R + row) * p.D;
        if (h == 0 && (WQ == 4 || wave == 0)) { float* q = p.ml + ((size_t)split * p.B * p.Hk * p.R + row) * 2; q[0] = m; q[1] = l; }
#pragma unroll
        for (int d = 0; d < (WQ == 1 ? 1 : ND); ++d)
#pragma unroll
            for (int a = 0; a < 4; ++a) {
                const int dd = (WQ == 1 ? wave : d) * 32 + 8 * a + 4 * h;
                if (dd < p.D) *reinterpret_cast<float4*>(o + dd) = make_float4(oacc[d][4 * a], oacc[d][4 * a + 1], oacc[d][4 * a + 2], oacc[d][4 * a + 3]);
            }
        return;
    }
    const float inv = xa_inv(m, l);
    if (p.lse && h == 0 && (WQ == 4 || wave == 0)) p.lse[row] = xa_lse(m, l);
    const size_t o = (((size_t)b * p.Lq + iq) * (p.Hk * p.G) + head) * p.D;
#pragma unroll
    for (int d = 0; d < (WQ == 1 ? 1 : ND); ++d) xa_put<T>(reinterpret_cast<T*>(p.o) + o, oacc[d], inv, (WQ == 1 ? wave : d) * 32, p.D, p.lo ? p.lo + o : nullptr);
}

// The ns ranges of a row: 32 lanes a row, four dims a lane. The lanes take the ranges' maxima and sums side by side (at most XA_MAX_SPLITS), then walk the
// ranges' partial rows in range order, eight in flight. WIDE: a row's ranges are many, and all eight groups of 32 lanes walk every eighth of them.
#define XA_MAX_SPLITS 256
template <typename T, bool WIDE>
__global__ __launch_bounds__(256) void xa_join_kernel(XaArgs p) {
    __shared__ float ws[8][XA_MAX_SPLITS];
    const int grp = threadIdx.x >> 5, n = threadIdx.x & 31, d = n * 4;
    const long long rows = (long long)p.B * p.Hk * p.R, row = WIDE ? (long long)blockIdx.x : (long long)blockIdx.x * 8 + grp;
    if (row >= rows) return;
    float* w = ws[grp];
    float mm[XA_MAX_SPLITS / 32], ll[XA_MAX_SPLITS / 32], mn = -INFINITY, l = 0.f;
#pragma unroll
    for (int k = 0; k < XA_MAX_SPLITS / 32; ++k) {
        const int s = n + 32 * k;
        const float2 q = s < p.ns ? *reinterpret_cast<const float2*>(p.ml + ((size_t)s * rows + row) * 2) : make_float2(-INFINITY, 0.f);
        mm[k] = q.x; ll[k] = q.y;
        mn = fmaxf(mn, q.x);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mn = fmaxf(mn, __shfl_xor(mn, o, 64));
    const float ref = mn == -INFINITY ? 0.f : mn;
#pragma unroll
    for (int k = 0; k < XA_MAX_SPLITS / 32; ++k) {
        const float f = xa_exp2(mm[k] - ref);
        l += ll[k] * f;
        w[n + 32 * k] = f;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) l += __shfl_xor(l, o, 64);
    asm volatile("" ::: "memory");   // (a row's lanes lie in one wave, whose LDS accesses run in order)
    float o[4] = {0.f, 0.f, 0.f, 0.f};
    if (d < p.D) {
        const float* src = p.part + row * p.D + d;
#pragma unroll 8
        for (int s = WIDE ? grp : 0; s < p.ns; s += WIDE ? 8 : 1) {
            const float4 a = *reinterpret_cast<const float4*>(src + (size_t)s * rows * p.D);
            o[0] = fmaf(a.x, w[s], o[0]); o[1] = fmaf(a.y, w[s], o[1]); o[2] = fmaf(a.z, w[s], o[2]); o[3] = fmaf(a.w, w[s], o[3]);
        }
    }
    if (WIDE) {
        __shared__ __attribute__((aligned(16))) float4 os[8][32];
        os[grp][n] = make_float4(o[0], o[1], o[2], o[3]);
        __syncthreads();
        if (grp) return;
#pragma unroll
        for (int g = 1; g < 8; ++g) {
            const float4 a = os[g][n];
            o[0] += a.x; o[1] += a.y; o[2] += a.z; o[3] += a.w;
        }
    }
    const float inv = xa_inv(mn, l);
    if (p.lse && d == 0) p.lse[row] = xa_lse(mn, l);
    if (d >= p.D) return;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] *= inv;
    const int bh = (int)(row / p.R), r = (int)(row - (long long)bh * p.R), b = bh / p.Hk, hk = bh - b * p.Hk;
    const int iq = xa_row_query(p, r), head = hk * p.G + r - iq * p.G;
    const size_t at = (((size_t)b * p.Lq + iq) * (p.Hk * p.G) + head) * p.D + d;
    Op4<T>::store(reinterpret_cast<T*>(p.o) + at, o);
    if (sizeof(T) == 2 && p.lo) {
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] -= bf2f(f2bf(o[e]));
        Op4<bf16_t>::store(p.lo + at, o);
    }
}

// ------------------------------------------------------------------------------------------------ backward: dq (and D)
// Four waves x 32 rows, tiles of 64 keys, as the forward, in ns ranges joined by xa_fold_dq_kernel; also leaves D for the kernel behind it. 4096 queries over up to 512 states of 8 x 64, 16 images, bf16:
// 135 us (570 TFLOP/s), of which reading q, g, out and what rounding left of it and writing dq (335 MB) takes 94 by itself.
// In f32 up to 64 values a head fit two waves a SIMD (4096 queries over 200 states of 4 x 64, 16 images: 290 us at one, 235 at two).
template <typename T, int DP>
__global__ __launch_bounds__(256, sizeof(T) == 4 && DP == 128 ? 1 : 2) void xa_dq_kernel(XaArgs p, int nqt, int ns, int total) {
    constexpr int CH = DP * (int)sizeof(T) / 16, ND = DP / 32, S = CH / 2, KT = 64, BYTES = KT * CH * 16;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int id = xa_tile_id(total);
    if (id >= total) return;
    const int j = id / (nqt * ns), rest = id - j * nqt * ns, split = rest / nqt, qt = rest - split * nqt;
    const int hk = j / p.B, b = j - hk * p.B, bh = b * p.Hk + hk;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5;
    const int r = qt * 128 + wave * 32 + (lane & 31);
    const bool on = r < p.R;
    const int iq = on ? xa_row_query(p, r) : 0, head = hk * p.G + (on ? r - iq * p.G : 0);
    const XaStates<T> st(p, b, hk);
    const int nt = p.dq ? (st.len + KT - 1) / KT : 0, per = (nt + ns - 1) / ns, t0 = split * per, t1 = min(nt, t0 + per);
    const size_t orow = (((size_t)b * p.Lq + iq) * (p.Hk * p.G) + head) * p.D;
    const unsigned char* mrow = st.mb && !st.kmask ? st.mb + (long long)iq * p.mq : nullptr;
    const unsigned lds = lds_addr_of(smem);
    XaDma<T, CH, KT, 256> dk, dv;
    dk.init(p.kl, p.D);
    dv.init(p.vl, p.D);
    auto issue = [&](int t, int buf) {
        const T *kp = st.k + (long long)t * KT * p.kl, *vp = st.v + (long long)t * KT * p.vl;
        const unsigned at = lds + buf * 2 * BYTES;
        if (st.kmask || (t + 1) * KT > st.len) {
            auto rows = [&](int i) { return st.live(t * KT + i); };
            dk.issue(kp, at, rows);
            dv.issue(vp, at + BYTES, rows);
        } else {
            dk.issue(kp, at);
            dv.issue(vp, at + BYTES);
        }
    };
    if (t0 < t1) issue(t0, 0);
    uint4 qf[S], gf[S];
    xa_row_frag<T, CH>(qf, on ? reinterpret_cast<const T*>(p.q) + b * p.qb + (long long)iq * p.ql + head * p.qh : nullptr, p.D, p.scale < 0.f);
    xa_row_frag<T, CH>(gf, on ? reinterpret_cast<const T*>(p.g) + orow : nullptr, p.D);
    float dl = 0.f;
    {
        const bool two = sizeof(T) == 2 && p.lo;   // (what rounding the result left; both parts' loads are in flight together)
        uint4 of[S], lf[sizeof(T) == 2 ? S : 1];
        xa_row_frag<T, CH>(of, on ? reinterpret_cast<const T*>(p.o) + orow : nullptr, p.D);
        if constexpr (sizeof(T) == 2) xa_row_frag<T, CH>(lf, on && two ? p.lo + orow : nullptr, p.D);
#pragma unroll
        for (int s = 0; s < S; ++s) {
            dl = xa_chunk_dot<T>(gf[s], of[s], dl);
            if constexpr (sizeof(T) == 2) dl = xa_chunk_dot<T>(gf[s], lf[s], dl);
        }
        dl += __shfl_xor(dl, 32, 64);
    }
    const float ls = on ? p.lse[(size_t)bh * p.R + r] : INFINITY;
    if (ls == INFINITY) dl = 0.f;   // (a row that sees nothing)
    if (on && h == 0 && split == 0) p.delta[(size_t)bh * p.R + r] = dl;
    XaAddr<T, CH> ad;
    f32x16_t acc[ND];
    xa_zero(acc);
    // masked: 0: every key is live. 1: some are dead for all queries: their rows are zeros in LDS, so that whatever finite number stands in their places
    // adds nothing (a score of 0 lies far above a row of very low ones: 2^8 at most). 2: by the query's own mask.
    auto work = [&](auto masked, const char* ks, const unsigned (&live)[2]) {
        constexpr int M = decltype(masked)::value;
        const char* vs = ks + BYTES;
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
            f32x16_t sc, dp;
            xa_rows_dot2<T, CH>(sc, dp, ks + kb * 32 * CH * 16, vs + kb * 32 * CH * 16, ad, qf, gf);
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                float x = fmaf(sc[e], p.c, -ls);
                if constexpr (M == 1) x = x > 8.f ? 8.f : x;   // (not fminf: a NaN stays)
                sc[e] = xa_exp2(x) * (dp[e] - dl);
                if constexpr (M == 2) sc[e] = xa_pick(live[kb], e, sc[e], 0u);
            }
            xa_tdot<CH, ND>(acc, ks + kb * 32 * CH * 16, ad, sc);
            __builtin_amdgcn_sched_barrier(0);   // (one block of 32 keys at a time: two would not fit the registers)
        }
    };
    auto turn = [&](int t, int buf) {
        xa_wait_dma<0>();
        __syncthreads();
        if (t + 1 < t1) issue(t + 1, buf ^ 1);
    };
    const unsigned none[2] = {};
    const int tf = st.mb ? t0 : min(t1, st.len / KT);
    int t = t0;
    for (; t + 1 < tf; t += 2) {
        turn(t, 0);
        work(std::integral_constant<int, 0>(), smem, none);
        turn(t + 1, 1);
        work(std::integral_constant<int, 0>(), smem + 2 * BYTES, none);
    }
    int buf = 0;
    if (!st.mb || st.kmask)
        for (; t < t1; ++t, buf ^= 1) {
            turn(t, buf);
            work(std::integral_constant<int, 1>(), smem + buf * 2 * BYTES, none);
        }
    for (; t < t1; ++t, buf ^= 1) {
        const unsigned long long kbits = __ballot(st.live(t * KT + lane));
        unsigned live[2];
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) live[kb] = xa_live((unsigned)(kbits >> (32 * kb)), mrow, t * KT + 32 * kb, p.Lk);
        turn(t, buf);
        work(std::integral_constant<int, 2>(), smem + buf * 2 * BYTES, live);
    }
    xa_settle();
    if (!on || !p.dq) return;
    if (ns > 1) {
        float* part = p.part + (((size_t)split * p.B * p.Hk + bh) * p.R + r) * p.D;
#pragma unroll
        for (int d = 0; d < ND; ++d) xa_put<float>(part, acc[d], p.scale, d * 32, p.D);
    } else {
#pragma unroll
        for (int d = 0; d < ND; ++d) xa_put<T>(reinterpret_cast<T*>(p.dq) + orow, acc[d], p.scale, d * 32, p.D);
    }
}
// dq of rows whose states were cut in ns ranges: the ranges' shares, in range order
template <typename T>
__global__ __launch_bounds__(256) void xa_fold_dq_kernel(XaArgs p, int ns) {
    const long long n = (long long)p.B * p.Hk * p.R * p.D, i = ((long long)blockIdx.x * 256 + threadIdx.x) * 4;
    if (i >= n) return;
    float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
    for (int k = 0; k < ns; ++k) {
        const float4 a = *reinterpret_cast<const float4*>(p.part + (size_t)k * n + i);
        s[0] += a.x; s[1] += a.y; s[2] += a.z; s[3] += a.w;
    }
    const long long row = i / p.D;
    const int d = (int)(i - row * p.D), bh = (int)(row / p.R), r = (int)(row - (long long)bh * p.R), b = bh / p.Hk, hk = bh - b * p.Hk, iq = xa_row_query(p, r);
    Op4<T>::store(reinterpret_cast<T*>(p.dq) + (((size_t)b * p.Lq + iq) * (p.Hk * p.G) + hk * p.G + r - iq * p.G) * p.D + d, s);
}

// ------------------------------------------------------------------------------------------------ backward: dk, dv
// A lane owns one key. WK = 4: four waves x 32 keys, every wave reads all 64 rows of a tile of queries and their gradients. WK = 2: two x 32 keys, a
// pair of waves each take half of the rows of a tile and are joined at the end. ns > 1: the rows are cut in ns ranges, added in range order by xa_fold_kernel.
// 16 images of 4096 queries, up to 512 states of 8 x 64, bf16: 155 us (660 TFLOP/s); a workgroup's chain of products and exponentials takes 1.9 us a tile where
// it is alone on its CU, two share 2.5. Three waves a SIMD do not fit the registers, and 64-row blocks side by side came out the same.
template <typename T, int DP, int WK>
__global__ __launch_bounds__(256, DP == 128 || (sizeof(T) == 4 && DP == 64) ? 1 : 2) void xa_dkv_kernel(XaArgs p, int nkt, int total) {
    constexpr int CH = DP * (int)sizeof(T) / 16, ND = DP / 32, S = CH / 2, RT = 64, BYTES = RT * CH * 16, KEYS = 32 * WK, ROWS = RT * WK / 4;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    float* rowv = reinterpret_cast<float*>(smem + 4 * BYTES);   // two of: [RT] lse, [RT] -D, [RT] query of the row
    const int id = xa_tile_id(total);
    if (id >= total) return;
    const int j = id / (nkt * p.ns), rest = id - j * nkt * p.ns, kt = rest / p.ns, split = rest - kt * p.ns;
    const int hk = j / p.B, b = j - hk * p.B, bh = b * p.Hk + hk;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5;
    const int key = kt * KEYS + (wave % WK) * 32 + (lane & 31), first = wave / WK * ROWS;   // first: of the wave's rows in a tile
    const XaStates<T> st(p, b, hk);
    const bool klive = st.live(key), qmask = st.mb && !st.kmask;
    const int nt = kt * KEYS < st.len ? (p.R + RT - 1) / RT : 0, per = (nt + p.ns - 1) / p.ns;
    const int t0 = split * per, t1 = min(nt, t0 + per);
    const unsigned lds = lds_addr_of(smem);
    const T* qp = reinterpret_cast<const T*>(p.q) + b * p.qb + hk * p.G * p.qh;
    const T* gp = reinterpret_cast<const T*>(p.g) + ((size_t)b * p.Lq * p.Hk + hk) * p.G * p.D;
    const long long gl = (long long)p.Hk * p.G * p.D;   // a query's step in g
    XaDma<T, CH, RT, 256> dq, dg;
    dq.init(p.ql, p.D);
    dg.init(gl, p.D);
    const float rG = 1.f / (float)p.G;
    float nls = INFINITY, ndl = 0.f;
    int niq = 0;
    auto issue = [&](int t, int buf) {
        const int r0 = t * RT, left = p.R - r0;
        const unsigned at = lds + buf * 2 * BYTES;
        if (p.G == 1) {
            const T *a = qp + (long long)r0 * p.ql, *c = gp + (long long)r0 * gl;
            if (left >= RT) { dq.issue(a, at); dg.issue(c, at + BYTES); }
            else {
                auto rows = [&](int i) { return i < left; };
                dq.issue(a, at, rows);
                dg.issue(c, at + BYTES, rows);
            }
        } else {
            xa_issue_heads<T, CH, RT, 256>(p, qp, gp, gl, r0, rG, at, at + BYTES);
        }
        if (threadIdx.x < RT) {
            const bool on = (int)threadIdx.x < left;
            const size_t row = (size_t)bh * p.R + r0 + (on ? threadIdx.x : 0);
            nls = on ? p.lse[row] : INFINITY;   // (a row behind the last: probabilities 0)
            ndl = on ? p.delta[row] : 0.f;
            niq = on ? xa_row_query(p, r0 + threadIdx.x) : 0;
        }
    };
    if (t0 < t1) issue(t0, 0);
    uint4 kf[S], vf[S];
    xa_row_frag<T, CH>(kf, klive ? st.k + key * p.kl : nullptr, p.D, p.scale < 0.f);
    xa_row_frag<T, CH>(vf, klive ? st.v + key * p.vl : nullptr, p.D);
    f32x16_t dk[ND], dv[ND];
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int e = 0; e < 16; ++e) { dk[d][e] = 0.f; dv[d][e] = 0.f; }
    XaAddr<T, CH> ad;
    if (WK == 2) ad.move(first * CH * 16);
    const float* const mine = rowv + first;
    auto work = [&](auto masked, const char* qs, const float* rv) {
        const char* gs = qs + BYTES;
#pragma unroll
        for (int row0 = 0; row0 < ROWS; row0 += 32) {
            unsigned live = 0;
            if constexpr (decltype(masked)::value) {
                if (klive) {
#pragma unroll
                    for (int e = 0; e < 16; ++e)
                        live |= (st.mb[(long long)reinterpret_cast<const int*>(rv)[2 * RT + row0 + 8 * (e >> 2) + 4 * h + (e & 3)] * p.mq + key] != 0 ? 1u : 0u) << e;
                }
            }
            f32x16_t pr, ds;
#pragma unroll
            for (int a = 0; a < 4; ++a) {   // (dP - D: the products are added to -D)
                const float4 dl = *reinterpret_cast<const float4*>(rv + RT + row0 + 8 * a + 4 * h);
                ds[4 * a] = dl.x; ds[4 * a + 1] = dl.y; ds[4 * a + 2] = dl.z; ds[4 * a + 3] = dl.w;
            }
            xa_rows_dot2<T, CH>(pr, ds, qs + row0 * CH * 16, gs + row0 * CH * 16, ad, kf, vf, false);
#pragma unroll
            for (int a = 0; a < 4; ++a) {
                const float4 ls = *reinterpret_cast<const float4*>(rv + row0 + 8 * a + 4 * h);
                const float lv[4] = {ls.x, ls.y, ls.z, ls.w};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int e = 4 * a + i;
                    pr[e] = xa_exp2(fmaf(pr[e], p.c, -lv[i]));
                    if constexpr (decltype(masked)::value) pr[e] = xa_pick(live, e, pr[e], 0u);
                    ds[e] = pr[e] * ds[e];
                    if constexpr (decltype(masked)::value) ds[e] = xa_pick(live, e, ds[e], 0u);
                }
            }
            xa_tdot<CH, ND>(dv, gs + row0 * CH * 16, ad, pr);
            xa_tdot<CH, ND>(dk, qs + row0 * CH * 16, ad, ds);
            __builtin_amdgcn_sched_barrier(0);   // (32 rows at a time: 64 would not fit the registers)
        }
    };
    auto turn = [&](int t, int buf) {
        float* rv = rowv + buf * 3 * RT;
        if (threadIdx.x < RT) { rv[threadIdx.x] = nls; rv[RT + threadIdx.x] = -ndl; reinterpret_cast<int*>(rv)[2 * RT + threadIdx.x] = niq; }
        xa_wait_dma<0>();
        __syncthreads();
        if (t + 1 < t1) issue(t + 1, buf ^ 1);
    };
    int t = t0;
    if (qmask) {
        for (int buf = 0; t < t1; ++t, buf ^= 1) {
            turn(t, buf);
            work(std::true_type(), smem + buf * 2 * BYTES, mine + buf * 3 * RT);
        }
    } else {   // (a dead key's lane works on zeros; what it sums is dropped below)
        for (; t + 1 < t1; t += 2) {
            turn(t, 0);
            work(std::false_type(), smem, mine);
            turn(t + 1, 1);
            work(std::false_type(), smem + 2 * BYTES, mine + 3 * RT);
        }
        if (t < t1) {
            turn(t, 0);
            work(std::false_type(), smem, mine);
        }
    }
    xa_settle();
    if (!klive) {
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int e = 0; e < 16; ++e) { dk[d][e] = 0.f; dv[d][e] = 0.f; }
    }
    if constexpr (WK == 2) {   // the second half's sums through LDS to the first
        float* ob = reinterpret_cast<float*>(smem) + (wave & 1) * DP * 64 + (lane & 31);   // [2 DP][32]
        __syncthreads();
        if (wave >= 2) {
#pragma unroll
            for (int d = 0; d < ND; ++d)
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const int dd = d * 32 + 8 * (e >> 2) + 4 * h + (e & 3);
                    ob[dd * 32] = dk[d][e];
                    ob[(DP + dd) * 32] = dv[d][e];
                }
        }
        __syncthreads();
        if (wave >= 2) return;
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int dd = d * 32 + 8 * (e >> 2) + 4 * h + (e & 3);
                dk[d][e] += ob[dd * 32];
                dv[d][e] += ob[(DP + dd) * 32];
            }
    }
    if (key >= p.Lk) return;
    if (p.ns > 1) {
        const size_t n = (size_t)p.B * p.Hk * p.Lk * p.D, at = ((size_t)bh * p.Lk + key) * p.D;
#pragma unroll
        for (int d = 0; d < ND; ++d) {
            xa_put<float>(p.part + (size_t)split * n + at, dk[d], p.scale, d * 32, p.D);
            xa_put<float>(p.part + (size_t)(p.ns + split) * n + at, dv[d], 1.f, d * 32, p.D);
        }
    } else {
        const size_t at = (((size_t)b * p.Lk + key) * p.Hk + hk) * p.D;
#pragma unroll
        for (int d = 0; d < ND; ++d) {
            xa_put<T>(reinterpret_cast<T*>(p.dk) + at, dk[d], p.scale, d * 32, p.D);
            xa_put<T>(reinterpret_cast<T*>(p.dv) + at, dv[d], 1.f, d * 32, p.D);
        }
    }
}
template <typename T>
__global__ __launch_bounds__(256) void xa_fold_kernel(XaArgs p) {
    const long long n = (long long)p.B * p.Hk * p.Lk * p.D, i = ((long long)blockIdx.x * 256 + threadIdx.x) * 4;
    if (i >= n) return;
    const float* src = p.part + (size_t)blockIdx.y * p.ns * n + i;
    float s[4] = {0.f, 0.f, 0.f, 0.f};
    for (int k = 0; k < p.ns; ++k) {
        const float4 a = *reinterpret_cast<const float4*>(src + (size_t)k * n);
        s[0] += a.x; s[1] += a.y; s[2] += a.z; s[3] += a.w;
    }
    const long long row = i / p.D;
    const int d = (int)(i - row * p.D), bh = (int)(row / p.Lk), key = (int)(row - (long long)bh * p.Lk), b = bh / p.Hk, hk = bh - b * p.Hk;
    Op4<T>::store(reinterpret_cast<T*>(blockIdx.y ? p.dv : p.dk) + (((size_t)b * p.Lk + key) * p.Hk + hk) * p.D + d, s);
}

// ------------------------------------------------------------------------------------------------ states that fit one tile
// 32 images of 4096 queries over 31 states of 4 x 32 with a mask a query, bf16: forward 22 us (71 MB), backward 30 (105 MB) and 4 for the fold.
// At most 32 states (a layout's objects): K and V stand in LDS for a whole workgroup, whose waves each walk row blocks of 32 on their own, with no
// barrier. Bound by bytes: q and out forward; q, g and dq backward -- S, P and D = sum_j P_ij (g_i . v_j) are made from them in registers, so
// that one launch gives dq and (through a transpose of P and dS in LDS) its rows' share of dk and dv.
template <typename T, int DP> struct XaShort {
    static constexpr int CH = DP * (int)sizeof(T) / 16, TILE = 32 * CH * 16;
    static constexpr int SQ = XaSquare<T>::BYTES;
    static constexpr int NBUF = 2 * TILE + 4 * (4 * TILE + 2 * SQ) <= 160 * 1024 ? 2 : 1;
    static constexpr int WAVE = 2 * TILE * NBUF + 2 * SQ;             // of a wave, backward
    static constexpr int BWD = 2 * TILE + 4 * WAVE;
    static constexpr bool OK = BWD <= 160 * 1024;
};
template <typename T, int CH> __device__ __forceinline__ void xa_stage32(char* tile, const T* src, long long stride, int D, const XaStates<T>& st) {
    for (int i = threadIdx.x; i < 32 * CH; i += 256) {
        const int row = i / CH, chunk = i - row * CH;
        uint4 a = make_uint4(0, 0, 0, 0);
        if (chunk * 16 < D * (int)sizeof(T) && st.live(row)) a = *reinterpret_cast<const uint4*>(src + row * stride + chunk * (16 / (int)sizeof(T)));
        *reinterpret_cast<uint4*>(tile + xa_at<CH>(row, chunk)) = a;
    }
}

template <typename T, int DP>
__global__ __launch_bounds__(256, DP == 128 || sizeof(T) == 4 ? 2 : 4) void xa_short_fwd_kernel(XaArgs p, int nwg, int total) {
    constexpr int CH = DP * (int)sizeof(T) / 16, ND = DP / 32, S = CH / 2;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    char *ks = smem, *vs = smem + 32 * CH * 16;
    const int id = xa_tile_id(total);
    if (id >= total) return;
    const int bh = id / nwg, part = id - bh * nwg, b = bh / p.Hk, hk = bh - b * p.Hk;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5;
    const int nblk = (p.R + 31) / 32, step = 4 * nwg;
    const XaStates<T> st(p, b, hk);
    const unsigned kbits = (unsigned)__ballot(lane < 32 && st.live(lane));
    const bool qmask = st.mb && !st.kmask, all = !qmask && kbits == 0xffffffffu;
    uint4 nq[S];
    unsigned nlive = 0;
    auto fetch = [&](int blk) {   // the block's queries and their live keys, on the way while the block before is worked on
        const int r = blk * 32 + (lane & 31), iq = r < p.R ? xa_row_query(p, r) : 0;
        const T* src = r < p.R ? reinterpret_cast<const T*>(p.q) + b * p.qb + (long long)iq * p.ql + (hk * p.G + r - iq * p.G) * p.qh : nullptr;
        xa_row_frag<T, CH>(nq, src, p.D, p.scale < 0.f);
        nlive = xa_live(kbits, qmask ? st.mb + (long long)iq * p.mq : nullptr, 0, p.Lk);
    };
    int blk = part * 4 + wave;
    if (blk < nblk) fetch(blk);
    xa_stage32<T, CH>(ks, st.k, p.kl, p.D, st);
    xa_stage32<T, CH>(vs, st.v, p.vl, p.D, st);
    __syncthreads();
    const XaAddr<T, CH> ad;
    for (; blk < nblk; blk += step) {
        uint4 qf[S];
#pragma unroll
        for (int s = 0; s < S; ++s) qf[s] = nq[s];
        const unsigned live = nlive;
        if (blk + step < nblk) fetch(blk + step);
        f32x16_t sc, oacc[ND];
        xa_rows_dot<T, CH>(sc, ks, ad, qf);
        float m = -INFINITY, l = 0.f;
#pragma unroll
        for (int e = 0; e < 16; ++e) { sc[e] = xa_pick(live, e, sc[e], XA_NINF); m = fmaxf(m, sc[e]); }
        m = fmaxf(m, __shfl_xor(m, 32, 64));
        const float ref = m == -INFINITY ? 0.f : m * p.c;
#pragma unroll
        for (int e = 0; e < 16; ++e) { sc[e] = xa_exp2(fmaf(sc[e], p.c, -ref)); l += sc[e]; }
        l += __shfl_xor(l, 32, 64);
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int e = 0; e < 16; ++e) oacc[d][e] = 0.f;
        xa_tdot<CH, ND>(oacc, vs, ad, sc);
        const float inv = xa_inv(m, l);
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int e = 0; e < 16; ++e) oacc[d][e] *= inv;   // (here, in front of the branch below)
        const int r = blk * 32 + (lane & 31);
        if (r < p.R) {
            const int iq = xa_row_query(p, r), head = hk * p.G + r - iq * p.G;
            if (p.lse && h == 0) p.lse[(size_t)bh * p.R + r] = xa_lse(m == -INFINITY ? m : ref, l);
            T* o = reinterpret_cast<T*>(p.o) + (((size_t)b * p.Lq + iq) * (p.Hk * p.G) + head) * p.D;
#pragma unroll
            for (int d = 0; d < ND; ++d) xa_put<T>(o, oacc[d], 1.f, d * 32, p.D);
        }
    }
}

template <typename T, int DP>
__global__ __launch_bounds__(256, DP == 128 || sizeof(T) == 4 ? 1 : DP == 64 ? 2 : 3) void xa_short_bwd_kernel(XaArgs p, int nwg, int total) {
    using Sh = XaShort<T, DP>;
    constexpr int CH = Sh::CH, ND = DP / 32, S = CH / 2, NBUF = Sh::NBUF;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    char *ks = smem, *vs = smem + Sh::TILE;
    const int id = xa_tile_id(total);
    if (id >= total) return;
    const int bh = id / nwg, part = id - bh * nwg, b = bh / p.Hk, hk = bh - b * p.Hk;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5;
    const int nblk = (p.R + 31) / 32, step = 4 * nwg;
    char* mine = smem + 2 * Sh::TILE + wave * Sh::WAVE;      // q and g tiles, NBUF of each; P, dS
    char *sp = mine + 2 * Sh::TILE * NBUF, *sd = sp + Sh::SQ;
    const unsigned lds = lds_addr_of(mine);
    const XaStates<T> st(p, b, hk);
    const unsigned kbits = (unsigned)__ballot(lane < 32 && st.live(lane));
    const bool qmask = st.mb && !st.kmask;
    const T* qp = reinterpret_cast<const T*>(p.q) + b * p.qb + hk * p.G * p.qh;
    const T* gp = reinterpret_cast<const T*>(p.g) + ((size_t)b * p.Lq * p.Hk + hk) * p.G * p.D;
    const long long gl = (long long)p.Hk * p.G * p.D;   // a query's step in g
    XaDma<T, CH, 32, 64> dq, dg;
    dq.init(p.ql, p.D);
    dg.init(gl, p.D);
    const float rG = 1.f / (float)p.G;
    auto issue = [&](int blk, int buf) {
        const int r0 = blk * 32, left = p.R - r0;
        const unsigned at = lds + buf * 2 * Sh::TILE;
        if (p.G == 1) {
            const T *a = qp + (long long)r0 * p.ql, *c = gp + (long long)r0 * gl;
            if (left >= 32) { dq.issue(a, at); dg.issue(c, at + Sh::TILE); }
            else {
                auto rows = [&](int i) { return i < left; };
                dq.issue(a, at, rows);
                dg.issue(c, at + Sh::TILE, rows);
            }
        } else {
            xa_issue_heads<T, CH, 32, 64>(p, qp, gp, gl, r0, rG, at, at + Sh::TILE);
        }
    };
    int blk = part * 4 + wave, buf = 0;
    if (blk < nblk) issue(blk, 0);
    xa_stage32<T, CH>(ks, st.k, p.kl, p.D, st);
    xa_stage32<T, CH>(vs, st.v, p.vl, p.D, st);
    __syncthreads();
    f32x16_t dk[ND], dv[ND];
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int e = 0; e < 16; ++e) { dk[d][e] = 0.f; dv[d][e] = 0.f; }
    const XaAddr<T, CH> ad;
    const XaAddr<T, XaSquare<T>::CH> as;
    for (; blk < nblk; blk += step) {
        const int r = blk * 32 + (lane & 31);
        const bool on = r < p.R;
        const int iq = on ? xa_row_query(p, r) : 0;
        const float ls = on ? p.lse[(size_t)bh * p.R + r] : INFINITY;   // (a row behind the last: probabilities 0)
        const unsigned live = xa_live(kbits, qmask ? st.mb + (long long)iq * p.mq : nullptr, 0, p.Lk);
        if (NBUF == 2 && blk + step < nblk) {
            issue(blk + step, buf ^ 1);
            xa_wait_dma<2 * XaDma<T, CH, 32, 64>::N>();
        } else {
            xa_wait_dma<0>();
        }
        const char *qs = mine + buf * 2 * Sh::TILE, *gs = qs + Sh::TILE;
        uint4 qf[S], gf[S];
        const unsigned flip = p.scale < 0.f ? (sizeof(T) == 2 ? 0x80008000u : 0x80000000u) : 0u;
#pragma unroll
        for (int s = 0; s < S; ++s) {
            qf[s] = *reinterpret_cast<const uint4*>(qs + ad.row[s]);
            gf[s] = *reinterpret_cast<const uint4*>(gs + ad.row[s]);
            qf[s].x ^= flip; qf[s].y ^= flip; qf[s].z ^= flip; qf[s].w ^= flip;
        }
        f32x16_t sc, dp, dqa[ND];
        xa_rows_dot2<T, CH>(sc, dp, ks, vs, ad, qf, gf);
        float dl = 0.f;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            sc[e] = xa_pick(live, e, xa_exp2(fmaf(sc[e], p.c, -ls)), 0u);
            dl = fmaf(sc[e], dp[e], dl);
        }
        dl += __shfl_xor(dl, 32, 64);
        XaSquare<T>::store(sp, sc);
#pragma unroll
        for (int e = 0; e < 16; ++e) sc[e] *= dp[e] - dl;
        XaSquare<T>::store(sd, sc);
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int e = 0; e < 16; ++e) dqa[d][e] = 0.f;
        xa_tdot<CH, ND>(dqa, ks, ad, sc);
        xa_tdot<CH, ND>(dv, gs, ad, sp, as);
        xa_tdot<CH, ND>(dk, qs, ad, sd, as);
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int e = 0; e < 16; ++e) dqa[d][e] *= p.scale;   // (here, in front of the branch below)
        if (on && p.dq) {
            T* o = reinterpret_cast<T*>(p.dq) + (((size_t)b * p.Lq + iq) * (p.Hk * p.G) + hk * p.G + r - iq * p.G) * p.D;
#pragma unroll
            for (int d = 0; d < ND; ++d) xa_put<T>(o, dqa[d], 1.f, d * 32, p.D);
        }
        if (NBUF == 2) buf ^= 1;
        else if (blk + step < nblk) issue(blk + step, 0);
    }
    xa_settle();
    if (!p.dk) return;
    // the four waves' shares, in wave order: [4][DP][32] f32 over the waves' tiles, dk then dv; wave d keeps block d of the dims
    float* ob = reinterpret_cast<float*>(smem);
    const int n = lane & 31;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        __syncthreads();
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int e = 0; e < 16; ++e) ob[(wave * DP + d * 32 + 8 * (e >> 2) + 4 * h + (e & 3)) * 32 + n] = which ? dv[d][e] : dk[d][e] * p.scale;
        __syncthreads();
        if (wave < ND && n < p.Lk) {
            float v[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int dd = wave * 32 + 8 * (e >> 2) + 4 * h + (e & 3);
                v[e] = (ob[dd * 32 + n] + ob[(DP + dd) * 32 + n]) + (ob[(2 * DP + dd) * 32 + n] + ob[(3 * DP + dd) * 32 + n]);
                if (!(kbits >> n & 1)) v[e] = 0.f;   // (a dead key, whatever the rows hold)
            }
#pragma unroll
            for (int a = 0; a < 4; ++a) {
                const int dd = wave * 32 + 8 * a + 4 * h;
                if (dd >= p.D) continue;
                const float w[4] = {v[4 * a], v[4 * a + 1], v[4 * a + 2], v[4 * a + 3]};
                if (p.ns > 1) {
                    const size_t all = (size_t)p.B * p.Hk * p.Lk * p.D;
                    Op4<float>::store(p.part + (size_t)(which * p.ns + part) * all + ((size_t)bh * p.Lk + n) * p.D + dd, w);
                } else {
                    Op4<T>::store(reinterpret_cast<T*>(which ? p.dv : p.dk) + (((size_t)b * p.Lk + n) * p.Hk + hk) * p.D + dd, w);
                }
            }
        }
    }
}

// ------------------------------------------------------------------------------------------------ entry points
#define XA_WGS 512   // workgroups that fill the chip: 256 CUs, two each. Kernels of one workgroup a CU (few rows forward; wide heads, as the registers of each
                     // kernel allow) take half of it: 32768 states of 128 x 8 heads, one query: 33 us at 512, 31 at 256; 32 images of 4096 x 8 x 64: 50 and 46;
                     // 1024 queries over 1024 states of 8 x 128, 4 images, f32, with the gradients: 834 and 758
static int xa_dp(int D) { return D <= 32 ? 32 : D <= 64 ? 64 : 128; }
// ranges of the states (forward) or rows (backward) for `tiles` workgroups over `nt` tiles of them: `wgs` workgroups, at least two tiles each
static int xa_splits(long long tiles, long long nt, int wgs) {
    if (tiles < 1 || tiles >= wgs || nt < 2) return 1;   // (no tiles: a list without states)
    long long ns = (wgs + tiles - 1) / tiles;
    if (ns > nt / 2) ns = nt / 2;
    if (ns > XA_MAX_SPLITS) ns = XA_MAX_SPLITS;
    return ns < 1 ? 1 : (int)ns;
}
struct XaPlan { int wq, nqt, ns, wk, nkt, nsb, nsq, nwf, nwb; };   // nwf, nwb: workgroups an (image, state head) of the one-tile form has, 0: not that form
static bool xa_short_fits(int dp, int dtype) {
    return dtype ? (dp == 32 ? XaShort<bf16_t, 32>::OK : dp == 64 ? XaShort<bf16_t, 64>::OK : XaShort<bf16_t, 128>::OK)
                 : (dp == 32 ? XaShort<float, 32>::OK : dp == 64 ? XaShort<float, 64>::OK : XaShort<float, 128>::OK);
}
static XaPlan xa_plan(int B, long long R, int Lk, int Hk, int D, int dtype) {
    XaPlan q;
    const int dp = xa_dp(D);
    const bool f32 = !dtype;
    const long long bh = (long long)B * Hk, groups = (R + 127) / 128;   // a workgroup's four waves take at least a block of 32 rows each
    q.nwf = q.nwb = 0;
    // the one-tile form, forward and forward with backward, against the general one: 32 images of 4096 queries over 31 states of 4 x 32 bf16 17 and 42 us, not 25
    // and 100 (with a mask a query 22 and 54, not 37 and 135); of 4 x 64 f32 73 and 245, not 109 and 488; one query of 8 x 64 bf16 5 and 12, not 6 and 16.
    // Workgroups: 1024 and 512 in all (2048 and 1024: 18 and 51 where these took 17 and 47, 4096 each: 23 and 73): staging the states and joining the shares of dk
    // and dv are paid less often
    if (Lk <= 32 && xa_short_fits(dp, dtype)) {
        q.nwf = (int)std::min(groups, std::max(1LL, (1024 + bh - 1) / bh));
        q.nwb = (int)std::min(groups, std::max(1LL, (512 + bh - 1) / bh));
    }
    // up to 32 rows a wave a tile of its own, four tiles at once: 16 rows over 4096 states of 8 x 64 x 8 images 20 us, not 21; 64 images of 256 states 8.7, not 10.1. From
    // 33 rows on it would read the states twice: 64 images of 64 rows over 100 states 12.5 us, not 8.6 (though over 4096 states 20, not 23)
    q.wq = R <= 32 ? 1 : 4;
    q.nqt = (int)((R + 32 * q.wq - 1) / (32 * q.wq));
    const int kt = q.wq == 4 ? 64 : 128;   // keys a workgroup takes at a time
    q.ns = xa_splits((long long)B * Hk * q.nqt, (Lk + kt - 1) / kt, q.wq == 4 && !(f32 && dp == 128) ? XA_WGS : XA_WGS / 2);
    // 64 keys a workgroup where 128 would leave waves or CUs without any (f32, 64 states of 64 x 4 heads x 16 images: 278 -> 218 us for dq, dk, dv;
    // 77 states of 40 x 2 x 8, f32: 22 -> 16 us for dk, dv), else 128, which stage the rows half as often (2048 states, bf16: 510 us, not 560)
    q.wk = Lk <= 64 || (Lk <= 128 && bh * ((Lk + 127) / 128) < 256) ? 2 : 4;
    q.nkt = (Lk + 32 * q.wk - 1) / (32 * q.wk);
    q.nsb = q.nwb ? q.nwb : xa_splits((long long)B * Hk * q.nkt, (R + 63) / 64, dp == 128 || (f32 && dp == 64) ? XA_WGS / 2 : XA_WGS);
    // (few rows over many states, f32 with the gradients: 300 queries of 4 x 128 over 2000 states of 2 x 128 526 us unsplit, 140 split; 1000 of 8 x 128 over
    // 2000 of 4 x 128 718 and 389)
    q.nsq = q.nwb ? 1 : xa_splits(bh * groups, (Lk + 63) / 64, f32 && dp == 128 ? XA_WGS / 2 : XA_WGS);
    if (q.nwf) q.ns = 1;
    return q;
}
static bool xa_bad(int B, int Lq, int Lk, int Hk, int G, int D, int dtype) {
    if (B < 1 || Lq < 1 || Lk < 0 || Hk < 1 || G < 1 || D < 8 || D > 128 || D % 8 || (dtype & ~1)) return true;
    const long long R = (long long)Lq * G, bh = (long long)B * Hk, most = (1LL << 24) - 8;
    // (rows are counted in 32 bits, their offsets in 64; a launch has less than 2^32 threads: 2^24 workgroups; a group's head is found by a f32 product)
    return G > 65536 || R > (1LL << 30) || Lk > (1 << 30) || bh > most || bh * ((R + 127) / 128) > most || bh * (((long long)Lk + 63) / 64) > most;
}
extern "C" int l2i_cross_attention_scratch(int B, int Lq, int Lk, int Hk, int G, int D, int dtype, int bwd, long long* floats) {
    if (!floats || xa_bad(B, Lq, Lk, Hk, G, D, dtype)) return L2I_ERR_ARG;
    const long long R = (long long)Lq * G;
    const XaPlan q = xa_plan(B, R, Lk, Hk, D, dtype);
    // (dq's shares are folded before the first of dk's and dv's is written: one place for both)
    if (bwd) *floats = ((long long)B * Hk * R + 3) / 4 * 4 + std::max(q.nsb > 1 ? 2LL * q.nsb * B * Hk * Lk * D : 0LL, q.nsq > 1 ? (long long)q.nsq * B * Hk * R * D : 0LL);
    else *floats = q.ns > 1 ? (long long)q.ns * B * Hk * R * (D + 2) : 0;
    return L2I_OK;
}
template <typename K>
static int xa_lds(K kernel, size_t lds) {
    return lds > 64 * 1024 && hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds) != hipSuccess ? L2I_ERR_LAUNCH : L2I_OK;
}
static unsigned xa_grid(long long total) { return (unsigned)((total + 7) / 8 * 8); }

template <typename T, int DP, int WQ>
static int xa_fwd_launch(const XaArgs& a, const XaPlan& q, hipStream_t s) {
    const int total = a.B * a.Hk * q.nqt * a.ns;
    const size_t lds = XaFwdTile<T, DP, WQ>::TOTAL;
    if (int e = xa_lds(xa_fwd_kernel<T, DP, WQ>, lds)) return e;
    hipLaunchKernelGGL((xa_fwd_kernel<T, DP, WQ>), dim3(xa_grid(total)), dim3(256), lds, s, a, q.nqt, total);
    return L2I_OK;
}
template <typename T, int DP>
static int xa_short_fwd_launch(const XaArgs& a, const XaPlan& q, hipStream_t s) {
    if constexpr (XaShort<T, DP>::OK) {
        const int total = a.B * a.Hk * q.nwf;
        hipLaunchKernelGGL((xa_short_fwd_kernel<T, DP>), dim3(xa_grid(total)), dim3(256), (size_t)2 * 32 * DP * sizeof(T), s, a, q.nwf, total);
    }
    return L2I_OK;
}
template <typename T>
static int xa_fwd_type(const XaArgs& a, const XaPlan& q, hipStream_t s) {
    const int dp = xa_dp(a.D);
    int e;
    if (q.nwf) return dp == 32 ? xa_short_fwd_launch<T, 32>(a, q, s) : dp == 64 ? xa_short_fwd_launch<T, 64>(a, q, s) : xa_short_fwd_launch<T, 128>(a, q, s);
    if (q.wq == 1) e = dp == 32 ? xa_fwd_launch<T, 32, 1>(a, q, s) : dp == 64 ? xa_fwd_launch<T, 64, 1>(a, q, s) : xa_fwd_launch<T, 128, 1>(a, q, s);
    else e = dp == 32 ? xa_fwd_launch<T, 32, 4>(a, q, s) : dp == 64 ? xa_fwd_launch<T, 64, 4>(a, q, s) : xa_fwd_launch<T, 128, 4>(a, q, s);
    if (e) return e;
    if (a.ns > 1) {
        const long long rows = (long long)a.B * a.Hk * a.R;
        // (one query over 262144 states of 128, 128 ranges: 59 us for both kernels with 32 lanes a row, 31 with 256)
        if (a.ns > 16) hipLaunchKernelGGL((xa_join_kernel<T, true>), dim3((unsigned)rows), dim3(256), 0, s, a);
        else hipLaunchKernelGGL((xa_join_kernel<T, false>), dim3((unsigned)((rows + 7) / 8)), dim3(256), 0, s, a);
    }
    return L2I_OK;
}
template <typename T>
static void xa_fold_launch(const XaArgs& a, hipStream_t s) {
    const long long n = (long long)a.B * a.Hk * a.Lk * a.D;
    hipLaunchKernelGGL((xa_fold_kernel<T>), dim3((unsigned)((n / 4 + 255) / 256), 2), dim3(256), 0, s, a);
}
template <typename T, int DP>
static int xa_bwd_launch(const XaArgs& a, const XaPlan& q, hipStream_t s) {
    if (q.nwb) {
        if constexpr (XaShort<T, DP>::OK) {
            const int total = a.B * a.Hk * q.nwb;
            // (the waves' shares of dk are joined over the whole of LDS: at least 512 DP bytes)
            const size_t lds = XaShort<T, DP>::BWD > 512 * DP ? XaShort<T, DP>::BWD : 512 * DP;
            if (int e = xa_lds(xa_short_bwd_kernel<T, DP>, lds)) return e;
            hipLaunchKernelGGL((xa_short_bwd_kernel<T, DP>), dim3(xa_grid(total)), dim3(256), lds, s, a, q.nwb, total);
            if (a.dk && a.Lk && a.ns > 1) xa_fold_launch<T>(a, s);
        }
        return L2I_OK;
    }
    const int nqt = (a.R + 127) / 128, nsq = a.dq ? q.nsq : 1, tq = a.B * a.Hk * nqt * nsq, tk = a.B * a.Hk * q.nkt * a.ns;
    const size_t lq = (size_t)4 * 64 * DP * sizeof(T), lk = lq + 6 * 64 * sizeof(float);
    if (int e = xa_lds(xa_dq_kernel<T, DP>, lq)) return e;
    hipLaunchKernelGGL((xa_dq_kernel<T, DP>), dim3(xa_grid(tq)), dim3(256), lq, s, a, nqt, nsq, tq);
    if (nsq > 1) {
        const long long n = (long long)a.B * a.Hk * a.R * a.D;
        hipLaunchKernelGGL((xa_fold_dq_kernel<T>), dim3((unsigned)((n / 4 + 255) / 256)), dim3(256), 0, s, a, nsq);
    }
    if (!a.dk || a.Lk == 0) return L2I_OK;
    if (q.wk == 4) {
        if (int e = xa_lds(xa_dkv_kernel<T, DP, 4>, lk)) return e;
        hipLaunchKernelGGL((xa_dkv_kernel<T, DP, 4>), dim3(xa_grid(tk)), dim3(256), lk, s, a, q.nkt, tk);
    } else {
        if (int e = xa_lds(xa_dkv_kernel<T, DP, 2>, lk)) return e;
        hipLaunchKernelGGL((xa_dkv_kernel<T, DP, 2>), dim3(xa_grid(tk)), dim3(256), lk, s, a, q.nkt, tk);
    }
    if (a.ns > 1) xa_fold_launch<T>(a, s);
    return L2I_OK;
}
// strides: 16-byte steps between any two rows, so that every row starts on a 16-byte boundary; the rows of a tile (64 positions and the G heads
// of a group) span less than 2^31 bytes
static bool xa_rows_ok(const void* t, long long sb, long long sl, long long sh, int heads, int dtype) {
    const long long e = dtype ? 8 : 4, most = 1LL << 31;
    if (((size_t)t & 15) || sb % e || sl % e || sh % e || sb < 0 || sl < 0 || sh < 0) return false;
    return sl < most / 512 && sh < most && 65 * sl * (16 / e) + heads * sh * (16 / e) + 1024 < most;
}
// the same for dout, which is contiguous: a tile's 64 rows lie in its first query and at most 1 + 62 / G further ones, Hk G D values apart
static bool xa_dout_ok(int Lq, int Hk, int G, int D, int dtype) {
    const long long steps = std::min(Lq - 1, 1 + 62 / G), values = steps * Hk * G * D + (long long)G * D;
    return values * (dtype ? 2 : 4) < 1LL << 31;
}
static void xa_setup(XaArgs& a, const void* q, const void* k, const void* v, const int* lengths, const unsigned char* mask, int B, int Lq, int Lk, int Hk,
                     int G, int D, long long qb, long long ql, long long qh, long long kb, long long kl, long long kh, long long vb, long long vl, long long vh,
                     long long mb, long long mq, float scale) {
    a.q = q; a.k = k; a.v = v; a.len = lengths; a.mask = mask; a.B = B; a.Lq = Lq; a.Lk = Lk; a.Hk = Hk; a.G = G; a.D = D; a.R = Lq * G;
    a.qb = qb; a.ql = ql; a.qh = qh; a.kb = kb; a.kl = kl; a.kh = kh; a.vb = vb; a.vl = vl; a.vh = vh; a.mb = mb; a.mq = mq;
    a.scale = scale; a.c = fabsf(scale) * 1.44269504088896340736f;
    if (a.c < 1.17549435e-38f) a.c = 1.17549435e-38f;   // (a scale of 0: scores of 0 all the same, and a dead key's -inf stays)
}
// whether out_lo is of use to the backward pass of these sizes: not in f32, nor where D does not come from out
extern "C" int l2i_cross_attention_wants_lo(int B, int Lq, int Lk, int Hk, int G, int D, int dtype) {
    return !xa_bad(B, Lq, Lk, Hk, G, D, dtype) && dtype && !xa_plan(B, (long long)Lq * G, Lk, Hk, D, dtype).nwb;
}
extern "C" int l2i_cross_attention_fwd(const void* q, const void* k, const void* v, int dtype, const int* lengths, const unsigned char* mask, void* out,
                                       void* out_lo, float* lse, int B, int Lq, int Lk, int Hk, int G, int D, long long qb, long long ql, long long qh, long long kb,
                                       long long kl, long long kh, long long vb, long long vl, long long vh, long long mb, long long mq, float scale,
                                       float* scratch, long long scratch_floats, void* stream) {
    long long need = 0;
    if (xa_bad(B, Lq, Lk, Hk, G, D, dtype) || !q || !out || (Lk && (!k || !v)) || mb < 0 || mq < 0 || (((size_t)out | (size_t)out_lo) & 15) || (out_lo && !dtype)) return L2I_ERR_ARG;
    if (!xa_rows_ok(q, qb, ql, qh, G, dtype) || !xa_rows_ok(k, kb, kl, kh, 0, dtype) || !xa_rows_ok(v, vb, vl, vh, 0, dtype)) return L2I_ERR_ARG;
    if (l2i_cross_attention_scratch(B, Lq, Lk, Hk, G, D, dtype, 0, &need) != L2I_OK) return L2I_ERR_ARG;
    if (need && (!scratch || ((size_t)scratch & 15) || scratch_floats < need)) return L2I_ERR_ARG;
    XaArgs a = {};
    xa_setup(a, q, k, v, lengths, mask, B, Lq, Lk, Hk, G, D, qb, ql, qh, kb, kl, kh, vb, vl, vh, mb, mq, scale);
    const XaPlan pl = xa_plan(B, a.R, Lk, Hk, D, dtype);
    a.o = out; a.lo = (bf16_t*)out_lo; a.lse = lse; a.ns = pl.ns;
    a.part = scratch; a.ml = scratch + (size_t)pl.ns * B * Hk * a.R * D;
    const int e = dtype ? xa_fwd_type<bf16_t>(a, pl, (hipStream_t)stream) : xa_fwd_type<float>(a, pl, (hipStream_t)stream);
    return e ? e : l2i_check_launch();
}
extern "C" int l2i_cross_attention_bwd(const void* q, const void* k, const void* v, int dtype, const int* lengths, const unsigned char* mask, const void* out,
                                       const void* out_lo, const float* lse, const void* dout, void* dq, void* dk, void* dv, int B, int Lq, int Lk, int Hk, int G, int D,
                                       long long qb, long long ql, long long qh, long long kb, long long kl, long long kh, long long vb, long long vl,
                                       long long vh, long long mb, long long mq, float scale, float* scratch, long long scratch_floats, void* stream) {
    long long need = 0;
    if (xa_bad(B, Lq, Lk, Hk, G, D, dtype) || !q || !out || !lse || !dout || (Lk && (!k || !v)) || mb < 0 || mq < 0) return L2I_ERR_ARG;
    if ((dk == nullptr) != (dv == nullptr) || (out_lo && !dtype) || (((size_t)out | (size_t)out_lo | (size_t)dout | (size_t)dq | (size_t)dk | (size_t)dv) & 15)) return L2I_ERR_ARG;
    if (!xa_rows_ok(q, qb, ql, qh, G, dtype) || !xa_rows_ok(k, kb, kl, kh, 0, dtype) || !xa_rows_ok(v, vb, vl, vh, 0, dtype) || !xa_dout_ok(Lq, Hk, G, D, dtype)) return L2I_ERR_ARG;
    if (l2i_cross_attention_scratch(B, Lq, Lk, Hk, G, D, dtype, 1, &need) != L2I_OK || !scratch || ((size_t)scratch & 15) || scratch_floats < need) return L2I_ERR_ARG;
    XaArgs a = {};
    xa_setup(a, q, k, v, lengths, mask, B, Lq, Lk, Hk, G, D, qb, ql, qh, kb, kl, kh, vb, vl, vh, mb, mq, scale);
    const XaPlan pl = xa_plan(B, a.R, Lk, Hk, D, dtype);
    a.o = const_cast<void*>(out); a.lo = (bf16_t*)const_cast<void*>(out_lo); a.lse = const_cast<float*>(lse); a.g = dout; a.dq = dq; a.dk = dk; a.dv = dv; a.ns = pl.nsb;
    a.delta = scratch; a.part = scratch + ((long long)B * Hk * a.R + 3) / 4 * 4;
    hipStream_t s = (hipStream_t)stream;
    const int dp = xa_dp(D);
    int e;
    if (dtype) e = dp == 32 ? xa_bwd_launch<bf16_t, 32>(a, pl, s) : dp == 64 ? xa_bwd_launch<bf16_t, 64>(a, pl, s) : xa_bwd_launch<bf16_t, 128>(a, pl, s);
    else e = dp == 32 ? xa_bwd_launch<float, 32>(a, pl, s) : dp == 64 ? xa_bwd_launch<float, 64>(a, pl, s) : xa_bwd_launch<float, 128>(a, pl, s);
    return e ? e : l2i_check_launch();
}
