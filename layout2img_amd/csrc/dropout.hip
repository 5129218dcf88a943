// Elementwise dropout whose mask comes from a counter-based generator and is never stored.
//
//   out[i] = keep_i ? in[i] * scale : 0   (+ res[i]),     keep_i = word_i >= threshold
//   word_{4 j + e} = word e of Philox4x32 (ten rounds) with key = seed and counter = (j, layer, offset)
// (Salmon, Moraes, Dror, Shaw, "Parallel random numbers: as easy as 1, 2, 3", 2011: the rounds and their four constants are the paper's).
// Bound by bytes: ten rounds are some 70 integer instructions for four elements, hidden under the loads. 33.5 M elements, bf16 in, f32 residual and
// out: 56 us (6.0 TB/s); their gradient, f32 to bf16: 38 us (5.2 TB/s). 79 k elements: 2.5 us, a launch.
// The words depend on (seed, offset, layer, i) alone: the backward pass calls the same entry point with in = dy and the (seed, offset)
// the forward read, and a mask is the same for every launch shape, type and GPU.
#include "common.h"

struct DropArgs {
    const void* in; const void* res; void* out;
    const long long* rng;   // device: seed, offset
    long long* used;        // device, optional: the pair this launch read
    long long n, j0;        // j0: first block of four of the launch
    unsigned threshold; int all, layer; float scale;   // all: threshold 2^32, nothing is kept
};

__device__ __forceinline__ uint4 philox4x32(unsigned k0, unsigned k1, uint4 c) {
#pragma unroll
    for (int r = 0; r < 10; ++r) {
        const unsigned long long p0 = (unsigned long long)c.x * 0xD2511F53u, p1 = (unsigned long long)c.z * 0xCD9E8D57u;
        c = make_uint4((unsigned)(p1 >> 32) ^ c.y ^ k0, (unsigned)p1, (unsigned)(p0 >> 32) ^ c.w ^ k1, (unsigned)p0);
        k0 += 0x9E3779B9u; k1 += 0xBB67AE85u;
    }
    return c;
}

// One generator block (four words) per four elements. VEC: all pointers allow 4-element accesses; otherwise element by element.
template <typename TI, typename TO, bool VEC>
__global__ __launch_bounds__(256) void dropout_kernel(DropArgs p) {
    const unsigned long long seed = (unsigned long long)p.rng[0], off = (unsigned long long)p.rng[1];
    if (p.used && p.j0 == 0 && blockIdx.x == 0 && threadIdx.x == 0) { p.used[0] = (long long)seed; p.used[1] = (long long)off; }
    const long long j = p.j0 + (long long)blockIdx.x * 256 + threadIdx.x, i = 4 * j;
    if (i >= p.n) return;
    const TI* in = reinterpret_cast<const TI*>(p.in) + i;
    const TO* res = p.res ? reinterpret_cast<const TO*>(p.res) + i : nullptr;
    TO* out = reinterpret_cast<TO*>(p.out) + i;
    const int m = p.n - i < 4 ? (int)(p.n - i) : 4;
    float v[4] = {0.f, 0.f, 0.f, 0.f}, q[4] = {0.f, 0.f, 0.f, 0.f};
    if (VEC && m == 4) {
        Op4<TI>::load(in, v);
        if (res) Op4<TO>::load(res, q);
    } else {
        for (int e = 0; e < m; ++e) { v[e] = OpT<TI>::to(in[e]); if (res) q[e] = OpT<TO>::to(res[e]); }
    }
    const uint4 w = philox4x32((unsigned)seed, (unsigned)(seed >> 32), make_uint4((unsigned)j, (unsigned)p.layer, (unsigned)off, (unsigned)(off >> 32)));
    const unsigned ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = ((!p.all && ww[e] >= p.threshold) ? v[e] * p.scale : 0.f) + q[e];   // (a select: a dropped infinity or NaN is 0)
    if (VEC && m == 4) Op4<TO>::store(out, v);
    else
        for (int e = 0; e < m; ++e) out[e] = OpT<TO>::from(v[e]);
}

template <typename TI, typename TO>
static void dropout_launch(DropArgs a, hipStream_t s) {
    const bool vec = !((size_t)a.in & (4 * sizeof(TI) - 1)) && !(((size_t)a.out | (size_t)a.res) & (4 * sizeof(TO) - 1));
    const long long blocks = ((a.n + 3) / 4 + 255) / 256, most = 1LL << 23;   // (a launch has less than 2^32 threads)
    for (long long i = 0; i < blocks; i += most) {
        a.j0 = i * 256;
        const dim3 grid((unsigned)(blocks - i < most ? blocks - i : most));
        if (vec) hipLaunchKernelGGL((dropout_kernel<TI, TO, true>), grid, dim3(256), 0, s, a);
        else hipLaunchKernelGGL((dropout_kernel<TI, TO, false>), grid, dim3(256), 0, s, a);
    }
}

extern "C" int l2i_dropout(const void* in, int in_dtype, const void* res, void* out, int out_dtype, const long long* rng, long long* used,
                           long long n, long long threshold, float scale, int layer, void* stream) {
    if (n < 0 || n > (1LL << 34) || threshold < 0 || threshold > (1LL << 32) || layer < 0 || (in_dtype | out_dtype) & ~1) return L2I_ERR_ARG;
    if (n == 0) return L2I_OK;
    if (!in || !out || !rng) return L2I_ERR_ARG;
    DropArgs a;
    a.in = in; a.res = res; a.out = out; a.rng = rng; a.used = used; a.n = n; a.layer = layer; a.scale = scale;
    a.all = threshold == (1LL << 32); a.threshold = a.all ? 0u : (unsigned)threshold;
    hipStream_t s = (hipStream_t)stream;
    if (in_dtype == 0) { if (out_dtype == 0) dropout_launch<float, float>(a, s); else dropout_launch<float, bf16_t>(a, s); }
    else { if (out_dtype == 0) dropout_launch<bf16_t, float>(a, s); else dropout_launch<bf16_t, bf16_t>(a, s); }
    return l2i_check_launch();
}
