// Global norm of a list of gradient tensors, and clipping by it (include/m355.h m355_grad_clip).
//
//   norm = |scale| sqrt(sum_i sum(g_i^2)),   c = min(1, max_norm / (norm + 1e-6)),   out_i = g_i * (scale c)
//
// Bound: HBM (2 - 3 operations a value).  The squares are added in 64 bits -- a gradient of 1e-25 or 1e+25 has a norm, where 32-bit
// squares give 0 or infinity -- and in a fixed order: one partial sum per workgroup, added by every workgroup of the second launch for
// itself in the same order, so there is no third launch, no atomic and no counter to clear.
// 24 layers of 3 x 3 x 1100 x 1100, bf16 and fp32 in turn (790 MB): squares 137 us, 5.8 TB/s, scaling 288 us, 5.5 TB/s (a copy reaches 5.4);
// the norm alone of the bf16 list (527 MB) 84 us, 6.6 TB/s with loads past the memory-side cache.  37 tensors of 47 MB 29 us; 7 of 2 MB 10
// us, both launches.
// The tensors' addresses travel in the kernel arguments (kMaxT a launch): nothing is copied to the device, and a captured graph holds them.
#include <algorithm>
#include <math.h>
#include <new>

#include "common.h"

namespace m355 {
namespace gc {

constexpr int kT = 256;
constexpr int kMaxT = 112;           // tensors a launch: 3.3 KB of kernel arguments (4 KB is the limit)
constexpr int kGrid = 1024;          // workgroups (= partial sums) a launch at most
constexpr int kU = 8;                // 16-byte vectors a thread has in flight
constexpr int kPiece = 32768;        // bytes of a piece of work: kU vectors of every thread

struct Table {
    const void *in[kMaxT];
    void *out[kMaxT];
    long long n[kMaxT];
    unsigned start[kMaxT + 1];       // first piece of each tensor
    unsigned char dtype[kMaxT];
    int count;
    unsigned per;                    // pieces a workgroup, one behind the other
};

__device__ __forceinline__ double block_sum(double v, double *s)
{
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
    __syncthreads();
    return (s[0] + s[1]) + (s[2] + s[3]);
}

__device__ __forceinline__ int tensor_of(const Table &t, unsigned piece)
{
    int lo = 0, hi = t.count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (t.start[mid] <= piece) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

// global memory takes a vector at any element's address
template <typename T, int V> struct Any {
    typedef T vt __attribute__((ext_vector_type(V), aligned(sizeof(T))));
};

// a vector at any element's address; NT: past the memory-side cache
template <bool NT, typename T> __device__ __forceinline__ typename Any<T, 16 / sizeof(T)>::vt get(const T *p)
{
    typedef typename Any<T, 16 / sizeof(T)>::vt vt;
    if constexpr (NT) return __builtin_nontemporal_load(reinterpret_cast<const vt *>(p));
    else return *reinterpret_cast<const vt *>(p);
}
template <bool NT, typename T> __device__ __forceinline__ void put(T *p, const typename Any<T, 16 / sizeof(T)>::vt &v)
{
    typedef typename Any<T, 16 / sizeof(T)>::vt vt;
    if constexpr (NT) __builtin_nontemporal_store(v, reinterpret_cast<vt *>(p));
    else *reinterpret_cast<vt *>(p) = v;
}

// f(offset, vector) over a piece of n values, one(offset) over those behind the last vector
template <bool NT, typename T, typename F, typename G> __device__ __forceinline__ void walk(const T *p, int n, F f, G one)
{
    constexpr int V = 16 / sizeof(T);
    typedef typename Any<T, V>::vt vt;
    int i = (int)threadIdx.x * V;
    if (n == kPiece / (int)sizeof(T)) {
        vt v[kU];
#pragma unroll
        for (int u = 0; u < kU; ++u) v[u] = get<NT>(p + i + u * kT * V);
#pragma unroll
        for (int u = 0; u < kU; ++u) f(i + u * kT * V, v[u]);
        return;
    }
    for (; i + V <= n; i += kT * V) f(i, get<false>(p + i));
    for (int k = 0; k < V && i + k < n; ++k) one(i + k);
}

// f(tensor, first value, values) over the workgroup's pieces
template <typename F> __device__ __forceinline__ void pieces_of(const Table &t, F f)
{
    const unsigned all = t.start[t.count];
    unsigned k = blockIdx.x * t.per;
    const unsigned end = min(all, k + t.per);
    if (k >= end) return;
    for (int i = tensor_of(t, k); k < end; ++k) {
        while (k >= t.start[i + 1]) ++i;   // (every tensor of the table has a piece)
        const long long len = t.dtype[i] == M355_F32 ? kPiece / 4 : kPiece / 2, o = (long long)(k - t.start[i]) * len;
        f(i, o, (int)min(len, t.n[i] - o));
    }
}

template <bool NT, typename T> __device__ __forceinline__ double piece_square(const T *p, int n)
{
    constexpr int V = 16 / sizeof(T);
    double a0 = 0.0, a1 = 0.0;
    walk<NT>(
        p, n,
        [&](int, const typename Any<T, V>::vt &v) {
#pragma unroll
            for (int j = 0; j < V; j += 2) {
                const double d = (double)(float)v[j], e = (double)(float)v[j + 1];
                a0 += d * d;
                a1 += e * e;
            }
        },
        [&](int i) {
            const double d = (double)(float)p[i];
            a0 += d * d;
        });
    return a0 + a1;
}

template <bool NT> __global__ __launch_bounds__(kT) void k_grad_square(const Table t, double *__restrict__ part)
{
    __shared__ double s[4];
    double acc = 0.0;
    pieces_of(t, [&](int i, long long o, int n) {
        if (t.dtype[i] == M355_F32) acc += piece_square<NT>((const float *)t.in[i] + o, n);
        else if (t.dtype[i] == M355_F16) acc += piece_square<NT>((const _Float16 *)t.in[i] + o, n);
        else acc += piece_square<NT>((const __bf16 *)t.in[i] + o, n);
    });
    const double v = block_sum(acc, s);
    if (threadIdx.x == 0) part[blockIdx.x] = v;
}

// the norm, the same bits in every workgroup
__device__ __forceinline__ double norm_of(const double *__restrict__ part, int nparts, double scale, double *s)
{
    double v = 0.0;
    for (int i = threadIdx.x; i < nparts; i += kT) v += part[i];
    return fabs(scale) * sqrt(block_sum(v, s));
}

__global__ __launch_bounds__(kT) void k_grad_norm(const double *__restrict__ part, int nparts, double scale, float *__restrict__ norm)
{
    __shared__ double s[4];
    const double v = norm_of(part, nparts, scale, s);
    if (threadIdx.x == 0) *norm = (float)v;
}

template <bool NT, typename T> __device__ __forceinline__ void piece_scale(const T *p, T *q, int n, float c)
{
    constexpr int V = 16 / sizeof(T);
    typedef typename Any<T, V>::vt vt;
    walk<NT>(
        p, n,
        [&](int i, vt v) {
#pragma unroll
            for (int j = 0; j < V; ++j) v[j] = (T)((float)v[j] * c);
            put<NT>(q + i, v);
        },
        [&](int i) { q[i] = (T)((float)p[i] * c); });
}

template <bool NT>
__global__ __launch_bounds__(kT) void k_grad_scale(const Table t, const double *__restrict__ part, int nparts, double scale, double max_norm,
                                                   float *__restrict__ norm, int write_norm)
{
    __shared__ double s[4];
    const double v = norm_of(part, nparts, scale, s);
    if (write_norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)v;
    // (a NaN norm fails the comparison: every gradient becomes NaN; an infinite one makes the factor 0)
    const double q = isinf(max_norm) && v == v ? 1.0 : max_norm / (v + 1e-6);   // (an infinite threshold clips nothing, not even an infinite norm)
    const float c = (float)(scale * (q >= 1.0 ? 1.0 : q));
    pieces_of(t, [&](int i, long long o, int n) {
        if (c == 1.0f && t.in[i] == t.out[i]) return;   // (times one in place)
        if (t.dtype[i] == M355_F32) piece_scale<NT>((const float *)t.in[i] + o, (float *)t.out[i] + o, n, c);
        else if (t.dtype[i] == M355_F16) piece_scale<NT>((const _Float16 *)t.in[i] + o, (_Float16 *)t.out[i] + o, n, c);
        else piece_scale<NT>((const __bf16 *)t.in[i] + o, (__bf16 *)t.out[i] + o, n, c);
    });
}

struct Span {
    uintptr_t lo, hi;
    int tensor, write;
};

static inline int esize(int dtype) { return dtype == M355_F32 ? 4 : 2; }

static inline unsigned long long pieces(long long numel, int dtype)
{
    const long long len = kPiece / esize(dtype);
    return (unsigned long long)((numel + len - 1) / len);
}

// no output may share memory with another output, or with another tensor's input
static int check_overlap(const void *const *in, void *const *out, const long long *numel, const int *dtype, int n)
{
    Span *sp = new (std::nothrow) Span[(size_t)2 * n];
    if (!sp) {
        set_error("grad_clip: out of host memory");
        return M355_ERR_BAD_ARG;
    }
    int k = 0;
    for (int i = 0; i < n; ++i) {
        if (numel[i] == 0) continue;
        const uintptr_t b = (uintptr_t)numel[i] * esize(dtype[i]);
        sp[k++] = {(uintptr_t)out[i], (uintptr_t)out[i] + b, i, 1};
        if (in[i] != out[i]) sp[k++] = {(uintptr_t)in[i], (uintptr_t)in[i] + b, i, 0};
    }
    std::sort(sp, sp + k, [](const Span &a, const Span &b) { return a.lo != b.lo ? a.lo < b.lo : a.write > b.write; });
    uintptr_t read_hi = 0, write_hi = 0;   // ends of the spans that began so far
    int bad = -1;
    for (int i = 0; i < k && bad < 0; ++i) {
        if (sp[i].lo < write_hi || (sp[i].write && sp[i].lo < read_hi)) bad = sp[i].tensor;
        uintptr_t &hi = sp[i].write ? write_hi : read_hi;
        hi = std::max(hi, sp[i].hi);
    }
    delete[] sp;
    if (bad >= 0) {
        set_error("grad_clip: tensor %d shares memory with another one (the same gradient twice, or overlapping outputs)", bad);
        return M355_ERR_BAD_ARG;
    }
    return M355_OK;
}

}  // namespace gc
}  // namespace m355

using namespace m355;

extern "C" size_t m355_grad_clip_ws_bytes(int n)
{
    if (n < 0) return 0;
    const size_t launches = (size_t)(n + gc::kMaxT - 1) / gc::kMaxT;
    return (launches > 0 ? launches : 1) * gc::kGrid * sizeof(double);
}

extern "C" int m355_grad_clip(const void *const *in, void *const *out, const long long *numel, const int *dtype, int n, double scale,
                              double max_norm, float *norm, void *ws, void *stream)
{
    M355_REQUIRE(n >= 0 && norm && ws && (n == 0 || (in && numel && dtype)), "grad_clip: null pointer");
    M355_REQUIRE(scale == scale && fabs(scale) <= 3.0e38, "grad_clip: scale must be finite");
    M355_REQUIRE(!out || max_norm >= 0.0, "grad_clip: max_norm %g", max_norm);
    unsigned long long total = 0;   // pieces: a launch counts them in 32 bits
    for (int i = 0; i < n; ++i) {
        M355_REQUIRE(dtype[i] == M355_F32 || dtype[i] == M355_F16 || dtype[i] == M355_BF16, "grad_clip: unknown dtype %d", dtype[i]);
        M355_REQUIRE(numel[i] >= 0 && numel[i] < (1LL << 40), "grad_clip: tensor %d has %lld values", i, numel[i]);
        M355_REQUIRE(numel[i] == 0 || (in[i] && (!out || out[i])), "grad_clip: tensor %d is null", i);
        M355_REQUIRE(((uintptr_t)in[i] % gc::esize(dtype[i])) == 0 && (!out || ((uintptr_t)out[i] % gc::esize(dtype[i])) == 0),
                     "grad_clip: tensor %d is not aligned to its element", i);
        total += gc::pieces(numel[i], dtype[i]);
        M355_REQUIRE(total < (1ULL << 32), "grad_clip: the list is too large");
    }
    if (out && n > 0) {
        const int rc = gc::check_overlap(in, out, numel, dtype, n);
        if (rc != M355_OK) return rc;
    }
    const bool nt = total * gc::kPiece >= (160ULL << 20);   // (more than the memory-side cache keeps between the passes)
    hipStream_t s = (hipStream_t)stream;
    double *part = (double *)ws;
    int nparts = 0;
    for (int pass = 0; pass < (out ? 2 : 1); ++pass) {
        bool first = true;
        for (int i = 0; i < n || (pass == 1 && first);) {
            gc::Table t;
            t.count = 0;
            unsigned long long pieces = 0;
            for (; i < n && t.count < gc::kMaxT; ++i) {
                if (numel[i] == 0) continue;
                const unsigned long long k = gc::pieces(numel[i], dtype[i]);
                t.in[t.count] = in[i];
                t.out[t.count] = out ? out[i] : nullptr;
                t.n[t.count] = numel[i];
                t.dtype[t.count] = (unsigned char)dtype[i];
                t.start[t.count] = (unsigned)pieces;
                pieces += k;
                ++t.count;
            }
            t.start[t.count] = (unsigned)pieces;
            unsigned grid = (unsigned)std::min<unsigned long long>(pieces, gc::kGrid);
            t.per = grid > 0 ? (unsigned)((pieces + grid - 1) / grid) : 1;
            if (grid > 0) grid = (unsigned)((pieces + t.per - 1) / t.per);
            if (pass == 0) {
                if (grid > 0) {
                    if (nt && !out) hipLaunchKernelGGL(gc::k_grad_square<true>, dim3(grid), dim3(gc::kT), 0, s, t, part + nparts);
                    else hipLaunchKernelGGL(gc::k_grad_square<false>, dim3(grid), dim3(gc::kT), 0, s, t, part + nparts);
                    nparts += (int)grid;
                }
            } else if (grid > 0 || first) {   // (an empty list still has a norm: 0)
                const dim3 g(grid > 0 ? grid : 1);
                if (nt) hipLaunchKernelGGL(gc::k_grad_scale<true>, g, dim3(gc::kT), 0, s, t, part, nparts, scale, max_norm, norm, first ? 1 : 0);
                else hipLaunchKernelGGL(gc::k_grad_scale<false>, g, dim3(gc::kT), 0, s, t, part, nparts, scale, max_norm, norm, first ? 1 : 0);
                first = false;
            }
        }
    }
    if (!out) hipLaunchKernelGGL(gc::k_grad_norm, dim3(1), dim3(gc::kT), 0, s, part, nparts, scale, norm);
    return check_launch("grad_clip");
}
