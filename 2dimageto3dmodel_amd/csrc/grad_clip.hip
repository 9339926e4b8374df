// Global norm of a list of gradient tensors, and clipping by it (include/m355.h m355_grad_clip).
//
//   norm = |scale| sqrt(sum_i sum(g_i^2)),   c = min(1, max_norm / (norm + 1e-6)),   out_i = g_i * (scale c)
//
// Bound: HBM (2 - 3 operations a value).  The squares are added in 64 bits -- a gradient of 1e-25 or 1e+25 has a norm, where 32-bit
// squares give 0 or infinity -- and in a fixed order: one partial sum per workgroup, added by every workgroup of the second launch for
// itself in the same order, so there is no third launch, no atomic and no counter to clear.
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
constexpr int kChunk = 8192;         // values of a piece of work

struct Table {
    const void *in[kMaxT];
    void *out[kMaxT];
    long long n[kMaxT];
    unsigned start[kMaxT + 1];       // first piece of each tensor
    unsigned char dtype[kMaxT];
    int count;
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

template <typename T> __device__ __forceinline__ double piece_square(const T *p, int n)
{
    constexpr int V = 16 / sizeof(T);
    double acc = 0.0;
    int i = (int)threadIdx.x * V;
    for (; i + V <= n; i += kT * V) {
        const typename Any<T, V>::vt v = *reinterpret_cast<const typename Any<T, V>::vt *>(p + i);
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const double d = (double)(float)v[j];
            acc += d * d;
        }
    }
    for (int k = 0; k < V && i + k < n; ++k) {
        const double d = (double)(float)p[i + k];
        acc += d * d;
    }
    return acc;
}

__global__ __launch_bounds__(kT) void k_grad_square(const Table t, double *__restrict__ part)
{
    __shared__ double s[4];
    double acc = 0.0;
    const unsigned pieces = t.start[t.count];
    for (unsigned k = blockIdx.x; k < pieces; k += gridDim.x) {
        const int i = tensor_of(t, k);
        const long long o = (long long)(k - t.start[i]) * kChunk;
        const int n = (int)min((long long)kChunk, t.n[i] - o);
        if (t.dtype[i] == M355_F32) acc += piece_square((const float *)t.in[i] + o, n);
        else if (t.dtype[i] == M355_F16) acc += piece_square((const _Float16 *)t.in[i] + o, n);
        else acc += piece_square((const __bf16 *)t.in[i] + o, n);
    }
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

template <typename T> __device__ __forceinline__ void piece_scale(const T *p, T *q, int n, float c)
{
    constexpr int V = 16 / sizeof(T);
    int i = (int)threadIdx.x * V;
    for (; i + V <= n; i += kT * V) {
        typename Any<T, V>::vt v = *reinterpret_cast<const typename Any<T, V>::vt *>(p + i);
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] = (T)((float)v[j] * c);
        *reinterpret_cast<typename Any<T, V>::vt *>(q + i) = v;
    }
    for (int k = 0; k < V && i + k < n; ++k) q[i + k] = (T)((float)p[i + k] * c);
}

__global__ __launch_bounds__(kT) void k_grad_scale(const Table t, const double *__restrict__ part, int nparts, double scale, double max_norm,
                                                   float *__restrict__ norm, int write_norm)
{
    __shared__ double s[4];
    const double v = norm_of(part, nparts, scale, s);
    if (write_norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)v;
    // (a NaN norm fails the comparison: every gradient becomes NaN; an infinite one makes the factor 0)
    const double q = isinf(max_norm) ? 1.0 : max_norm / (v + 1e-6);   // (an infinite threshold never clips)
    const float c = (float)(scale * (q >= 1.0 ? 1.0 : q));
    const unsigned pieces = t.start[t.count];
    for (unsigned k = blockIdx.x; k < pieces; k += gridDim.x) {
        const int i = tensor_of(t, k);
        const long long o = (long long)(k - t.start[i]) * kChunk;
        const int n = (int)min((long long)kChunk, t.n[i] - o);
        if (c == 1.0f && t.in[i] == t.out[i]) continue;   // (times one in place)
        if (t.dtype[i] == M355_F32) piece_scale((const float *)t.in[i] + o, (float *)t.out[i] + o, n, c);
        else if (t.dtype[i] == M355_F16) piece_scale((const _Float16 *)t.in[i] + o, (_Float16 *)t.out[i] + o, n, c);
        else piece_scale((const __bf16 *)t.in[i] + o, (__bf16 *)t.out[i] + o, n, c);
    }
}

struct Span {
    uintptr_t lo, hi;
    int tensor, write;
};

static inline int esize(int dtype) { return dtype == M355_F32 ? 4 : 2; }

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
        total += (unsigned long long)(numel[i] + gc::kChunk - 1) / gc::kChunk;
        M355_REQUIRE(total < (1ULL << 32), "grad_clip: the list is too large");
    }
    if (out && n > 0) {
        const int rc = gc::check_overlap(in, out, numel, dtype, n);
        if (rc != M355_OK) return rc;
    }
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
                const unsigned long long k = (unsigned long long)(numel[i] + gc::kChunk - 1) / gc::kChunk;
                t.in[t.count] = in[i];
                t.out[t.count] = out ? out[i] : nullptr;
                t.n[t.count] = numel[i];
                t.dtype[t.count] = (unsigned char)dtype[i];
                t.start[t.count] = (unsigned)pieces;
                pieces += k;
                ++t.count;
            }
            t.start[t.count] = (unsigned)pieces;
            const unsigned grid = (unsigned)std::min<unsigned long long>(pieces, gc::kGrid);
            if (pass == 0) {
                if (grid > 0) {
                    hipLaunchKernelGGL(gc::k_grad_square, dim3(grid), dim3(gc::kT), 0, s, t, part + nparts);
                    nparts += (int)grid;
                }
            } else if (grid > 0 || first) {   // (an empty list still has a norm: 0)
                hipLaunchKernelGGL(gc::k_grad_scale, dim3(grid > 0 ? grid : 1), dim3(gc::kT), 0, s, t, part, nparts, scale, max_norm, norm,
                                   first ? 1 : 0);
                first = false;
            }
        }
    }
    if (!out) hipLaunchKernelGGL(gc::k_grad_norm, dim3(1), dim3(gc::kT), 0, s, part, nparts, scale, norm);
    return check_launch("grad_clip");
}
