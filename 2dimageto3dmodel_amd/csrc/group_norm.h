// Group norm with an activation on channels-last tensors: the kernels (group_norm_f32.hip, _f16.hip and _bf16.hip instantiate
// them for a type each; the entry points are in group_norm.hip).
//
//   m = HW * D values per (sample, group of D = C / G neighbouring channels)
//   mean = sum x / m,  var = sum (x - mean)^2 / m,  rstd = 1 / sqrt(var + eps),  xhat = (x - mean) rstd
//   z = xhat * w + b,  y = act(z) [+ res],  act = LeakyReLU(slope) or SiLU z / (1 + e^-z)
//   backward, dz = dy act'(z):  db = sum_hw dz,  dw = sum_hw dz xhat,
//   dx = rstd (w dz - mean_g(w dz) - xhat mean_g(w dz xhat)),  dres = dy (2 x 2 sums when res is stored at half resolution)
//
// A thread owns one vector of V channels (16 bytes where the sizes allow) and every PL-th pixel of its workgroup's range, so its
// affine and statistics stay in registers.  A vector is cut into A segments of V / A channels that never straddle a group.
//
// Statistics do not subtract large numbers from each other: a thread adds deviations from K, the mean of its own first values; the
// threads' means are joined first, and the squared deviations are then taken about the joined mean.  All sums are 32-bit, in a fixed
// order: the same bits on every run.
//
// Bound: HBM and launches; some 10 operations a value.  Figures below: "large" is 64 x 256 x 128 x 64 bf16 (268 MB) in 32 groups with a
// half-resolution residual, where counters see no byte read or written that the kernel's formula does not name.  A kernel that only reads
// reaches 6.2 TB/s on this card, one that copies 5.4 (8 when both tensors fit the memory-side cache).
#pragma once
#include "common.h"

namespace m355 {
namespace gn {

// division by a number the host knows: exact for dividends below 2^31
struct Div {
    unsigned d, mul, shift;
    __host__ void set(unsigned by)
    {
        d = by;
        mul = shift = 0;
        if (by > 1) {
            int l = 0;
            while ((1ULL << l) < by) ++l;
            mul = (unsigned)(((1ULL << (31 + l)) / by) + 1);
            shift = (unsigned)(l - 1);
        }
    }
    __device__ __forceinline__ unsigned of(unsigned n) const { return d == 1 ? n : __umulhi(n, mul) >> shift; }
};

struct Args {
    const void *x, *dy, *res;
    void *y, *dres;               // y: forward's result, backward's dx (NULL: not wanted)
    const float *w, *b;           // NULL: 1 / 0
    float *mean, *rstd;           // [N][G]
    float2 *gpart;                // [N][nblk][G]: forward (mean, M2); backward (sum w dz, sum w dz xhat)
    float2 *gsum;                 // backward, with `finished`: [N][G] (mean_g(w dz), mean_g(w dz xhat))
    float *cpart;                 // backward [N][nblk][2][C]: (sum dz, sum dz xhat)
    float *dw, *db;               // backward, NULL: not wanted
    long long aff_stride;         // floats between the samples' rows of w and b (0: one row for all)
    long long hw;                 // pixels of a sample
    long long items, per;         // what a kernel walks: pixels, or 2 x 2 blocks of them (quad); those of a workgroup's range
    long long gper;               // values a channel of a gpart range covers (the last one fewer)
    int N, C, G, D;
    int SC, LV, PL, nslab;        // channels of a slab (whole groups, whole vectors), vectors across it, pixel lanes, slabs
    int nblk, gnblk;              // ranges of a sample in this kernel; rows of gpart / cpart a sample
    int act, per_sample, quad, finished;
    int nt;                       // outputs and the second pass's inputs go past the memory-side cache
    int W2;                       // quad: half the width
    Div by_w2, by_lv, by_pl, by_nslab, by_nblk, by_d, by_sg;   // sg = D / (channels of a segment)
    float w_off, eps, slope, out_slope;
};

template <typename T, int V> struct IO {
    typedef T raw __attribute__((ext_vector_type(V)));
    static __device__ __forceinline__ raw load(const T *p) { return *reinterpret_cast<const raw *>(p); }
    static __device__ __forceinline__ void open(const raw &v, float (&f)[V])
    {
#pragma unroll
        for (int j = 0; j < V; ++j) f[j] = (float)v[j];
    }
    // NT: past the memory-side cache
    template <bool NT> static __device__ __forceinline__ raw load(const T *p)
    {
        if constexpr (NT) return __builtin_nontemporal_load(reinterpret_cast<const raw *>(p));
        else return *reinterpret_cast<const raw *>(p);
    }
    static __device__ __forceinline__ raw pack(const float (&f)[V])
    {
        raw v;
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] = (T)f[j];   // to nearest even, once, from the 32-bit result
        return v;
    }
    template <bool NT> static __device__ __forceinline__ void put(T *p, const raw &v)
    {
        if constexpr (NT) __builtin_nontemporal_store(v, reinterpret_cast<raw *>(p));
        else *reinterpret_cast<raw *>(p) = v;
    }
    template <bool NT> static __device__ __forceinline__ void store(T *p, const float (&f)[V]) { put<NT>(p, pack(f)); }
};

// the registers of a loaded vector are used again later: keeps the compiler from carrying its 32-bit form (twice the registers) along
template <typename R> __device__ __forceinline__ void keep(R &v)
{
    if constexpr (sizeof(R) >= 4) {
        struct U {
            unsigned w[sizeof(R) / 4];
        } u = __builtin_bit_cast(U, v);
#pragma unroll
        for (unsigned i = 0; i < sizeof(R) / 4; ++i) asm volatile("" : "+v"(u.w[i]));
        v = __builtin_bit_cast(R, u);
    }
}

constexpr int kT = 256;   // threads of a workgroup

struct Place {   // what a workgroup and a thread of it own
    int n, slab, blk, lv, pl, c0, ng;   // ng: groups of the slab
    bool on;
    long long i0, ni;                   // items
    __device__ __forceinline__ Place(const Args &a, unsigned id, int V)
    {
        const unsigned r = a.by_nblk.of(id);   // (below 2^31: the host's launches)
        blk = (int)(id - r * (unsigned)a.nblk);
        n = (int)a.by_nslab.of(r);
        slab = (int)r - n * a.nslab;
        pl = (int)a.by_lv.of(threadIdx.x);
        lv = (int)threadIdx.x - pl * a.LV;
        c0 = slab * a.SC + lv * V;
        on = pl < a.PL && c0 < a.C;
        ng = (int)a.by_d.of((unsigned)min(a.SC, a.C - slab * a.SC));
        i0 = (long long)blk * a.per;
        ni = min(a.per, a.items - i0);
    }
    __device__ __forceinline__ int g0(const Args &a) const { return slab * (int)a.by_d.of((unsigned)a.SC); }
};

__device__ __forceinline__ int vectors_of(const Args &a, const Place &pc)
{
    return pc.on && pc.pl < pc.ni ? (int)a.by_pl.of((unsigned)((int)pc.ni - pc.pl + a.PL - 1)) : 0;   // (a range has fewer than 2^31 items: checked by the host)
}

// first pixel of item i (quad: the block's top left one; the others are 1, W and W + 1 further)
__device__ __forceinline__ long long first_pixel(const Args &a, long long i)
{
    if (!a.quad) return i;
    const long long h = a.items < (1LL << 31) ? (long long)a.by_w2.of((unsigned)i) : i / a.W2;
    return 2 * (i + h * a.W2);
}

__device__ __forceinline__ float sigmoid(float z) { return __builtin_amdgcn_rcpf(1.0f + __expf(-z)); }

// ---- sums over a workgroup's threads by group.  sh: [rows][stride], row = pixel lane, sg columns a group; odd strides keep the
// lanes of a group off each other's banks.  tpg (a power of two, at most 64) neighbouring threads add up a group, its first one has f.
template <typename F> __device__ __forceinline__ void by_group(int ng, F f)
{
    int l = 6;
    while (l > 0 && (ng << l) > kT) --l;
    const int k = (int)threadIdx.x & ((1 << l) - 1);
    for (int g = (int)threadIdx.x >> l; g < ng; g += kT >> l) f(g, k, 1 << l);
}

__device__ __forceinline__ float lanes_sum(float v, int tpg)
{
    for (int o = tpg >> 1; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

__device__ __forceinline__ float columns_sum(const float *sh, int stride, int rows, const Div &by_sg, int g, int k, int tpg)
{
    float s = 0.0f;
    const int sg = (int)by_sg.d, total = rows * sg;
    for (int e = k; e < total; e += tpg) {
        const int r = (int)by_sg.of((unsigned)e);
        s += sh[r * stride + g * sg + e - r * sg];
    }
    return lanes_sum(s, tpg);
}

// the affine of the thread's channels
template <int V> __device__ __forceinline__ void affine(const Args &a, const Place &pc, float (&w)[V], float (&b)[V])
{
    typedef float row __attribute__((ext_vector_type(V), aligned(4)));   // (the rows may start at any float)
    const long long i = (long long)pc.n * a.aff_stride + pc.c0;
    row wv = {}, bv = {};
    if (pc.on && a.w) wv = *reinterpret_cast<const row *>(a.w + i);
    if (pc.on && a.b) bv = *reinterpret_cast<const row *>(a.b + i);
    const float off = a.w ? a.w_off : 1.0f;
#pragma unroll
    for (int j = 0; j < V; ++j) {
        w[j] = wv[j] + off;
        b[j] = bv[j];
    }
}

// a thread's own (mean, M2) of each segment, from deviations about K
template <int V, int A> struct Stat {
    static constexpr int S = V / A;
    float K[A], s[A], q[A];
    __device__ __forceinline__ void start()
    {
#pragma unroll
        for (int a = 0; a < A; ++a) K[a] = s[a] = q[a] = 0.0f;
    }
    __device__ __forceinline__ void about(const float (&f)[V], float part)   // K += part * (the vector's segment sums)
    {
#pragma unroll
        for (int a = 0; a < A; ++a) {
            float t = 0.0f;
#pragma unroll
            for (int j = 0; j < S; ++j) t += f[a * S + j];
            K[a] += t * part;
        }
    }
    __device__ __forceinline__ void add(const float (&f)[V])
    {
#pragma unroll
        for (int a = 0; a < A; ++a)
#pragma unroll
            for (int j = 0; j < S; ++j) {
                const float d = f[a * S + j] - K[a];
                s[a] += d;
                q[a] += d * d;
            }
    }
    // pixels -> K: mean, q: M2
    __device__ __forceinline__ void close(float pixels)
    {
        const float n = pixels * S, r = n > 0.0f ? 1.0f / n : 0.0f;
#pragma unroll
        for (int a = 0; a < A; ++a) {
            const float m = q[a] - s[a] * (s[a] * r);
            q[a] = m < 0.0f ? 0.0f : m;   // (a NaN stays)
            K[a] += s[a] * r;
        }
    }
};

// joins the threads' statistics: s_mean / s_m2 [groups of the slab].  `pixels`: this thread's, `all`: the workgroup's.  sh: kT * (A + 1)
template <int V, int A>
__device__ __forceinline__ void join_threads(const Args &a, const Place &pc, const Stat<V, A> &st, float pixels, float all, float *sh,
                                             float *s_mean, float *s_m2)
{
    constexpr int S = V / A;
    const int stride = (a.LV * A) | 1;
    const float inv = 1.0f / (all * (float)a.D);
    float *mine = sh + pc.pl * stride + pc.lv * A;
    if (pc.pl < a.PL) {
#pragma unroll
        for (int k = 0; k < A; ++k) mine[k] = pc.on ? pixels * S * st.K[k] : 0.0f;
    }
    __syncthreads();
    by_group(pc.ng, [&](int g, int k, int tpg) {
        const float v = columns_sum(sh, stride, a.PL, a.by_sg, g, k, tpg);
        if (k == 0) s_mean[g] = v * inv;
    });
    __syncthreads();
    if (pc.on) {
#pragma unroll
        for (int k = 0; k < A; ++k) {
            const float d = st.K[k] - s_mean[a.by_sg.of((unsigned)(pc.lv * A + k))];
            mine[k] = st.q[k] + pixels * S * d * d;
        }
    }
    __syncthreads();
    by_group(pc.ng, [&](int g, int k, int tpg) {
        const float v = columns_sum(sh, stride, a.PL, a.by_sg, g, k, tpg);
        if (k == 0) s_m2[g] = v;
    });
}

// y of one vector; `add`: plus the residual's vector
template <typename T, int V, int A, int ACT, bool NT>
__device__ __forceinline__ void finish_store(const Args &a, const float (&f)[V], const float (&mu)[A], const float (&k)[V], const float (&b)[V],
                                             bool add, const typename IO<T, V>::raw &res, T *y)
{
    constexpr int S = V / A;
    float z[V];
#pragma unroll
    for (int j = 0; j < V; ++j) z[j] = (f[j] - mu[j / S]) * k[j] + b[j];
    if constexpr (ACT == 0) {
#pragma unroll
        for (int j = 0; j < V; ++j) z[j] = z[j] >= 0.0f ? z[j] : z[j] * a.slope;
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j) z[j] = z[j] * sigmoid(z[j]);
    }
    if (add) {
        float r[V];
        IO<T, V>::open(res, r);
#pragma unroll
        for (int j = 0; j < V; ++j) z[j] += r[j];
    }
    if (a.out_slope != 1.0f) {
#pragma unroll
        for (int j = 0; j < V; ++j) z[j] = z[j] >= 0.0f ? z[j] : z[j] * a.out_slope;
    }
    IO<T, V>::template store<NT>(y, z);
}

// xc = x - mean and dz of one vector.  z is computed as the forward computes it: the sign a LeakyReLU's gradient goes by is the forward's
template <int V, int A, int ACT>
__device__ __forceinline__ void grad_of(const Args &a, const float (&f)[V], const float (&d)[V], const float (&mu)[A], const float (&k)[V],
                                        const float (&b)[V], float (&xc)[V], float (&dz)[V])
{
    constexpr int S = V / A;
#pragma unroll
    for (int j = 0; j < V; ++j) xc[j] = f[j] - mu[j / S];
    if constexpr (ACT == 0) {
#pragma unroll
        for (int j = 0; j < V; ++j) dz[j] = xc[j] * k[j] + b[j] >= 0.0f ? d[j] : d[j] * a.slope;
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const float z = xc[j] * k[j] + b[j], s = sigmoid(z);
            dz[j] = d[j] * (s * (1.0f + z * (1.0f - s)));
        }
    }
}

// ---- forward, first of two passes: gpart[n][blk][g] = (mean, M2) of the workgroup's pixels.  Four 16-byte loads in flight a thread (eight
// are no faster).  Large: 48 us, 5.6 TB/s; 16 x 64 x 32 x 256 bf16 6.1 us, most of it the launch and the join
template <typename T, int V, int A> __global__ __launch_bounds__(kT) void k_gn_stats(const Args a)
{
    constexpr int R = 4;   // loads in flight a thread
    __shared__ float sh[kT * (A + 1)], s_mean[kT * A], s_m2[kT * A];
    const Place pc(a, blockIdx.x, V);
    const T *x = (const T *)a.x + ((size_t)pc.n * a.hw + pc.i0) * a.C + pc.c0;
    Stat<V, A> st;
    st.start();
    const int ni = (int)pc.ni;   // (a range has fewer than 2^31 pixels: checked by the host)
    const int mine = vectors_of(a, pc);
    if (mine > 0) {
        const size_t step = (size_t)a.PL * a.C;
        const T *p = x + (size_t)pc.pl * a.C;
        int i = 0;
        if (mine >= R) {
            float f[R][V];
#pragma unroll
            for (int u = 0; u < R; ++u) IO<T, V>::open(IO<T, V>::load(p + u * step), f[u]);
#pragma unroll
            for (int u = 0; u < R; ++u) st.about(f[u], 1.0f / (R * (V / A)));
#pragma unroll
            for (int u = 0; u < R; ++u) st.add(f[u]);
            for (i = R; i + R <= mine; i += R) {
                p += R * step;
                typename IO<T, V>::raw v[R];
#pragma unroll
                for (int u = 0; u < R; ++u) v[u] = IO<T, V>::load(p + u * step);
#pragma unroll
                for (int u = 0; u < R; ++u) {
                    float g[V];
                    IO<T, V>::open(v[u], g);
                    st.add(g);
                }
            }
            p += R * step;
        }
        for (; i < mine; ++i, p += step) {
            float f[V];
            IO<T, V>::open(IO<T, V>::load(p), f);
            if (i == 0) st.about(f, 1.0f / (V / A));
            st.add(f);
        }
        st.close((float)mine);
    }
    join_threads<V, A>(a, pc, st, (float)mine, (float)ni, sh, s_mean, s_m2);
    __syncthreads();
    float2 *out = a.gpart + ((size_t)pc.n * a.gnblk + pc.blk) * a.G + pc.g0(a);
    for (int g = threadIdx.x; g < pc.ng; g += kT) out[g] = make_float2(s_mean[g], s_m2[g]);
}

// mean and rstd of a group from its ranges' parts, by tpg lanes: the parts of up to kBatch ranges a lane are loaded at once
constexpr int kBatch = 8;
__device__ __forceinline__ void join_ranges(const Args &a, int n, int g, int k, int tpg, float &mu, float &rs)
{
    const float2 *p = a.gpart + (size_t)n * a.gnblk * a.G + g;
    const float m = (float)((double)a.hw * a.D), full = (float)a.gper * a.D;
    const float tail = (float)(a.hw - (long long)(a.gnblk - 1) * a.gper) * a.D;   // values of the last range
    float s = 0.0f, q = 0.0f;
    if (a.gnblk <= kBatch * tpg) {
        float2 v[kBatch];
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
            const int i = k + u * tpg;
            v[u] = i < a.gnblk ? p[(size_t)i * a.G] : make_float2(0.0f, 0.0f);
        }
#pragma unroll
        for (int u = 0; u < kBatch; ++u) s += v[u].x * (k + u * tpg < a.gnblk - 1 ? full : tail);
        mu = lanes_sum(s, tpg) / m;
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
            const int i = k + u * tpg;
            const float d = v[u].x - mu;
            if (i < a.gnblk) q += v[u].y + d * d * (i < a.gnblk - 1 ? full : tail);
        }
    } else {
        for (int i = k; i < a.gnblk; i += tpg) s += p[(size_t)i * a.G].x * (i < a.gnblk - 1 ? full : tail);
        mu = lanes_sum(s, tpg) / m;
        for (int i = k; i < a.gnblk; i += tpg) {
            const float2 v = p[(size_t)i * a.G];
            const float d = v.x - mu;
            q += v.y + d * d * (i < a.gnblk - 1 ? full : tail);
        }
    }
    rs = 1.0f / sqrtf(lanes_sum(q, tpg) / m + a.eps);
}

// ---- between the passes when a sample has many ranges: mean, rstd [N][G], a wave a group
static __global__ __launch_bounds__(kT) void k_gn_finish(const Args a)
{
    const long long i = ((long long)blockIdx.x * kT + threadIdx.x) >> 6;
    if (i >= (long long)a.N * a.G) return;
    const int n = (int)(i / a.G), g = (int)(i - (long long)n * a.G), k = threadIdx.x & 63;
    float mu, rs;
    join_ranges(a, n, g, k, 64, mu, rs);
    if (k == 0) {
        a.mean[i] = mu;
        a.rstd[i] = rs;
    }
}

// A walk over a thread's vectors in steps of R, the next step's loads in flight while f works on this one and stores: a wait for a load also
// waits for the stores issued before it (one counter, in order), and a loop that loads behind its stores pays their way to memory each
// time round.  start() issues the first loads; run() walks.
template <int R, typename Raw, int K> struct Ahead {
    Raw v[K][R];
    template <typename G> __device__ __forceinline__ void start(int mine, G get)
    {
#pragma unroll
        for (int u = 0; u < R; ++u)
            if (u < mine) get(v, u, u);
    }
    template <typename G, typename F> __device__ __forceinline__ void run(int mine, G get, F f)
    {
        for (int i = 0; i < mine; i += R) {
            Raw n[K][R];
#pragma unroll
            for (int u = 0; u < R; ++u)
                if (i + R + u < mine) get(n, u, i + R + u);
#pragma unroll
            for (int u = 0; u < R; ++u)
                if (i + u < mine) f(v, u, i + u);
#pragma unroll
            for (int u = 0; u < R; ++u)
#pragma unroll
                for (int k = 0; k < K; ++k) v[k][u] = n[k][u];
        }
    }
};

// mean and rstd of the slab's groups
__device__ __forceinline__ void slab_stats(const Args &a, const Place &pc, float *s_mean, float *s_rstd)
{
    const int g0 = pc.g0(a);
    if (a.finished) {
        for (int g = threadIdx.x; g < pc.ng; g += kT) {
            s_mean[g] = a.mean[(size_t)pc.n * a.G + g0 + g];
            s_rstd[g] = a.rstd[(size_t)pc.n * a.G + g0 + g];
        }
        return;
    }
    by_group(pc.ng, [&](int g, int k, int tpg) {
        float mu, rs;
        join_ranges(a, pc.n, g0 + g, k, tpg, mu, rs);
        if (k == 0) {
            s_mean[g] = mu;
            s_rstd[g] = rs;
            if (pc.blk == 0) {
                a.mean[(size_t)pc.n * a.G + g0 + g] = mu;
                a.rstd[(size_t)pc.n * a.G + g0 + g] = rs;
            }
        }
    });
}

// ---- forward, second pass.  Every workgroup joins its sample's ranges for itself: no launch between the passes.  Large: 93 us, 6.5 TB/s
// (the residual is read once for its four pixels: 603 MB); 16 x 64 x 32 x 256 bf16 9.1 us
template <typename T, int V, int A, int ACT, bool NT> __global__ __launch_bounds__(kT) void k_gn_apply(const Args a)
{
    constexpr int S = V / A;
    typedef typename IO<T, V>::raw raw;
    __shared__ float s_mean[kT * A], s_rstd[kT * A];
    const Place pc(a, blockIdx.x, V);
    const int mine = vectors_of(a, pc);
    const size_t base = (size_t)pc.n * a.hw * a.C + pc.c0, step = (size_t)a.PL * a.C;
    const T *x = (const T *)a.x + base;
    T *y = (T *)a.y + base;
    float k[V], b[V], mu[A];
    auto coefficients = [&]() {
        affine<V>(a, pc, k, b);
        slab_stats(a, pc, s_mean, s_rstd);
        __syncthreads();
        if (!pc.on) return;
#pragma unroll
        for (int j = 0; j < A; ++j) {
            const int g = (int)a.by_sg.of((unsigned)(pc.lv * A + j));
            mu[j] = s_mean[g];
#pragma unroll
            for (int u = 0; u < S; ++u) k[j * S + u] *= s_rstd[g];
        }
    };
    if (a.quad) {   // the residual is read once for its four pixels
        const T *res = (const T *)a.res + (size_t)pc.n * a.items * a.C + pc.c0;
        const size_t row = (size_t)2 * a.W2 * a.C;
        const long long i0 = pc.i0 + pc.pl;
        Ahead<1, raw, 5> w;
        auto get = [&](raw (&v)[5][1], int, int i) {
            const long long q = i0 + (long long)i * a.PL;
            const T *p = x + (size_t)first_pixel(a, q) * a.C;
            v[0][0] = IO<T, V>::template load<NT>(p);
            v[1][0] = IO<T, V>::template load<NT>(p + a.C);
            v[2][0] = IO<T, V>::template load<NT>(p + row);
            v[3][0] = IO<T, V>::template load<NT>(p + row + a.C);
            v[4][0] = IO<T, V>::template load<NT>(res + (size_t)q * a.C);
        };
        w.start(mine, get);
        coefficients();
        w.run(mine, get, [&](raw (&v)[5][1], int, int i) {
            T *p = y + (size_t)first_pixel(a, i0 + (long long)i * a.PL) * a.C;
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                float f[V];
                IO<T, V>::open(v[u][0], f);
                finish_store<T, V, A, ACT, NT>(a, f, mu, k, b, true, v[4][0], p + (u & 1) * a.C + (u >> 1) * row);
            }
        });
        return;
    }
    const T *res = a.res ? (const T *)a.res + base : nullptr;
    const size_t o = (size_t)(pc.i0 + pc.pl) * a.C;
    Ahead<2, raw, 2> w;
    auto get = [&](raw (&v)[2][2], int u, int i) {
        v[0][u] = IO<T, V>::template load<NT>(x + o + i * step);
        if (res) v[1][u] = IO<T, V>::template load<NT>(res + o + i * step);
    };
    w.start(mine, get);
    coefficients();
    w.run(mine, get, [&](raw (&v)[2][2], int u, int i) {
        float f[V];
        IO<T, V>::open(v[0][u], f);
        finish_store<T, V, A, ACT, NT>(a, f, mu, k, b, res != nullptr, v[1][u], y + o + i * step);
    });
}

// statistics and affine of the thread's channels for the backward: k = rstd * w as the forward multiplied it
template <int V, int A>
__device__ __forceinline__ void saved(const Args &a, const Place &pc, float (&mu)[A], float (&rs)[A], float (&k)[V], float (&b)[V])
{
    constexpr int S = V / A;
    affine<V>(a, pc, k, b);
#pragma unroll
    for (int j = 0; j < A; ++j) {
        const size_t g = (size_t)pc.n * a.G + (pc.on ? a.by_d.of((unsigned)(pc.c0 + j * S)) : 0u);
        mu[j] = a.mean[g];
        rs[j] = a.rstd[g];
#pragma unroll
        for (int u = 0; u < S; ++u) k[j * S + u] *= rs[j];
    }
}

// joins the threads' per-channel sums (t1: dz, t2: dz (x - mean)): cpart row `row` (unless NULL), and per group
// s1 / s2 [groups of the slab] = sum w dz, sum w dz xhat.  sh1, sh2: kT * (V + 1)
template <int V, int A>
__device__ __forceinline__ void join_grads(const Args &a, const Place &pc, const float (&t1)[V], const float (&t2)[V], const float (&rs)[A],
                                           float *sh1, float *sh2, float *s1, float *s2, float *out1, float *out2)
{
    constexpr int S = V / A;
    const int cols = a.LV * V, stride = cols | 1;
    if (pc.pl < a.PL) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
            sh1[pc.pl * stride + pc.lv * V + j] = pc.on ? t1[j] : 0.0f;
            sh2[pc.pl * stride + pc.lv * V + j] = pc.on ? t2[j] * rs[j / S] : 0.0f;
        }
    }
    __syncthreads();
    const int cs = pc.slab * a.SC, nc = pc.ng * a.D;
    by_group(nc, [&](int c, int k, int tpg) {
        float u1 = 0.0f, u2 = 0.0f;
#pragma unroll 2
        for (int r = k; r < a.PL; r += tpg) {
            u1 += sh1[r * stride + c];
            u2 += sh2[r * stride + c];
        }
        u1 = lanes_sum(u1, tpg);
        u2 = lanes_sum(u2, tpg);
        if (k == 0) {
            if (out1) out1[cs + c] = u1;
            if (out2) out2[cs + c] = u2;
            const float w = a.w ? a.w[(size_t)pc.n * a.aff_stride + cs + c] + a.w_off : 1.0f;
            sh1[c] = w * u1;   // (row 0 of this column: read by this thread's own lanes only, before this)
            sh2[c] = w * u2;
        }
    });
    __syncthreads();
    by_group(pc.ng, [&](int g, int k, int tpg) {
        float u1 = 0.0f, u2 = 0.0f;
        for (int c = k; c < a.D; c += tpg) {
            u1 += sh1[g * a.D + c];
            u2 += sh2[g * a.D + c];
        }
        u1 = lanes_sum(u1, tpg);
        u2 = lanes_sum(u2, tpg);
        if (k == 0) {
            s1[g] = u1;
            s2[g] = u2;
        }
    });
}

// ---- backward, first pass: per-channel sums of dz and dz xhat, their weighted sums per group; the half-resolution residual's gradient (from
// the dy that is here anyway: a kernel of its own would read it again).  Sums are kept per channel in registers over the whole range, so a
// range costs one join.  Large: 118 us, 5.1 TB/s (604 MB); 16 x 64 x 32 x 256 bf16 11.0 us
template <typename T, int V, int A, int ACT, bool NT>
__device__ __forceinline__ void grads_of_range(const Args &a, unsigned id, float *sh1, float *sh2, float *s1, float *s2)
{
    const Place pc(a, id, V);
    const size_t base = (size_t)pc.n * a.hw * a.C + pc.c0;
    const T *x = (const T *)a.x + base, *dy = (const T *)a.dy + base;
    float mu[A], rs[A], k[V], b[V], t1[V], t2[V];
    saved<V, A>(a, pc, mu, rs, k, b);
#pragma unroll
    for (int j = 0; j < V; ++j) t1[j] = t2[j] = 0.0f;
    auto add = [&](const typename IO<T, V>::raw &vx, const float (&d)[V]) {
        float f[V], xc[V], dz[V];
        IO<T, V>::open(vx, f);
        grad_of<V, A, ACT>(a, f, d, mu, k, b, xc, dz);
#pragma unroll
        for (int j = 0; j < V; ++j) {
            t1[j] += dz[j];
            t2[j] += dz[j] * xc[j];
        }
    };
    if (pc.on && a.quad) {
        const size_t row = (size_t)2 * a.W2 * a.C;
        T *dres = (T *)a.dres + (size_t)pc.n * a.items * a.C + pc.c0, *last = nullptr;
        typename IO<T, V>::raw kept = {};   // (stored behind the next loads, as the forward does)
#pragma unroll 1
        for (long long i = pc.i0 + pc.pl; i < pc.i0 + pc.ni; i += a.PL) {
            const size_t o = (size_t)first_pixel(a, i) * a.C;
            const size_t at[4] = {o, o + a.C, o + row, o + row + a.C};
            typename IO<T, V>::raw vx[4], vd[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                vx[u] = IO<T, V>::load(x + at[u]);
                vd[u] = IO<T, V>::load(dy + at[u]);
            }
            if (last) IO<T, V>::template put<NT>(last, kept);
            float sum[V];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                float d[V];
                IO<T, V>::open(vd[u], d);
#pragma unroll
                for (int j = 0; j < V; ++j) sum[j] = u ? sum[j] + d[j] : d[j];
                add(vx[u], d);
                __builtin_amdgcn_sched_barrier(0);   // (one vector at a time is enough arithmetic: fewer registers, more waves)
            }
            if (a.dres) {
                kept = IO<T, V>::pack(sum);
                last = dres + (size_t)i * a.C;
            }
        }
        if (last) IO<T, V>::template put<NT>(last, kept);
    } else if (pc.on) {
        constexpr int R = 4;
        const size_t step = (size_t)a.PL * a.C;
        const int mine = vectors_of(a, pc);
        size_t o = (size_t)(pc.i0 + pc.pl) * a.C;
        int i = 0;
#pragma unroll 1
        for (; i + R <= mine; i += R, o += R * step) {
            typename IO<T, V>::raw vx[R], vd[R];
#pragma unroll
            for (int u = 0; u < R; ++u) {
                vx[u] = IO<T, V>::load(x + o + u * step);
                vd[u] = IO<T, V>::load(dy + o + u * step);
            }
#pragma unroll
            for (int u = 0; u < R; ++u) {
                float d[V];
                IO<T, V>::open(vd[u], d);
                add(vx[u], d);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        for (; i < mine; ++i, o += step) {
            float d[V];
            IO<T, V>::open(IO<T, V>::load(dy + o), d);
            add(IO<T, V>::load(x + o), d);
        }
    }
    float *cp = a.cpart ? a.cpart + ((size_t)pc.n * a.gnblk + pc.blk) * 2 * a.C : nullptr;
    join_grads<V, A>(a, pc, t1, t2, rs, sh1, sh2, s1, s2, cp, cp ? cp + a.C : nullptr);
    __syncthreads();
    float2 *out = a.gpart + ((size_t)pc.n * a.gnblk + pc.blk) * a.G + pc.g0(a);
    for (int g = threadIdx.x; g < pc.ng; g += kT) out[g] = make_float2(s1[g], s2[g]);
}

template <typename T, int V, int A, int ACT, bool NT> __global__ __launch_bounds__(kT) void k_gn_bwd_reduce(const Args a)
{
    __shared__ float sh1[kT * (V + 1)], sh2[kT * (V + 1)], s1[kT * A], s2[kT * A];
    grads_of_range<T, V, A, ACT, NT>(a, blockIdx.x, sh1, sh2, s1, s2);
}

__device__ __forceinline__ float2 join_group_grads(const Args &a, int n, int g, int k, int tpg)
{
    const float2 *p = a.gpart + (size_t)n * a.gnblk * a.G + g;
    const float m = (float)((double)a.hw * a.D);
    float u1 = 0.0f, u2 = 0.0f;
#pragma unroll 4
    for (int i = k; i < a.gnblk; i += tpg) {
        const float2 v = p[(size_t)i * a.G];
        u1 += v.x;
        u2 += v.y;
    }
    return make_float2(lanes_sum(u1, tpg) / m, lanes_sum(u2, tpg) / m);
}

static __global__ __launch_bounds__(kT) void k_gn_bwd_finish(const Args a)
{
    const long long i = ((long long)blockIdx.x * kT + threadIdx.x) >> 6;
    if (i >= (long long)a.N * a.G) return;
    const int n = (int)(i / a.G), g = (int)(i - (long long)n * a.G), k = threadIdx.x & 63;
    const float2 u = join_group_grads(a, n, g, k, 64);
    if (k == 0) a.gsum[i] = u;
}

// dx of one vector
template <typename T, int V, int A, int ACT, bool NT>
__device__ __forceinline__ void dx_store(const Args &a, const float (&f)[V], const float (&d)[V], const float (&mu)[A], const float (&rs)[A],
                                         const float (&k)[V], const float (&b)[V], const float (&u1)[A], const float (&u2)[A], T *dx)
{
    constexpr int S = V / A;
    float xc[V], dz[V];
    grad_of<V, A, ACT>(a, f, d, mu, k, b, xc, dz);
    // rstd (w dz - u1 - xc rstd u2) with k = rstd w, u1 and u2 already times rstd and rstd^2
#pragma unroll
    for (int j = 0; j < V; ++j) xc[j] = k[j] * dz[j] - (u1[j / S] + xc[j] * u2[j / S]);
    IO<T, V>::template store<NT>(dx, xc);
}

// ---- backward, second pass: dx.  Large: 126 us, 6.4 TB/s (805 MB); 16 x 64 x 32 x 256 bf16 9.9 us
template <typename T, int V, int A, int ACT, bool NT> __global__ __launch_bounds__(kT) void k_gn_bwd_apply(const Args a)
{
    typedef typename IO<T, V>::raw raw;
    __shared__ float s1[kT * A], s2[kT * A];
    const Place pc(a, blockIdx.x, V);
    const int mine = vectors_of(a, pc), g0 = pc.g0(a);
    const size_t base = (size_t)pc.n * a.hw * a.C + pc.c0 + (size_t)(pc.i0 + pc.pl) * a.C, step = (size_t)a.PL * a.C;
    const T *x = (const T *)a.x + base, *dy = (const T *)a.dy + base;
    T *dx = (T *)a.y + base;
    Ahead<2, raw, 2> w;
    auto get = [&](raw (&v)[2][2], int u, int i) {
        v[0][u] = IO<T, V>::template load<NT>(x + i * step);
        v[1][u] = IO<T, V>::template load<NT>(dy + i * step);
    };
    w.start(mine, get);
    float mu[A], rs[A], k[V], b[V], u1[A], u2[A];
    saved<V, A>(a, pc, mu, rs, k, b);
    if (a.finished) {
        for (int g = threadIdx.x; g < pc.ng; g += kT) {
            const float2 v = a.gsum[(size_t)pc.n * a.G + g0 + g];
            s1[g] = v.x;
            s2[g] = v.y;
        }
    } else {
        by_group(pc.ng, [&](int g, int k, int tpg) {
            const float2 v = join_group_grads(a, pc.n, g0 + g, k, tpg);
            if (k == 0) {
                s1[g] = v.x;
                s2[g] = v.y;
            }
        });
    }
    __syncthreads();
    if (!pc.on) return;
#pragma unroll
    for (int j = 0; j < A; ++j) {
        const int g = (int)a.by_sg.of((unsigned)(pc.lv * A + j));
        u1[j] = s1[g] * rs[j];
        u2[j] = s2[g] * rs[j] * rs[j];
    }
    w.run(mine, get, [&](raw (&v)[2][2], int u, int i) {
        float f[V], d[V];
        IO<T, V>::open(v[0][u], f);
        IO<T, V>::open(v[1][u], d);
        dx_store<T, V, A, ACT, NT>(a, f, d, mu, rs, k, b, u1, u2, dx + i * step);
    });
}

// ---- dw / db from cpart (3 to 5 us: the launch and one way to memory): row blockIdx.y of the result (a sample, or the one row) adds `rows` partial rows `gap` apart; `all` rows lie
// between two results' first ones.  With `chunk` < rows a workgroup adds rows [z chunk, (z + 1) chunk) and leaves the sum in the first of
// them, which no other one reads
static __global__ __launch_bounds__(1024) void k_gn_affine_grad(float *cpart, float *dw, float *db, int C, long long all, long long rows,
                                                                long long gap, long long chunk)
{
    __shared__ float s1[32][33], s2[32][33];
    const int cl = threadIdx.x & 31, rl = threadIdx.x >> 5;
    const int c = blockIdx.x * 32 + cl;
    const bool part = chunk < rows;
    const long long z0 = (long long)blockIdx.z * chunk, end = min(rows, z0 + chunk);
    float *from = cpart + (size_t)blockIdx.y * all * 2 * C;
    float t1 = 0.0f, t2 = 0.0f;
    if (c < C) {
#pragma unroll 4
        for (long long r = z0 + rl; r < end; r += 32) {
            t1 += from[r * gap * 2 * C + c];
            t2 += from[(r * gap * 2 + 1) * C + c];
        }
    }
    s1[rl][cl] = t1;
    s2[rl][cl] = t2;
    __syncthreads();
    for (int h = 16; h > 0; h >>= 1) {
        if (rl < h) {
            s1[rl][cl] += s1[rl + h][cl];
            s2[rl][cl] += s2[rl + h][cl];
        }
        __syncthreads();
    }
    if (rl == 0 && c < C) {
        float *o1 = part ? from + z0 * gap * 2 * C : db ? db + (size_t)blockIdx.y * C : nullptr;
        float *o2 = part ? from + (z0 * gap * 2 + 1) * C : dw ? dw + (size_t)blockIdx.y * C : nullptr;
        if (o1) o1[c] = s1[0][cl];
        if (o2) o2[c] = s2[0][cl];
    }
}

// ---- a slab of a sample in the registers of one workgroup: one pass.  R vectors a thread.  8 x 4 x 512 bf16: one sample 5.4 us (the launch,
// one way to memory and back, three joins in LDS); 16 samples 6.0 forward, 6.3 backward
// pixel of a thread's vector r: every PL-th pixel, or -- quad -- four of every PL-th 2 x 2 block
template <int R> __device__ __forceinline__ bool held_at(const Args &a, const Place &pc, int r, unsigned &pix)
{
    if (!a.quad) {
        const unsigned p = (unsigned)(pc.pl + r * a.PL);
        pix = p;
        return pc.on && p < (unsigned)a.items;
    }
    const unsigned i = (unsigned)(pc.pl + (r >> 2) * a.PL);
    const bool ok = pc.on && i < (unsigned)a.items;
    const unsigned h = a.by_w2.of(i);
    pix = 2 * (i + h * (unsigned)a.W2) + (r & 1) + ((r & 2) ? 2 * (unsigned)a.W2 : 0u);
    return ok;
}

template <typename T, int V, int A, int ACT, int R> __global__ __launch_bounds__(kT) void k_gn_one(const Args a)
{
    constexpr int S = V / A;
    __shared__ float sh[kT * (A + 1)], s_mean[kT * A], s_m2[kT * A];
    const Place pc(a, blockIdx.x, V);
    const size_t base = (size_t)pc.n * a.hw * a.C + pc.c0;
    const T *x = (const T *)a.x + base;
    typename IO<T, V>::raw v[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        unsigned p;
        const bool ok = held_at<R>(a, pc, r, p);
        v[r] = ok ? IO<T, V>::load(x + (size_t)p * a.C) : typename IO<T, V>::raw(T(0));
    }
    Stat<V, A> st;
    st.start();
    int mine = 0;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        unsigned p;
        mine += held_at<R>(a, pc, r, p) ? 1 : 0;
    }
    // (all the thread's values are here: K is their mean, the deviations are exact to rounding)
    const float part = mine > 0 ? 1.0f / (float)(mine * S) : 0.0f;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        float f[V];
        IO<T, V>::open(v[r], f);
        st.about(f, 1.0f);
    }
#pragma unroll
    for (int k = 0; k < A; ++k) st.K[k] *= part;
#pragma unroll
    for (int r = 0; r < R; ++r) keep(v[r]);
#pragma unroll
    for (int r = 0; r < R; ++r) {
        unsigned p;
        if (held_at<R>(a, pc, r, p)) {
            float f[V];
            IO<T, V>::open(v[r], f);
            st.add(f);
        }
    }
    st.close((float)mine);
#pragma unroll
    for (int r = 0; r < R; ++r) keep(v[r]);
    float k[V], b[V], mu[A];
    affine<V>(a, pc, k, b);
    join_threads<V, A>(a, pc, st, (float)mine, (float)a.hw, sh, s_mean, s_m2);
    __syncthreads();
    const int g0 = pc.g0(a);
    const float m = (float)((double)a.hw * a.D);
    for (int g = threadIdx.x; g < pc.ng; g += kT) {
        const float rs = 1.0f / sqrtf(s_m2[g] / m + a.eps);
        a.mean[(size_t)pc.n * a.G + g0 + g] = s_mean[g];
        a.rstd[(size_t)pc.n * a.G + g0 + g] = rs;
        s_m2[g] = rs;
    }
    __syncthreads();
    if (!pc.on) return;
#pragma unroll
    for (int j = 0; j < A; ++j) {
        const int g = (int)a.by_sg.of((unsigned)(pc.lv * A + j));
        mu[j] = s_mean[g];
#pragma unroll
        for (int u = 0; u < S; ++u) k[j * S + u] *= s_m2[g];
    }
    T *y = (T *)a.y + base;
    const T *res = a.res ? (const T *)a.res + (size_t)pc.n * (a.quad ? a.items : a.hw) * a.C + pc.c0 : nullptr;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        unsigned p;
        if (held_at<R>(a, pc, r, p)) {
            float f[V];
            IO<T, V>::open(v[r], f);
            const unsigned i = a.quad ? (unsigned)(pc.pl + (r >> 2) * a.PL) : p;
            typename IO<T, V>::raw q = {};
            if (res) q = IO<T, V>::load(res + (size_t)i * a.C);
            finish_store<T, V, A, ACT, false>(a, f, mu, k, b, res != nullptr, q, y + (size_t)p * a.C);
        }
    }
}

// the backward in one pass: x and dy of the slab in registers; with an affine of its own a sample writes dw / db, else cpart rows
template <typename T, int V, int A, int ACT, int R> __global__ __launch_bounds__(kT) void k_gn_bwd_one(const Args a)
{
    __shared__ float sh1[kT * (V + 1)], sh2[kT * (V + 1)], s1[kT * A], s2[kT * A];
    const Place pc(a, blockIdx.x, V);
    const size_t base = (size_t)pc.n * a.hw * a.C + pc.c0;
    const T *x = (const T *)a.x + base, *dy = (const T *)a.dy + base;
    typename IO<T, V>::raw vx[R], vd[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        unsigned p;
        const bool ok = held_at<R>(a, pc, r, p);
        vx[r] = ok ? IO<T, V>::load(x + (size_t)p * a.C) : typename IO<T, V>::raw(T(0));
        vd[r] = ok ? IO<T, V>::load(dy + (size_t)p * a.C) : typename IO<T, V>::raw(T(0));
    }
    float mu[A], rs[A], k[V], b[V], t1[V], t2[V];
    saved<V, A>(a, pc, mu, rs, k, b);
#pragma unroll
    for (int j = 0; j < V; ++j) t1[j] = t2[j] = 0.0f;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        unsigned p;
        if (!held_at<R>(a, pc, r, p)) continue;
        float f[V], d[V], xc[V], dz[V];
        IO<T, V>::open(vx[r], f);
        IO<T, V>::open(vd[r], d);
        grad_of<V, A, ACT>(a, f, d, mu, k, b, xc, dz);
#pragma unroll
        for (int j = 0; j < V; ++j) {
            t1[j] += dz[j];
            t2[j] += dz[j] * xc[j];
        }
        __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
        keep(vx[r]);
        keep(vd[r]);
    }
    float *o1 = nullptr, *o2 = nullptr;
    if (a.per_sample) {
        if (a.db) o1 = a.db + (size_t)pc.n * a.C;
        if (a.dw) o2 = a.dw + (size_t)pc.n * a.C;
    } else if (a.dw || a.db) {
        o1 = a.cpart + (size_t)pc.n * 2 * a.C;
        o2 = o1 + a.C;
    }
    join_grads<V, A>(a, pc, t1, t2, rs, sh1, sh2, s1, s2, o1, o2);
    __syncthreads();
    if (!pc.on) return;
    const float m = (float)((double)a.hw * a.D);
    float u1[A], u2[A];
#pragma unroll
    for (int j = 0; j < A; ++j) {
        const int g = (int)a.by_sg.of((unsigned)(pc.lv * A + j));
        u1[j] = s1[g] / m * rs[j];
        u2[j] = s2[g] / m * rs[j] * rs[j];
    }
    if (a.y) {
        T *dx = (T *)a.y + base;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            unsigned p;
            if (!held_at<R>(a, pc, r, p)) continue;
            float f[V], d[V];
            IO<T, V>::open(vx[r], f);
            IO<T, V>::open(vd[r], d);
            dx_store<T, V, A, ACT, false>(a, f, d, mu, rs, k, b, u1, u2, dx + (size_t)p * a.C);
            __builtin_amdgcn_sched_barrier(0);
        }
    }
    if (a.dres) {
        if constexpr (R >= 4) {
            T *dres = (T *)a.dres + (size_t)pc.n * a.items * a.C + pc.c0;
#pragma unroll
            for (int r = 0; r < R; r += 4) {
                unsigned p;
                if (!held_at<R>(a, pc, r, p)) continue;
                float d0[V], d1[V], d2[V], d3[V];
                IO<T, V>::open(vd[r], d0);
                IO<T, V>::open(vd[r + 1], d1);
                IO<T, V>::open(vd[r + 2], d2);
                IO<T, V>::open(vd[r + 3], d3);
#pragma unroll
                for (int j = 0; j < V; ++j) d0[j] = ((d0[j] + d1[j]) + d2[j]) + d3[j];
                IO<T, V>::template store<false>(dres + (size_t)(pc.pl + (r >> 2) * a.PL) * a.C, d0);
            }
        }
    }
}

// ------------------------------------------------------------------------------------------------ launches (one per element type)
// what the host chose: vector, segments, and the vectors a thread of the one-pass kernels holds
struct Choice {
    int V, A, R;
};
struct Runner {
    void (*stats)(const Args &, int V, int A, hipStream_t);
    void (*apply)(const Args &, int V, int A, hipStream_t);
    void (*bwd_reduce)(const Args &, int V, int A, hipStream_t);
    void (*bwd_apply)(const Args &, int V, int A, hipStream_t);
    void (*one)(const Args &, const Choice &, hipStream_t);
    void (*bwd_one)(const Args &, const Choice &, hipStream_t);
};
Runner run_f32();
Runner run_f16();
Runner run_bf16();

}  // namespace gn
}  // namespace m355
