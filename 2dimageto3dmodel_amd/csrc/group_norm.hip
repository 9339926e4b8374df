// Group norm with an activation on channels-last tensors, forward and backward (include/m355.h m355_group_norm_*).
//
//   m = HW * D values per (sample, group of D = C / G neighbouring channels)
//   mean = sum x / m,  var = sum (x - mean)^2 / m,  rstd = 1 / sqrt(var + eps),  xhat = (x - mean) rstd
//   z = xhat * w + b,  y = act(z) [+ res],  act = LeakyReLU(slope) or SiLU z / (1 + e^-z)
//   backward, dz = dy act'(z):  db = sum_hw dz,  dw = sum_hw dz xhat,
//   dx = rstd (w dz - mean_g(w dz) - xhat mean_g(w dz xhat)),  dres = dy (2 x 2 sums when res is stored at half resolution)
//
// Bound: HBM.  About 10 (forward) / 25 (backward) operations a value against 4 / 6 bytes in 16 bits.
//
// Statistics never subtract two large numbers: a thread takes the mean of the few values it has in registers, adds their squared
// deviations from THAT, and every join of two parts (a, b) adds delta^2 n_a n_b / (n_a + n_b) with delta the difference of their
// means.  All sums are 32-bit, in a fixed order: the same bits on every run.
#include <type_traits>

#include "common.h"

namespace m355 {
namespace gn {

template <typename T, int V> using vec = T __attribute__((ext_vector_type(V)));
// element-aligned form: a sample's rows may start anywhere a multiple of the vector's channel count allows
template <typename T, int V> struct VecIO {
    static __device__ __forceinline__ void load(const T *p, float (&f)[V])
    {
        const vec<T, V> v = *reinterpret_cast<const vec<T, V> *>(p);
#pragma unroll
        for (int j = 0; j < V; ++j) f[j] = (float)v[j];
    }
    static __device__ __forceinline__ void store(T *p, const float (&f)[V])
    {
        vec<T, V> v;
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] = (T)f[j];   // round to nearest even, once, from the 32-bit result
        *reinterpret_cast<vec<T, V> *>(p) = v;
    }
};
template <typename T> struct VecIO<T, 1> {
    static __device__ __forceinline__ void load(const T *p, float (&f)[1]) { f[0] = (float)*p; }
    static __device__ __forceinline__ void store(T *p, const float (&f)[1]) { *p = (T)f[0]; }
};

struct Args {
    const void *x, *dy, *res;
    void *y;                      // forward: y; backward: dx
    void *dres;
    const float *w, *b;           // NULL: 1 / 0
    float *mean, *rstd;           // [N][G]
    float2 *gpart;                // [N][nblk][G]: forward (mean, M2); backward (sum w dz, sum w dz xhat)
    float *cpart;                 // backward [N][nblk][2][C]: (sum dz, sum dz xhat)
    long long aff_stride;         // floats between the samples' rows of w and b (0: one row for all)
    long long hw, ppb;            // pixels of a sample; pixels of a workgroup's range
    int N, C, G, D;
    int SC, LV, PL, nslab;        // channels of a slab (whole groups, whole vectors), vectors across it, pixel lanes, slabs
    int nblk;                     // pixel ranges of a sample
    int act, res_w;               // res_w > 0: res is [N][H/2][res_w/2][C]
    float w_off, eps, slope, out_slope;
};

constexpr int kT = 256;           // threads of a workgroup

__device__ __forceinline__ float wave_sum(float v)
{
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

// (n, mean, M2) joined with (nb, mb, Mb)
__device__ __forceinline__ void join(float &n, float &mean, float &M2, float nb, float mb, float Mb)
{
    const float t = n + nb;
    if (nb > 0.0f) {
        const float r = nb / t, d = mb - mean;
        mean += d * r;
        M2 += Mb + d * d * n * r;
        n = t;
    }
}

__device__ __forceinline__ float sigmoid(float z) { return __builtin_amdgcn_rcpf(1.0f + __expf(-z)); }

struct Place {   // what a workgroup and a thread of it own
    int n, slab, blk, lv, pl, c0, ng;   // ng: groups of the slab
    bool on;
    long long p0, np;
    __device__ __forceinline__ Place(const Args &a, long long id, int V)
    {
        blk = (int)(id % a.nblk);
        id /= a.nblk;
        slab = (int)(id % a.nslab);
        n = (int)(id / a.nslab);
        lv = (int)threadIdx.x % a.LV;
        pl = (int)threadIdx.x / a.LV;
        c0 = slab * a.SC + lv * V;
        on = pl < a.PL && c0 < a.C;
        ng = min(a.SC, a.C - slab * a.SC) / a.D;
        p0 = (long long)blk * a.ppb;
        np = min(a.ppb, a.hw - p0);
    }
};

__host__ __device__ __forceinline__ long long n_work(const Args &a) { return (long long)a.N * a.nslab * a.nblk; }

// the affine of the thread's channels
template <int V> __device__ __forceinline__ void affine(const Args &a, const Place &pc, float (&w)[V], float (&b)[V])
{
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const long long i = (long long)pc.n * a.aff_stride + pc.c0 + j;
        w[j] = (pc.on && a.w) ? a.w[i] + a.w_off : 1.0f;
        b[j] = (pc.on && a.b) ? a.b[i] : 0.0f;
    }
}

// ---- forward, first pass: gpart[n][blk][g] = (mean, M2) of the workgroup's pixels
template <typename T, int V> __global__ __launch_bounds__(kT) void k_gn_stats(const Args a)
{
    constexpr int R = 4;   // loads in flight a thread
    __shared__ float sm[kT * V], sq[kT * V], sn[kT];
    for (long long id = blockIdx.x; id < n_work(a); id += gridDim.x) {
        const Place pc(a, id, V);
        const T *x = (const T *)a.x + ((size_t)pc.n * a.hw + pc.p0) * a.C + pc.c0;
        float n = 0.0f, mean[V], M2[V];
#pragma unroll
        for (int j = 0; j < V; ++j) mean[j] = M2[j] = 0.0f;
        if (pc.on) {
            long long p = pc.pl;
            for (; p + (long long)(R - 1) * a.PL < pc.np; p += (long long)R * a.PL) {
                float f[R][V];
#pragma unroll
                for (int u = 0; u < R; ++u) VecIO<T, V>::load(x + (size_t)(p + (long long)u * a.PL) * a.C, f[u]);
                const float t = n + R, r = R / t;
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    float s = 0.0f, q = 0.0f;
#pragma unroll
                    for (int u = 0; u < R; ++u) s += f[u][j];
                    s *= 1.0f / R;
#pragma unroll
                    for (int u = 0; u < R; ++u) q += (f[u][j] - s) * (f[u][j] - s);
                    const float d = s - mean[j];
                    mean[j] += d * r;
                    M2[j] += q + d * d * n * r;
                }
                n = t;
            }
            for (; p < pc.np; p += a.PL) {
                float f[V];
                VecIO<T, V>::load(x + (size_t)p * a.C, f);
                const float t = n + 1.0f, r = 1.0f / t;
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const float d = f[j] - mean[j];
                    mean[j] += d * r;
                    M2[j] += d * d * n * r;
                }
                n = t;
            }
        }
        // over the pixel lanes (a tree of joins), then over the channels of a group
        const int tid = threadIdx.x;
        __syncthreads();
        if (pc.pl < a.PL) {
            if (pc.lv == 0) sn[pc.pl] = (float)max(0LL, (pc.np - pc.pl + a.PL - 1) / a.PL);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                sm[tid * V + j] = mean[j];
                sq[tid * V + j] = M2[j];
            }
        }
        __syncthreads();
        for (int w = a.PL; w > 1;) {
            const int h = (w + 1) >> 1;
            float nn = 0.0f, nb = 0.0f;
            if (pc.pl + h < w) {
                const int o = (tid + h * a.LV) * V;
                nb = sn[pc.pl + h];
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    nn = sn[pc.pl];
                    join(nn, sm[tid * V + j], sq[tid * V + j], nb, sm[o + j], sq[o + j]);
                }
            }
            __syncthreads();
            if (pc.pl + h < w && pc.lv == 0) sn[pc.pl] += nb;
            __syncthreads();
            w = h;
        }
        const int lane = tid & 63, wave = tid >> 6;
        const float np = (float)pc.np;
        for (int g = wave; g < pc.ng; g += kT / 64) {
            float s = 0.0f, q = 0.0f;
            for (int c = lane; c < a.D; c += 64) s += sm[g * a.D + c];
            const float mu = wave_sum(s) / (float)a.D;
            for (int c = lane; c < a.D; c += 64) {
                const float d = sm[g * a.D + c] - mu;
                q += sq[g * a.D + c] + np * d * d;
            }
            q = wave_sum(q);
            if (lane == 0)
                a.gpart[((size_t)pc.n * a.nblk + pc.blk) * a.G + (size_t)pc.slab * (a.SC / a.D) + g] = make_float2(mu, q);
        }
    }
}

// mean and rstd of the slab's groups from the partial ones -> s_mean / s_rstd [groups of the slab]
__device__ __forceinline__ void join_partials(const Args &a, const Place &pc, float *s_mean, float *s_rstd)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g0 = pc.slab * (a.SC / a.D);
    const float m = (float)((double)a.hw * a.D);
    for (int g = wave; g < pc.ng; g += kT / 64) {
        const float2 *p = a.gpart + (size_t)pc.n * a.nblk * a.G + g0 + g;
        float s = 0.0f;
        for (int k = lane; k < a.nblk; k += 64)
            s += p[(size_t)k * a.G].x * ((float)min(a.ppb, a.hw - (long long)k * a.ppb) * a.D);
        const float mu = wave_sum(s) / m;
        float q = 0.0f;
        for (int k = lane; k < a.nblk; k += 64) {
            const float2 v = p[(size_t)k * a.G];
            const float d = v.x - mu;
            q += v.y + d * d * ((float)min(a.ppb, a.hw - (long long)k * a.ppb) * a.D);
        }
        const float rs = 1.0f / sqrtf(wave_sum(q) / m + a.eps);
        if (lane == 0) {
            s_mean[g] = mu;
            s_rstd[g] = rs;
            if (pc.blk == 0) {
                a.mean[(size_t)pc.n * a.G + g0 + g] = mu;
                a.rstd[(size_t)pc.n * a.G + g0 + g] = rs;
            }
        }
    }
}

// y of one vector
template <typename T, int V>
__device__ __forceinline__ void act_store(const Args &a, const float (&f)[V], const float (&mu)[V], const float (&k)[V], const float (&b)[V],
                                          const T *res, T *y, long long p, long long n)
{
    float z[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        z[j] = (f[j] - mu[j]) * k[j] + b[j];
        z[j] = a.act == 0 ? (z[j] >= 0.0f ? z[j] : z[j] * a.slope) : z[j] * sigmoid(z[j]);
    }
    if (res) {
        float r[V];
        long long q = n * a.hw + p;
        if (a.res_w > 0) {
            const long long h = p / a.res_w, w = p - h * a.res_w;
            q = n * (a.hw / 4) + (h >> 1) * (a.res_w >> 1) + (w >> 1);
        }
        VecIO<T, V>::load(res + (size_t)q * a.C, r);
#pragma unroll
        for (int j = 0; j < V; ++j) z[j] += r[j];
    }
    if (a.out_slope != 1.0f) {
#pragma unroll
        for (int j = 0; j < V; ++j) z[j] = z[j] >= 0.0f ? z[j] : z[j] * a.out_slope;
    }
    VecIO<T, V>::store(y, z);
}

// ---- forward, second pass
template <typename T, int V> __global__ __launch_bounds__(kT) void k_gn_apply(const Args a)
{
    __shared__ float s_mean[kT * V], s_rstd[kT * V];
    for (long long id = blockIdx.x; id < n_work(a); id += gridDim.x) {
        const Place pc(a, id, V);
        __syncthreads();
        join_partials(a, pc, s_mean, s_rstd);
        __syncthreads();
        if (!pc.on) continue;
        float mu[V], k[V], b[V];
        affine<V>(a, pc, k, b);
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int g = (pc.lv * V + j) / a.D;
            mu[j] = s_mean[g];
            k[j] *= s_rstd[g];
        }
        const size_t base = ((size_t)pc.n * a.hw + pc.p0) * a.C + pc.c0;
        const T *x = (const T *)a.x + base, *res = a.res ? (const T *)a.res + pc.c0 : nullptr;
        T *y = (T *)a.y + base;
        for (long long p = pc.pl; p < pc.np; p += a.PL) {
            float f[V];
            VecIO<T, V>::load(x + (size_t)p * a.C, f);
            act_store<T, V>(a, f, mu, k, b, res, y + (size_t)p * a.C, pc.p0 + p, pc.n);
        }
    }
}

// dz and xhat of one vector
template <typename T, int V>
__device__ __forceinline__ void grad_of(const Args &a, const float (&f)[V], const float (&d)[V], const float (&mu)[V], const float (&rs)[V],
                                        const float (&w)[V], const float (&b)[V], float (&xh)[V], float (&dz)[V])
{
#pragma unroll
    for (int j = 0; j < V; ++j) {
        xh[j] = (f[j] - mu[j]) * rs[j];
        // (z as the forward computed it: the sign a LeakyReLU's gradient goes by is the forward's)
        const float z = (f[j] - mu[j]) * (rs[j] * w[j]) + b[j];
        if (a.act == 0) {
            dz[j] = z >= 0.0f ? d[j] : d[j] * a.slope;
        } else {
            const float s = sigmoid(z);
            dz[j] = d[j] * (s * (1.0f + z * (1.0f - s)));
        }
    }
}

template <int V> __device__ __forceinline__ void stats_of(const Args &a, const Place &pc, float (&mu)[V], float (&rs)[V])
{
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const size_t g = (size_t)pc.n * a.G + (pc.on ? (pc.c0 + j) / a.D : 0);
        mu[j] = a.mean[g];
        rs[j] = a.rstd[g];
    }
}

// ---- backward, first pass: per-channel sums of dz and dz xhat, and their weighted sums per group
template <typename T, int V> __global__ __launch_bounds__(kT) void k_gn_bwd_reduce(const Args a)
{
    __shared__ float s1[kT * V], s2[kT * V];
    for (long long id = blockIdx.x; id < n_work(a); id += gridDim.x) {
        const Place pc(a, id, V);
        const size_t base = ((size_t)pc.n * a.hw + pc.p0) * a.C + pc.c0;
        const T *x = (const T *)a.x + base, *dy = (const T *)a.dy + base;
        float w[V], b[V], mu[V], rs[V], t1[V], t2[V];
        affine<V>(a, pc, w, b);
        stats_of<V>(a, pc, mu, rs);
#pragma unroll
        for (int j = 0; j < V; ++j) t1[j] = t2[j] = 0.0f;
        if (pc.on)
            for (long long p = pc.pl; p < pc.np; p += a.PL) {
                float f[V], d[V], xh[V], dz[V];
                VecIO<T, V>::load(x + (size_t)p * a.C, f);
                VecIO<T, V>::load(dy + (size_t)p * a.C, d);
                grad_of<T, V>(a, f, d, mu, rs, w, b, xh, dz);
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    t1[j] += dz[j];
                    t2[j] += dz[j] * xh[j];
                }
            }
        const int tid = threadIdx.x;
        __syncthreads();
#pragma unroll
        for (int j = 0; j < V; ++j) {
            s1[tid * V + j] = t1[j];
            s2[tid * V + j] = t2[j];
        }
        __syncthreads();
        for (int v = a.PL; v > 1;) {
            const int h = (v + 1) >> 1;
            if (pc.pl + h < v) {
                const int o = (tid + h * a.LV) * V;
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    s1[tid * V + j] += s1[o + j];
                    s2[tid * V + j] += s2[o + j];
                }
            }
            __syncthreads();
            v = h;
        }
        float *cp = a.cpart + ((size_t)pc.n * a.nblk + pc.blk) * 2 * a.C;
        const int cs = pc.slab * a.SC;
        for (int c = tid; c < pc.ng * a.D; c += kT) {
            cp[cs + c] = s1[c];
            cp[a.C + cs + c] = s2[c];
        }
        const int lane = tid & 63, wave = tid >> 6;
        for (int g = wave; g < pc.ng; g += kT / 64) {
            float u1 = 0.0f, u2 = 0.0f;
            for (int c = lane; c < a.D; c += 64) {
                const float wc = a.w ? a.w[(size_t)pc.n * a.aff_stride + cs + g * a.D + c] + a.w_off : 1.0f;
                u1 += wc * s1[g * a.D + c];
                u2 += wc * s2[g * a.D + c];
            }
            u1 = wave_sum(u1);
            u2 = wave_sum(u2);
            if (lane == 0) a.gpart[((size_t)pc.n * a.nblk + pc.blk) * a.G + cs / a.D + g] = make_float2(u1, u2);
        }
        __syncthreads();
    }
}

// ---- backward, second pass: dx
template <typename T, int V> __global__ __launch_bounds__(kT) void k_gn_bwd_apply(const Args a)
{
    __shared__ float g1[kT * V], g2[kT * V];
    for (long long id = blockIdx.x; id < n_work(a); id += gridDim.x) {
        const Place pc(a, id, V);
        __syncthreads();
        {
            const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g0 = pc.slab * (a.SC / a.D);
            const float m = (float)((double)a.hw * a.D);
            for (int g = wave; g < pc.ng; g += kT / 64) {
                const float2 *p = a.gpart + (size_t)pc.n * a.nblk * a.G + g0 + g;
                float u1 = 0.0f, u2 = 0.0f;
                for (int k = lane; k < a.nblk; k += 64) {
                    const float2 v = p[(size_t)k * a.G];
                    u1 += v.x;
                    u2 += v.y;
                }
                u1 = wave_sum(u1) / m;
                u2 = wave_sum(u2) / m;
                if (lane == 0) {
                    g1[g] = u1;
                    g2[g] = u2;
                }
            }
        }
        __syncthreads();
        if (!pc.on) continue;
        const size_t base = ((size_t)pc.n * a.hw + pc.p0) * a.C + pc.c0;
        const T *x = (const T *)a.x + base, *dy = (const T *)a.dy + base;
        T *dx = (T *)a.y + base;
        float w[V], b[V], mu[V], rs[V], u1[V], u2[V];
        affine<V>(a, pc, w, b);
        stats_of<V>(a, pc, mu, rs);
#pragma unroll
        for (int j = 0; j < V; ++j) {
            u1[j] = g1[(pc.lv * V + j) / a.D];
            u2[j] = g2[(pc.lv * V + j) / a.D];
        }
        for (long long p = pc.pl; p < pc.np; p += a.PL) {
            float f[V], d[V], xh[V], dz[V];
            VecIO<T, V>::load(x + (size_t)p * a.C, f);
            VecIO<T, V>::load(dy + (size_t)p * a.C, d);
            grad_of<T, V>(a, f, d, mu, rs, w, b, xh, dz);
#pragma unroll
            for (int j = 0; j < V; ++j) f[j] = rs[j] * (w[j] * dz[j] - u1[j] - xh[j] * u2[j]);
            VecIO<T, V>::store(dx + (size_t)p * a.C, f);
        }
    }
}

// ---- dw / db from cpart: out row r (r = n: per sample; r = 0: all samples) sums `rows` partial rows
__global__ __launch_bounds__(1024) void k_gn_affine_grad(const float *__restrict__ cpart, float *__restrict__ dw, float *__restrict__ db,
                                                         int C, long long rows)
{
    __shared__ float s1[32][33], s2[32][33];
    const int cl = threadIdx.x & 31, rl = threadIdx.x >> 5;
    const int c = blockIdx.x * 32 + cl;
    const size_t r0 = (size_t)blockIdx.y * rows;
    float t1 = 0.0f, t2 = 0.0f;
    if (c < C)
        for (long long r = rl; r < rows; r += 32) {
            t1 += cpart[(r0 + r) * 2 * C + c];
            t2 += cpart[((r0 + r) * 2 + 1) * C + c];
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
        if (db) db[(size_t)blockIdx.y * C + c] = s1[0][cl];
        if (dw) dw[(size_t)blockIdx.y * C + c] = s2[0][cl];
    }
}

// ---- dres of a half-resolution residual: 2 x 2 sums of dy
template <typename T, int V> __global__ __launch_bounds__(kT) void k_gn_fold(const Args a)
{
    const int vecs = a.C / V, W2 = a.res_w >> 1;
    const long long q = a.hw / 4, total = (long long)a.N * q * vecs;
    const T *dy = (const T *)a.dy;
    for (long long i = (long long)blockIdx.x * kT + threadIdx.x; i < total; i += (long long)gridDim.x * kT) {
        const long long px = i / vecs, n = px / q, r = px - n * q, h = r / W2, w = r - h * W2;
        const int c0 = (int)(i - px * vecs) * V;
        const T *s = dy + ((size_t)n * a.hw + (size_t)(2 * h) * a.res_w + 2 * w) * a.C + c0;
        float f0[V], f1[V], f2[V], f3[V];
        VecIO<T, V>::load(s, f0);
        VecIO<T, V>::load(s + a.C, f1);
        VecIO<T, V>::load(s + (size_t)a.res_w * a.C, f2);
        VecIO<T, V>::load(s + (size_t)(a.res_w + 1) * a.C, f3);
#pragma unroll
        for (int j = 0; j < V; ++j) f0[j] = (f0[j] + f1[j]) + (f2[j] + f3[j]);
        VecIO<T, V>::store((T *)a.dres + (size_t)px * a.C + c0, f0);
    }
}

// ------------------------------------------------------------------------------------------------ host
static long long gcd_ll(long long a, long long b)
{
    while (b) {
        const long long t = a % b;
        a = b;
        b = t;
    }
    return a;
}

static inline int elem_bytes(int dtype) { return dtype == M355_F32 ? 4 : 2; }

// largest vector (16 bytes at most) that divides the channel count and every base address (`bits`: the addresses or-ed together)
static int pick_vec(int C, int dtype, uintptr_t bits)
{
    int v = 16 / elem_bytes(dtype);
    while (v > 1 && (C % v || bits % (uintptr_t)(v * elem_bytes(dtype)))) v >>= 1;
    return v;
}

// slab and range of a workgroup for a vector length; 0: a group is wider than a workgroup's vectors
static bool plan(Args &a, int V)
{
    const long long unit = (long long)a.D / gcd_ll(a.D, V) * V;   // channels: whole groups and whole vectors
    const long long most = (long long)kT * V;
    if (a.C <= most) a.SC = a.C;
    else if (unit <= most) a.SC = (int)(most / unit * unit);
    else return false;
    a.nslab = (a.C + a.SC - 1) / a.SC;
    a.LV = a.SC / V;
    a.PL = kT / a.LV;
    return true;
}

static void ranges(Args &a, int N, long long hw, int C)
{
    // a workgroup takes about 32 k values, a sample at most 64 ranges (the second pass joins them with one load a lane)
    long long nblk = ((double)hw * C + 32767.0) / 32768.0;
    if (nblk < 1) nblk = 1;
    if (nblk > 64) nblk = 64;
    if (nblk > hw) nblk = hw > 0 ? hw : 1;
    a.ppb = (hw + nblk - 1) / nblk;
    if (a.ppb < 1) a.ppb = 1;
    a.nblk = (int)((hw + a.ppb - 1) / a.ppb);
    if (a.nblk < 1) a.nblk = 1;
}

static int check_shape(long long N, long long HW, int C, int G, int dtype)
{
    M355_REQUIRE(N >= 0 && HW >= 0 && C > 0 && G > 0, "group_norm: N %lld, HW %lld, C %d, G %d", N, HW, C, G);
    M355_REQUIRE(C % G == 0, "group_norm: %d channels in %d groups", C, G);
    M355_REQUIRE(dtype == M355_F32 || dtype == M355_F16 || dtype == M355_BF16, "group_norm: unknown dtype %d", dtype);
    M355_REQUIRE(N < (1LL << 31) && HW < (1LL << 40), "group_norm: N %lld or HW %lld too large", N, HW);
    return M355_OK;
}

static unsigned grid_of(long long work)
{
    const long long most = 1 << 22;   // (grid * block stays below 2^32; the kernels loop over the rest)
    return (unsigned)(work < most ? work : most);
}

template <typename T, int V> static int run_fwd(const Args &a, hipStream_t s)
{
    const unsigned g = grid_of(n_work(a));
    hipLaunchKernelGGL((k_gn_stats<T, V>), dim3(g), dim3(kT), 0, s, a);
    hipLaunchKernelGGL((k_gn_apply<T, V>), dim3(g), dim3(kT), 0, s, a);
    return check_launch("group_norm_fwd");
}

template <typename T, int V> static int run_bwd(const Args &a, float *dw, float *db, int per_sample, hipStream_t s)
{
    const unsigned g = grid_of(n_work(a));
    hipLaunchKernelGGL((k_gn_bwd_reduce<T, V>), dim3(g), dim3(kT), 0, s, a);
    if (a.y) hipLaunchKernelGGL((k_gn_bwd_apply<T, V>), dim3(g), dim3(kT), 0, s, a);
    if (a.dres) {
        const long long items = (long long)a.N * (a.hw / 4) * (a.C / V);
        const long long blocks = (items + kT - 1) / kT;
        hipLaunchKernelGGL((k_gn_fold<T, V>), dim3((unsigned)(blocks < 8192 ? blocks : 8192)), dim3(kT), 0, s, a);
    }
    if (dw || db) {
        for (int n0 = 0; n0 < (per_sample ? a.N : 1); n0 += 65535) {
            const int rows = per_sample ? (a.N - n0 < 65535 ? a.N - n0 : 65535) : 1;
            hipLaunchKernelGGL(k_gn_affine_grad, dim3((unsigned)((a.C + 31) / 32), (unsigned)rows), dim3(1024), 0, s,
                               a.cpart + (size_t)n0 * a.nblk * 2 * a.C, dw ? dw + (size_t)n0 * a.C : nullptr,
                               db ? db + (size_t)n0 * a.C : nullptr, a.C, per_sample ? (long long)a.nblk : (long long)a.N * a.nblk);
        }
    }
    return check_launch("group_norm_bwd");
}

template <typename F> static int by_type(int dtype, int V, F f)
{
    if (dtype == M355_F32) return V == 4 ? f((float *)nullptr, std::integral_constant<int, 4>()) : V == 2 ? f((float *)nullptr, std::integral_constant<int, 2>())
                                                                                                     : f((float *)nullptr, std::integral_constant<int, 1>());
#define M355_GN_V(T)                                                                   \
    V == 8 ? f((T *)nullptr, std::integral_constant<int, 8>())                         \
           : V == 4 ? f((T *)nullptr, std::integral_constant<int, 4>())                \
                    : V == 2 ? f((T *)nullptr, std::integral_constant<int, 2>()) : f((T *)nullptr, std::integral_constant<int, 1>())
    if (dtype == M355_F16) return M355_GN_V(_Float16);
    return M355_GN_V(__bf16);
#undef M355_GN_V
}

}  // namespace gn
}  // namespace m355

using namespace m355;

extern "C" size_t m355_group_norm_ws_bytes(long long N, long long HW, int C, int G, int dtype, int backward)
{
    if (gn::check_shape(N, HW, C, G, dtype) != M355_OK) return 0;
    gn::Args a = {};
    gn::ranges(a, (int)N, HW, C);
    const size_t rows = (size_t)N * (size_t)a.nblk;
    size_t bytes = rows * (size_t)G * sizeof(float2);
    if (backward) bytes += rows * 2 * (size_t)C * sizeof(float);
    return bytes > 0 ? bytes : 8;
}

extern "C" int m355_group_norm_fwd(const void *x, const float *w, const float *b, long long aff_stride, float w_off, const void *res,
                                   int res_w, void *y, float *mean, float *rstd, void *ws, long long N, long long HW, int C, int G,
                                   float eps, int act, float slope, float out_slope, int dtype, void *stream)
{
    const int rc = gn::check_shape(N, HW, C, G, dtype);
    if (rc != M355_OK) return rc;
    if (N == 0 || HW == 0) return M355_OK;
    M355_REQUIRE(x && y && mean && rstd && ws, "group_norm_fwd: null pointer");
    M355_REQUIRE(x != y, "group_norm_fwd: y must not be x");
    M355_REQUIRE(act == 0 || act == 1, "group_norm_fwd: unknown activation %d", act);
    M355_REQUIRE(res_w >= 0 && (res_w == 0 || (res && res_w % 2 == 0 && HW % (2LL * res_w) == 0)),
                 "group_norm_fwd: a half-resolution residual needs even height and width (width %d, %lld pixels)", res_w, HW);
    gn::Args a = {};
    a.x = x; a.res = res; a.y = y; a.w = w; a.b = b; a.mean = mean; a.rstd = rstd; a.gpart = (float2 *)ws;
    a.aff_stride = aff_stride; a.hw = HW; a.N = (int)N; a.C = C; a.G = G; a.D = C / G; a.act = act; a.res_w = res_w;
    a.w_off = w_off; a.eps = eps; a.slope = slope; a.out_slope = out_slope;
    gn::ranges(a, (int)N, HW, C);
    const int V = gn::pick_vec(C, dtype, (uintptr_t)x | (uintptr_t)y | (uintptr_t)res);
    if (!gn::plan(a, V)) {
        set_error("group_norm_fwd: groups of %d channels (vectors of %d) are wider than a workgroup takes", a.D, V);
        return M355_ERR_UNSUPPORTED;
    }
    return gn::by_type(dtype, V, [&](auto *t, auto v) {
        return gn::run_fwd<std::remove_pointer_t<decltype(t)>, decltype(v)::value>(a, (hipStream_t)stream);
    });
}

extern "C" int m355_group_norm_bwd(const void *dy, const void *x, const float *w, const float *b, long long aff_stride, float w_off,
                                   const float *mean, const float *rstd, void *dx, float *dw, float *db, int per_sample, void *dres,
                                   int res_w, void *ws, long long N, long long HW, int C, int G, int act, float slope, int dtype,
                                   void *stream)
{
    const int rc = gn::check_shape(N, HW, C, G, dtype);
    if (rc != M355_OK) return rc;
    if (N == 0 || HW == 0) return M355_OK;   // (the caller zeroes dw / db of an empty batch)
    M355_REQUIRE(dy && x && mean && rstd && ws, "group_norm_bwd: null pointer");
    M355_REQUIRE(dx != x && dx != dy, "group_norm_bwd: dx must be a tensor of its own");
    M355_REQUIRE(act == 0 || act == 1, "group_norm_bwd: unknown activation %d", act);
    M355_REQUIRE(!dres || (res_w > 0 && res_w % 2 == 0 && HW % (2LL * res_w) == 0),
                 "group_norm_bwd: a half-resolution residual needs even height and width (width %d, %lld pixels)", res_w, HW);
    gn::Args a = {};
    a.x = x; a.dy = dy; a.y = dx; a.dres = dres; a.w = w; a.b = b; a.mean = (float *)mean; a.rstd = (float *)rstd;
    a.aff_stride = aff_stride; a.hw = HW; a.N = (int)N; a.C = C; a.G = G; a.D = C / G; a.act = act; a.res_w = dres ? res_w : 0;
    a.w_off = w_off; a.slope = slope; a.out_slope = 1.0f;
    gn::ranges(a, (int)N, HW, C);
    a.gpart = (float2 *)ws;
    a.cpart = (float *)(a.gpart + (size_t)N * a.nblk * G);
    const int V = gn::pick_vec(C, dtype, (uintptr_t)x | (uintptr_t)dy | (uintptr_t)dx | (uintptr_t)dres);
    if (!gn::plan(a, V)) {
        set_error("group_norm_bwd: groups of %d channels (vectors of %d) are wider than a workgroup takes", a.D, V);
        return M355_ERR_UNSUPPORTED;
    }
    return gn::by_type(dtype, V, [&](auto *t, auto v) {
        return gn::run_bwd<std::remove_pointer_t<decltype(t)>, decltype(v)::value>(a, dw, db, per_sample, (hipStream_t)stream);
    });
}
