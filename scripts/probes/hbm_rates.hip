// What a kernel that only reads, and one that copies, reaches by size, workgroups, loads in flight and cache policy (nt: past the
// memory-side cache).  hipcc -O3 --offload-arch=gfx950 -Xclang -target-feature -Xclang -packed-fp32-ops hbm_rates.hip -o hbm_rates
#include <hip/hip_runtime.h>
#include <stdio.h>
#include <stdlib.h>
#include <vector>
#include <algorithm>
#define OK(e) do { if ((e) != hipSuccess) { printf("failed: %s\n", #e); exit(1); } } while (0)
typedef float f4 __attribute__((ext_vector_type(4)));
// each workgroup reads a contiguous span of `per` vectors (blocked) or grid-strides
template <int U, bool NT> __global__ __launch_bounds__(256) void k_read(const f4 *x, float *out, size_t n, size_t per)
{
    size_t i = (size_t)blockIdx.x * per + threadIdx.x, e = min(n, (size_t)(blockIdx.x + 1) * per);
    f4 acc = {0, 0, 0, 0};
    for (; i + (U - 1) * 256 < e; i += U * 256) {
        f4 v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) v[u] = NT ? __builtin_nontemporal_load(x + i + u * 256) : x[i + u * 256];
#pragma unroll
        for (int u = 0; u < U; ++u) acc += v[u];
    }
    if (acc.x + acc.y + acc.z + acc.w == 12345.678f) out[0] = 1;
}
template <int U, bool NTS> __global__ __launch_bounds__(256) void k_copy(const f4 *x, f4 *y, size_t n, size_t per)
{
    size_t i = (size_t)blockIdx.x * per + threadIdx.x, e = min(n, (size_t)(blockIdx.x + 1) * per);
    for (; i + (U - 1) * 256 < e; i += U * 256) {
        f4 v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) v[u] = x[i + u * 256];
#pragma unroll
        for (int u = 0; u < U; ++u) { if (NTS) __builtin_nontemporal_store(v[u], y + i + u * 256); else y[i + u * 256] = v[u]; }
    }
}
int main()
{
    size_t big = (size_t)1 << 30;
    f4 *x, *y; float *o;
    OK(hipMalloc(&x, big)); OK(hipMalloc(&y, big)); OK(hipMalloc(&o, 64));
    OK(hipMemset(x, 0, big)); OK(hipMemset(y, 0, big));
    hipEvent_t a, b; OK(hipEventCreate(&a)); OK(hipEventCreate(&b));
    auto time = [&](auto f) {
        std::vector<float> t;
        for (int k = 0; k < 3; ++k) f();
        for (int r = 0; r < 7; ++r) { OK(hipEventRecord(a)); for (int k = 0; k < 5; ++k) f(); OK(hipEventRecord(b)); OK(hipEventSynchronize(b));
            float ms; OK(hipEventElapsedTime(&ms, a, b)); t.push_back(ms / 5); }
        std::sort(t.begin(), t.end()); return t[3] * 1e-3;
    };
    for (size_t mb : {16, 64, 128, 192, 1024}) {   // (a workgroup's span is a multiple of 8 x 256 vectors: nothing is read past n)
        size_t n = (mb << 20) / 16;
        for (size_t wgs : {1024, 2048, 4096, 8192, 16384}) {
            size_t per = n / wgs;
            if (per < 2048 || per % 2048) continue;
            double t4 = time([&] { hipLaunchKernelGGL((k_read<4, false>), dim3(wgs), dim3(256), 0, 0, x, o, n, per); });
            double t8 = time([&] { hipLaunchKernelGGL((k_read<8, false>), dim3(wgs), dim3(256), 0, 0, x, o, n, per); });
            double tn = time([&] { hipLaunchKernelGGL((k_read<8, true>), dim3(wgs), dim3(256), 0, 0, x, o, n, per); });
            double c4 = time([&] { hipLaunchKernelGGL((k_copy<4, false>), dim3(wgs), dim3(256), 0, 0, x, y, n, per); });
            double c8 = time([&] { hipLaunchKernelGGL((k_copy<8, false>), dim3(wgs), dim3(256), 0, 0, x, y, n, per); });
            double cn = time([&] { hipLaunchKernelGGL((k_copy<4, true>), dim3(wgs), dim3(256), 0, 0, x, y, n, per); });
            double B = (double)n * 16;
            printf("%5zu MB wgs %5zu  read U4 %.2f U8 %.2f U8nt %.2f | copy(r+w) U4 %.2f U8 %.2f U4nts %.2f TB/s\n", mb, wgs, B / t4 / 1e12, B / t8 / 1e12, B / tn / 1e12, 2 * B / c4 / 1e12, 2 * B / c8 / 1e12, 2 * B / cn / 1e12);
            fflush(stdout);
        }
    }
    return 0;
}
