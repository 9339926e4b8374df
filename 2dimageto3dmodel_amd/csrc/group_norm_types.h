// Instantiates the group norm kernels (group_norm.h) for the element type M355_GN_T as the launch table M355_GN_RUN.
#include "group_norm.h"

namespace m355 {
namespace gn {
namespace {

typedef M355_GN_T T;
constexpr int kV = 16 / sizeof(T);   // the widest vector

// f(V, A) of the vectors and segments that are built: pick_vec() in group_norm.hip chooses among these
template <typename F> void by_vector(int V, int A, F f)
{
    using std::integral_constant;
    if constexpr (kV == 8) {
        if (V == 8 && A == 1) return f(integral_constant<int, 8>(), integral_constant<int, 1>());
        if (V == 8 && A == 4) return f(integral_constant<int, 8>(), integral_constant<int, 4>());
        if (V == 8) return f(integral_constant<int, 8>(), integral_constant<int, 8>());
    }
    if (V == 4 && A == 1) return f(integral_constant<int, 4>(), integral_constant<int, 1>());
    if (V == 4) return f(integral_constant<int, 4>(), integral_constant<int, 4>());
    if (V == 2) return f(integral_constant<int, 2>(), integral_constant<int, 2>());
    return f(integral_constant<int, 1>(), integral_constant<int, 1>());
}

template <typename F> void by_all(int V, int A, int act, F f)
{
    by_vector(V, A, [&](auto v, auto g) {
        if (act == 0) f(v, g, std::integral_constant<int, 0>());
        else f(v, g, std::integral_constant<int, 1>());
    });
}

dim3 grid(const Args &a) { return dim3((unsigned)((size_t)a.N * a.nslab * a.nblk)); }

void stats(const Args &a, int V, int A, hipStream_t s)
{
    by_vector(V, A, [&](auto v, auto g) { hipLaunchKernelGGL((k_gn_stats<T, v(), g()>), grid(a), dim3(kT), 0, s, a); });
}
void apply(const Args &a, int V, int A, hipStream_t s)
{
    by_all(V, A, a.act, [&](auto v, auto g, auto t) {
        if (a.nt) hipLaunchKernelGGL((k_gn_apply<T, v(), g(), t(), true>), grid(a), dim3(kT), 0, s, a);
        else hipLaunchKernelGGL((k_gn_apply<T, v(), g(), t(), false>), grid(a), dim3(kT), 0, s, a);
    });
}
void bwd_reduce(const Args &a, int V, int A, hipStream_t s)
{
    by_all(V, A, a.act, [&](auto v, auto g, auto t) {
        if (a.nt) hipLaunchKernelGGL((k_gn_bwd_reduce<T, v(), g(), t(), true>), grid(a), dim3(kT), 0, s, a);
        else hipLaunchKernelGGL((k_gn_bwd_reduce<T, v(), g(), t(), false>), grid(a), dim3(kT), 0, s, a);
    });
}
void bwd_apply(const Args &a, int V, int A, hipStream_t s)
{
    by_all(V, A, a.act, [&](auto v, auto g, auto t) {
        if (a.nt) hipLaunchKernelGGL((k_gn_bwd_apply<T, v(), g(), t(), true>), grid(a), dim3(kT), 0, s, a);
        else hipLaunchKernelGGL((k_gn_bwd_apply<T, v(), g(), t(), false>), grid(a), dim3(kT), 0, s, a);
    });
}
void one(const Args &a, const Choice &c, hipStream_t s)
{
    by_all(c.V, c.A, a.act, [&](auto v, auto g, auto t) {
        if (c.R == 8) hipLaunchKernelGGL((k_gn_one<T, v(), g(), t(), 8>), grid(a), dim3(kT), 0, s, a);
        else hipLaunchKernelGGL((k_gn_one<T, v(), g(), t(), 4>), grid(a), dim3(kT), 0, s, a);
    });
}
void bwd_one(const Args &a, const Choice &c, hipStream_t s)
{
    by_all(c.V, c.A, a.act, [&](auto v, auto g, auto t) {
        if (c.R == 8) hipLaunchKernelGGL((k_gn_bwd_one<T, v(), g(), t(), 8>), grid(a), dim3(kT), 0, s, a);
        else hipLaunchKernelGGL((k_gn_bwd_one<T, v(), g(), t(), 4>), grid(a), dim3(kT), 0, s, a);
    });
}

}  // namespace
}  // namespace gn
}  // namespace m355

m355::gn::Runner m355::gn::M355_GN_RUN() { return {stats, apply, bwd_reduce, bwd_apply, one, bwd_one}; }
