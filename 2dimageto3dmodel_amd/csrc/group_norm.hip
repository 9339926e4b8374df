// Entry points of the group norm with an activation, channels last (include/m355.h m355_group_norm_*): argument checks and the choice
// of a kernel (group_norm.h).
#include <algorithm>

#include "group_norm.h"

namespace m355 {
namespace gn {

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

// the largest vector (16 bytes at most) that divides the channel count and every base address (`bits`: the addresses or-ed together),
// and its segments: V / gcd(V, D), rounded up to one that is built
static void pick_vec(int C, int D, int dtype, uintptr_t bits, int &V, int &A)
{
    V = 16 / elem_bytes(dtype);
    while (V > 1 && (C % V || bits % (uintptr_t)(V * elem_bytes(dtype)))) V >>= 1;
    A = V / (int)gcd_ll(V, D);
    if (A == 2 && V >= 4) A = 4;
    if (V == 2) A = 2;
}

// channels that are whole groups and whole vectors
static long long unit_of(int D, int V) { return (long long)D / gcd_ll(V, D) * V; }

static void set_slab(Args &a, long long SC, int V, int nt)
{
    a.SC = (int)SC;
    a.nslab = (int)((a.C + SC - 1) / SC);
    a.LV = (int)(SC / V);
    a.PL = nt / a.LV;
}

// two passes: all channels if a workgroup's vectors reach over them, else as many whole groups as they do.  false: a group is wider
static bool wide_slab(Args &a, int V)
{
    const long long unit = unit_of(a.D, V), most = (long long)kT * V;
    if (a.C <= most) set_slab(a, a.C, V, kT);
    else if (unit <= most) set_slab(a, most / unit * unit, V, kT);
    else return false;
    return true;
}

static void set_items(Args &a, int res_w, bool quad)
{
    a.quad = quad;
    a.items = quad ? a.hw / 4 : a.hw;
    a.W2 = res_w / 2;
    if (quad && a.W2 > 1) {
        int l = 0;
        while ((1LL << l) < a.W2) ++l;
        a.magic = (unsigned)(((1ULL << (31 + l)) / (unsigned)a.W2) + 1);   // exact for i < 2^31
        a.shift = (unsigned)(l - 1);
    }
}

// ranges of a sample: about `goal` values a workgroup, `pixels` an item
static int ranges_of(long long items, long long pixels, int C, int nslab, long long goal, long long &per)
{
    long long nblk = (long long)(((double)items * (double)(pixels * C) / nslab + goal - 1) / goal);
    nblk = std::max(1LL, std::min(nblk, std::min(std::max(items, 1LL), 4096LL / std::min(nslab, 64))));
    per = std::max(1LL, (items + nblk - 1) / nblk);
    return (int)std::max(1LL, (items + per - 1) / per);
}

constexpr long long kGoal = 32768;   // values of a workgroup's range in the two-pass kernels
constexpr int kJoin = 32;            // ranges a sample up to which the second pass joins them itself

// rows of partial sums a sample that any choice below may need (the workspace is sized before the pointers are known)
static long long most_rows(long long HW, int C, int)
{
    return std::max(1LL, std::min(std::max(HW, 1LL), std::min(4096LL, (long long)((double)HW * C / kGoal) + 2)));
}

// one pass: the narrowest slab of whole groups whose rows are `row` bytes, if a workgroup's registers hold it
static bool hold(Args &a, int V, int esize, int row, Choice &c, const int (&R)[3])
{
    const long long unit = unit_of(a.D, V);
    long long SC = unit;
    while (SC * esize < row && SC < a.C) SC += unit;
    if (SC > a.C) SC = a.C;
    static const int nts[3] = {256, 256, 1024};
    for (int k = 0; k < 3; ++k) {
        if (SC > (long long)nts[k] * V) continue;
        set_slab(a, SC, V, nts[k]);
        const long long need = (a.items + a.PL - 1) / a.PL * (a.quad ? 4 : 1);
        if (need <= R[k]) {
            c.nt = nts[k];
            c.R = R[k];
            return true;
        }
    }
    return false;
}

static int check_shape(long long N, long long HW, int C, int G, int dtype)
{
    M355_REQUIRE(N >= 0 && HW >= 0 && C > 0 && G > 0, "group_norm: N %lld, HW %lld, C %d, G %d", N, HW, C, G);
    M355_REQUIRE(C % G == 0, "group_norm: %d channels in %d groups", C, G);
    M355_REQUIRE(dtype == M355_F32 || dtype == M355_F16 || dtype == M355_BF16, "group_norm: unknown dtype %d", dtype);
    M355_REQUIRE(N < (1LL << 31) && HW < (1LL << 36) && C <= (1 << 20), "group_norm: N %lld, HW %lld or C %d too large", N, HW, C);
    return M355_OK;
}

static Runner runner(int dtype) { return dtype == M355_F32 ? run_f32() : dtype == M355_F16 ? run_f16() : run_bf16(); }

// f(args of these samples) over launches of at most 2^22 workgroups
template <typename F> static void by_samples(const Args &all, int esize, F f)
{
    const long long per = std::max(1LL, (1LL << 22) / ((long long)all.nslab * all.nblk));
    for (long long n0 = 0; n0 < all.N; n0 += per) {
        Args a = all;
        a.N = (int)std::min(per, all.N - n0);
        const size_t px = (size_t)n0 * a.hw * a.C * esize, rp = (size_t)n0 * (a.quad ? a.items : a.hw) * a.C * esize;
        if (a.x) a.x = (const char *)a.x + px;
        if (a.dy) a.dy = (const char *)a.dy + px;
        if (a.y) a.y = (char *)a.y + px;
        if (a.res) a.res = (const char *)a.res + rp;
        if (a.dres) a.dres = (char *)a.dres + rp;
        if (a.w) a.w += n0 * a.aff_stride;
        if (a.b) a.b += n0 * a.aff_stride;
        a.mean += n0 * a.G;
        a.rstd += n0 * a.G;
        if (a.gpart) a.gpart += (size_t)n0 * a.gnblk * a.G;
        if (a.gsum) a.gsum += (size_t)n0 * a.G;
        if (a.cpart) a.cpart += (size_t)n0 * a.gnblk * 2 * a.C;
        if (a.per_sample) {
            if (a.dw) a.dw += (size_t)n0 * a.C;
            if (a.db) a.db += (size_t)n0 * a.C;
        }
        f(a);
    }
}

static unsigned wave_grid(const Args &a) { return (unsigned)(((long long)a.N * a.G + kT / 64 - 1) / (kT / 64)); }

static void affine_grad(const Args &a, hipStream_t s)
{
    const long long rows = a.per_sample ? a.gnblk : (long long)a.N * a.gnblk;
    const int out = a.per_sample ? a.N : 1;
    for (int n0 = 0; n0 < out; n0 += 65535) {
        const int k = std::min(out - n0, 65535);
        hipLaunchKernelGGL(k_gn_affine_grad, dim3((unsigned)((a.C + 31) / 32), (unsigned)k), dim3(1024), 0, s,
                           a.cpart + (size_t)n0 * rows * 2 * a.C, a.dw ? a.dw + (size_t)n0 * a.C : nullptr,
                           a.db ? a.db + (size_t)n0 * a.C : nullptr, a.C, rows);
    }
}

}  // namespace gn
}  // namespace m355

using namespace m355;

extern "C" size_t m355_group_norm_ws_bytes(long long N, long long HW, int C, int G, int dtype, int backward)
{
    if (gn::check_shape(N, HW, C, G, dtype) != M355_OK) return 0;
    const size_t rows = (size_t)N * (size_t)gn::most_rows(HW, C, G);
    size_t bytes = rows * (size_t)G * sizeof(float2);
    if (backward) bytes += rows * 2 * (size_t)C * sizeof(float) + (size_t)N * G * sizeof(float2);
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
    a.aff_stride = aff_stride; a.hw = HW; a.N = (int)N; a.C = C; a.G = G; a.D = C / G; a.act = act;
    a.w_off = w_off; a.eps = eps; a.slope = slope; a.out_slope = out_slope;
    gn::Choice c = {};
    gn::pick_vec(C, a.D, dtype, (uintptr_t)x | (uintptr_t)y | (uintptr_t)res, c.V, c.A);
    if (!gn::wide_slab(a, c.V)) {
        set_error("group_norm_fwd: groups of %d channels (vectors of %d) are wider than a workgroup takes", a.D, c.V);
        return M355_ERR_UNSUPPORTED;
    }
    const gn::Runner run = gn::runner(dtype);
    hipStream_t s = (hipStream_t)stream;
    const int es = gn::elem_bytes(dtype);
    static const int R[3] = {4, 16, 16};
    gn::set_items(a, res_w, res_w > 0);
    a.nblk = a.gnblk = 1;
    a.per = a.items;
    if (gn::hold(a, c.V, es, 128, c, R) || gn::hold(a, c.V, es, 64, c, R)) {
        gn::by_samples(a, es, [&](const gn::Args &p) { run.one(p, c, s); });
        return check_launch("group_norm_fwd");
    }
    gn::wide_slab(a, c.V);
    gn::Args st = a;
    gn::set_items(st, 0, false);
    st.res = nullptr;
    st.nblk = gn::ranges_of(st.items, 1, C, st.nslab, gn::kGoal, st.per);
    st.gnblk = a.gnblk = st.nblk;
    st.gper = a.gper = st.per;
    a.nblk = gn::ranges_of(a.items, a.quad ? 4 : 1, C, a.nslab, gn::kGoal, a.per);
    a.finished = a.gnblk > gn::kJoin;
    gn::by_samples(st, es, [&](const gn::Args &p) { run.stats(p, c.V, c.A, s); });
    if (a.finished)
        gn::by_samples(st, es, [&](const gn::Args &p) { hipLaunchKernelGGL(gn::k_gn_finish, dim3(gn::wave_grid(p)), dim3(gn::kT), 0, s, p); });
    gn::by_samples(a, es, [&](const gn::Args &p) { run.apply(p, c.V, c.A, s); });
    return check_launch("group_norm_fwd");
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
    M355_REQUIRE(res_w >= 0 && (res_w == 0 ? !dres : res_w % 2 == 0 && HW % (2LL * res_w) == 0),
                 "group_norm_bwd: a half-resolution residual needs even height and width (width %d, %lld pixels)", res_w, HW);
    gn::Args a = {};
    a.x = x; a.dy = dy; a.y = dx; a.dres = dres; a.w = w; a.b = b; a.mean = (float *)mean; a.rstd = (float *)rstd;
    a.aff_stride = aff_stride; a.hw = HW; a.N = (int)N; a.C = C; a.G = G; a.D = C / G; a.act = act;
    a.w_off = w_off; a.slope = slope; a.out_slope = 1.0f;
    a.dw = dw; a.db = db; a.per_sample = per_sample != 0;
    gn::Choice c = {};
    gn::pick_vec(C, a.D, dtype, (uintptr_t)x | (uintptr_t)dy | (uintptr_t)dx | (uintptr_t)dres, c.V, c.A);
    if (!gn::wide_slab(a, c.V)) {
        set_error("group_norm_bwd: groups of %d channels (vectors of %d) are wider than a workgroup takes", a.D, c.V);
        return M355_ERR_UNSUPPORTED;
    }
    const gn::Runner run = gn::runner(dtype);
    hipStream_t s = (hipStream_t)stream;
    const int es = gn::elem_bytes(dtype);
    a.gpart = (float2 *)ws;
    a.gsum = a.gpart + (size_t)N * gn::most_rows(HW, C, G) * G;
    float *cpart = (float *)(a.gsum + (size_t)N * G);
    a.cpart = dw || db ? cpart : nullptr;
    static const int R[3] = {4, 8, 8};
    gn::set_items(a, res_w, res_w > 0);   // (the same order of additions whether or not dres is wanted)
    a.nblk = a.gnblk = 1;
    a.per = a.items;
    if (gn::hold(a, c.V, es, 128, c, R) || gn::hold(a, c.V, es, 64, c, R)) {
        gn::by_samples(a, es, [&](const gn::Args &p) { run.bwd_one(p, c, s); });
        if (!a.per_sample && a.cpart) gn::affine_grad(a, s);
        return check_launch("group_norm_bwd");
    }
    gn::wide_slab(a, c.V);
    a.nblk = gn::ranges_of(a.items, a.quad ? 4 : 1, C, a.nslab, gn::kGoal, a.per);
    a.gnblk = a.nblk;
    a.finished = a.gnblk > gn::kJoin;
    gn::by_samples(a, es, [&](const gn::Args &p) { run.bwd_reduce(p, c.V, c.A, s); });
    if (a.cpart) gn::affine_grad(a, s);
    if (dx) {
        if (a.finished)
            gn::by_samples(a, es, [&](const gn::Args &p) { hipLaunchKernelGGL(gn::k_gn_bwd_finish, dim3(gn::wave_grid(p)), dim3(gn::kT), 0, s, p); });
        gn::Args d = a;
        gn::set_items(d, 0, false);
        d.dres = nullptr;
        d.nblk = gn::ranges_of(d.items, 1, C, d.nslab, gn::kGoal, d.per);
        gn::by_samples(d, es, [&](const gn::Args &p) { run.bwd_apply(p, c.V, c.A, s); });
    }
    return check_launch("group_norm_bwd");
}
