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

static void set_slab(Args &a, long long SC, int V)
{
    a.SC = (int)SC;
    a.nslab = (int)((a.C + SC - 1) / SC);
    a.LV = (int)(SC / V);
    a.PL = kT / a.LV;
    a.by_lv.set((unsigned)a.LV);
    a.by_pl.set((unsigned)a.PL);
    a.by_nslab.set((unsigned)a.nslab);
}

static void set_ranges(Args &a, int nblk, long long per)
{
    a.nblk = nblk;
    a.per = per;
    a.by_nblk.set((unsigned)nblk);
}

// two passes: all channels if a workgroup's vectors reach over them, else as many whole groups as they do.  false: a group is wider
static bool wide_slab(Args &a, int V)
{
    const long long unit = unit_of(a.D, V), most = (long long)kT * V;
    if (a.C <= most) set_slab(a, a.C, V);
    else if (unit <= most) set_slab(a, most / unit * unit, V);
    else return false;
    return true;
}

constexpr long long kMostRanges = 4096;   // of a sample
// ranges a sample up to which the second pass joins them itself: 64 for 32 (with eight parts a lane in flight for four) saves a launch for
// the samples between, 31.2 -> 29.0 us forward and backward of 3x100x100x96 bf16; the others stay within 1 %
constexpr int kJoin = 64;

static void set_groups(Args &a, const Choice &c)
{
    a.by_d.set((unsigned)a.D);
    a.by_sg.set((unsigned)(a.D / (c.V / c.A)));
}

static void set_items(Args &a, int res_w, bool quad)
{
    a.quad = quad;
    a.items = quad ? a.hw / 4 : a.hw;
    a.W2 = res_w / 2;
    if (quad) a.by_w2.set((unsigned)a.W2);
}

// Values of a range: about total / few while that is within 4096 .. 16384, from there total / share up to `most`.  Small calls want
// workgroups (5x37x29x60 fp32 forward and backward 32.1 -> 23.2 us for 16384 throughout, 2x64x32x256 bf16 25.1 -> 22.3), the first passes
// fewer of them than the second ones, which add up what those leave (1x64x32x256 bf16 forward 10.7 us with 256 of both, 9.7); calls of
// 4 million values lose by shorter ranges (32x32x32x128 28.8 -> 31.0)
struct Share {
    double few, share, most;
    double goal(double total) const { return std::min(std::max(std::min(std::max(total / few, 4096.0), 16384.0), total / share), most); }
};
constexpr Share kStats = {64, 512, 131072}, kApply = {256, 1024, 32768}, kReduce = {64, 512, 32768}, kDx = {256, 1024, 32768};

static void take_ranges(Args &a, const Share &sh)
{
    const long long items = a.items;
    const double sample = (double)a.hw * a.C;
    long long nblk = (long long)(sample / a.nslab / sh.goal(sample * a.N) + 0.999);
    nblk = std::max(1LL, std::min(std::min(nblk, std::max(items, 1LL)), kMostRanges));
    const long long per = std::max(1LL, (items + nblk - 1) / nblk);
    set_ranges(a, (int)std::max(1LL, (items + per - 1) / per), per);
}

// rows of partial sums a sample that any choice below may need (the workspace is sized before the pointers are known)
static long long most_rows(long long N, long long HW, int C)
{
    const double sample = (double)HW * C, least = std::min(kStats.goal(sample * N), kReduce.goal(sample * N));
    return std::max(1LL, std::min(std::max(HW, 1LL), std::min(kMostRanges, (long long)(sample / least) + 2)));
}

constexpr long long kMany = 1024;   // workgroups that fill the card

// One pass: slabs of whole groups whose rows are `row` bytes, if a workgroup holds one with R vectors a thread
static bool hold(Args &a, int V, int esize, int row, int R, Choice &c)
{
    const long long unit = unit_of(a.D, V);
    long long SC = unit;
    while (SC * esize < row && SC < a.C) SC += unit;
    // samples of a few pixels: wider while no thread has more than one vector and workgroups abound (2048 x 512, one pixel, forward and
    // backward: 115 -> 30 us; the slab's few threads are waited for eight times less often)
    while (2 * SC <= a.C && a.items * (a.quad ? 4 : 1) * (2 * SC / V) <= kT && (long long)a.N * (a.C / (2 * SC)) >= kMany) SC *= 2;
    if (SC > (long long)kT * V) return false;
    set_slab(a, SC, V);
    c.R = R;
    return (a.items + a.PL - 1) / a.PL * (a.quad ? 4 : 1) <= R;
}

// Rows of 128 bytes are whole cache lines; rows of 64 give twice the workgroups, which is what a small call lacks.  Forward / forward and
// backward of 16x16x1024 bf16 with a half-resolution residual: one sample 6.5 / 13.2 us with 64-byte rows of 4 vectors, 9.5 / 18.4 with
// 128-byte rows of 8 (9.8 / 24.7 in two passes); 64 samples 24.3 / 75.6 and 18.9 / 48.7 (22.8 / 71.3).  8x4x512, 16 samples: 6.0 / 12.6,
// two passes 9.4 / 23.0
static bool one_pass(Args &a, int V, int esize, Choice &c)
{
    if (hold(a, V, esize, 128, 4, c)) return true;
    if (hold(a, V, esize, 64, 4, c) && (long long)a.N * a.nslab <= 1024) return true;
    return hold(a, V, esize, 128, 8, c) || hold(a, V, esize, 64, 8, c);
}

static int check_desc(const m355_gn_desc *d)
{
    M355_REQUIRE(d, "group_norm: null pointer");
    const long long N = d->N, HW = d->HW;
    const int C = d->C, G = d->G, dtype = d->dtype;
    M355_REQUIRE(N >= 0 && HW >= 0 && C > 0 && G > 0, "group_norm: N %lld, HW %lld, C %d, G %d", N, HW, C, G);
    M355_REQUIRE(C % G == 0, "group_norm: %d channels in %d groups", C, G);
    M355_REQUIRE(dtype == M355_F32 || dtype == M355_F16 || dtype == M355_BF16, "group_norm: unknown dtype %d", dtype);
    M355_REQUIRE(N < (1LL << 31) && HW < (1LL << 36) && C <= (1 << 20), "group_norm: N %lld, HW %lld or C %d too large", N, HW, C);
    M355_REQUIRE(d->act == 0 || d->act == 1, "group_norm: unknown activation %d", d->act);
    M355_REQUIRE(d->aff_stride >= 0, "group_norm: the affine's rows are %lld floats apart", d->aff_stride);
    M355_REQUIRE(d->res_w >= 0 && (d->res_w == 0 || (d->res_w % 2 == 0 && HW % (2LL * d->res_w) == 0)),
                 "group_norm: a half-resolution residual needs even height and width (width %d, %lld pixels)", d->res_w, HW);
    return M355_OK;
}

static Runner runner(int dtype) { return dtype == M355_F32 ? run_f32() : dtype == M355_F16 ? run_f16() : run_bf16(); }

// f(args of these samples) over launches of at most 2^22 workgroups (of the kernels that give a group a wave, too)
template <typename F> static void by_samples(const Args &all, int esize, F f)
{
    const long long per = std::max(1LL, (1LL << 22) / std::max((long long)all.nslab * all.nblk, ((long long)all.G + kT / 64 - 1) / (kT / 64)));
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

// A call whose inputs (`bytes` a value) come near the memory-side cache's 256 MB gains nothing from leaving its outputs there: written past
// it, they neither push out what the second pass reads again nor are written back under the next kernel.  64x256x128x64 bf16: the four
// kernels 487 -> 436 us; at 32 samples (134 MB in and out) past the cache is as fast as through it, below that slower for who reads y next.
static bool past_cache(const m355_gn_desc *d, int bytes) { return (double)d->N * (double)d->HW * d->C * bytes >= 160e6; }

static unsigned wave_grid(const Args &a) { return (unsigned)(((long long)a.N * a.G + kT / 64 - 1) / (kT / 64)); }

// More than kRows rows of partial sums are added in two launches, kChunk rows a workgroup in the first: 65536 x 64, forward and backward,
// 574 -> 402 us (one launch has two workgroups for its rows there); 512 to 2048 rows: the same either way
constexpr long long kRows = 1024, kChunk = 256;

static void affine_grad(const Args &a, hipStream_t s)
{
    const long long rows = a.per_sample ? a.gnblk : (long long)a.N * a.gnblk, cols = (a.C + 31) / 32;
    const long long chunk = std::max(kChunk, (rows + 65534) / 65535), parts = rows > kRows ? (rows + chunk - 1) / chunk : 1;
    const int out = a.per_sample ? a.N : 1, per = (int)std::max(1LL, std::min(65535LL, (1LL << 21) / (cols * parts)));
    for (int n0 = 0; n0 < out; n0 += per) {
        const unsigned k = (unsigned)std::min(out - n0, per);
        float *cpart = a.cpart + (size_t)n0 * rows * 2 * a.C;
        float *dw = a.dw ? a.dw + (size_t)n0 * a.C : nullptr, *db = a.db ? a.db + (size_t)n0 * a.C : nullptr;
        if (parts > 1)
            hipLaunchKernelGGL(k_gn_affine_grad, dim3((unsigned)cols, k, (unsigned)parts), dim3(1024), 0, s, cpart, dw, db, a.C, rows, rows, 1LL,
                               chunk);
        hipLaunchKernelGGL(k_gn_affine_grad, dim3((unsigned)cols, k), dim3(1024), 0, s, cpart, dw, db, a.C, rows, parts > 1 ? parts : rows,
                           parts > 1 ? chunk : 1LL, parts > 1 ? parts : rows);
    }
}

}  // namespace gn
}  // namespace m355

using namespace m355;

extern "C" size_t m355_group_norm_ws_bytes(const m355_gn_desc *d, int backward)
{
    if (gn::check_desc(d) != M355_OK) return 0;
    const size_t N = (size_t)d->N, rows = N * (size_t)gn::most_rows(d->N, d->HW, d->C);
    size_t bytes = (rows + N) * (size_t)d->G * sizeof(float2);
    if (backward) bytes += rows * 2 * (size_t)d->C * sizeof(float);
    return (bytes + 15) / 16 * 16;
}

static void fill(gn::Args &a, const m355_gn_desc *d, const void *x, const float *w, const float *b, float *stat)
{
    a.x = x; a.w = w; a.b = b; a.mean = stat; a.rstd = stat + (size_t)d->N * d->G;
    a.aff_stride = d->aff_stride; a.hw = d->HW; a.N = (int)d->N; a.C = d->C; a.G = d->G; a.D = d->C / d->G; a.act = d->act;
    a.w_off = d->w_off; a.eps = d->eps; a.slope = d->slope; a.out_slope = d->out_slope; a.per_sample = d->per_sample != 0;
}

extern "C" int m355_group_norm_fwd(const m355_gn_desc *d, const void *x, const float *w, const float *b, const void *res, void *y, float *stat,
                                   void *ws, void *stream)
{
    const int rc = gn::check_desc(d);
    if (rc != M355_OK) return rc;
    if (d->N == 0 || d->HW == 0) return M355_OK;
    M355_REQUIRE(x && y && stat && ws, "group_norm_fwd: null pointer");
    M355_REQUIRE(x != y, "group_norm_fwd: y must not be x");
    M355_REQUIRE(d->res_w == 0 || res, "group_norm_fwd: res_w without a residual");
    gn::Args a = {};
    fill(a, d, x, w, b, stat);
    a.res = res; a.y = y; a.gpart = (float2 *)ws;
    const int C = d->C, dtype = d->dtype, res_w = d->res_w;
    gn::Choice c = {};
    gn::pick_vec(C, a.D, dtype, (uintptr_t)x | (uintptr_t)y | (uintptr_t)res, c.V, c.A);
    gn::set_groups(a, c);
    if (!gn::wide_slab(a, c.V)) {
        set_error("group_norm_fwd: groups of %d channels (vectors of %d) are wider than a workgroup takes", a.D, c.V);
        return M355_ERR_UNSUPPORTED;
    }
    const gn::Runner run = gn::runner(dtype);
    hipStream_t s = (hipStream_t)stream;
    const int es = gn::elem_bytes(dtype);
    gn::set_items(a, res_w, res_w > 0);
    gn::set_ranges(a, 1, a.items);
    a.gnblk = 1;
    if (gn::one_pass(a, c.V, es, c)) {
        gn::by_samples(a, es, [&](const gn::Args &p) { run.one(p, c, s); });
        return check_launch("group_norm_fwd");
    }
    gn::wide_slab(a, c.V);
    gn::Args st = a;
    gn::set_items(st, 0, false);
    st.res = nullptr;
    gn::take_ranges(st, gn::kStats);
    st.gnblk = a.gnblk = st.nblk;
    st.gper = a.gper = st.per;
    gn::take_ranges(a, gn::kApply);
    a.nt = gn::past_cache(d, es);
    a.finished = a.gnblk > gn::kJoin;
    gn::by_samples(st, es, [&](const gn::Args &p) { run.stats(p, c.V, c.A, s); });
    if (a.finished)
        gn::by_samples(st, es, [&](const gn::Args &p) { hipLaunchKernelGGL(gn::k_gn_finish, dim3(gn::wave_grid(p)), dim3(gn::kT), 0, s, p); });
    gn::by_samples(a, es, [&](const gn::Args &p) { run.apply(p, c.V, c.A, s); });
    return check_launch("group_norm_fwd");
}

extern "C" int m355_group_norm_bwd(const m355_gn_desc *d, const void *dy, const void *x, const float *w, const float *b, const float *stat,
                                   void *dx, float *dw, float *db, void *dres, void *ws, void *stream)
{
    const int rc = gn::check_desc(d);
    if (rc != M355_OK) return rc;
    if (d->N == 0 || d->HW == 0) return M355_OK;   // (the caller zeroes dw / db of an empty batch)
    M355_REQUIRE(dy && x && stat && ws, "group_norm_bwd: null pointer");
    M355_REQUIRE(dx != x && dx != dy, "group_norm_bwd: dx must be a tensor of its own");
    M355_REQUIRE(!dres || d->res_w > 0, "group_norm_bwd: dres is the gradient of a half-resolution residual");
    gn::Args a = {};
    fill(a, d, x, w, b, (float *)stat);
    a.dy = dy; a.y = dx; a.dres = dres; a.dw = dw; a.db = db;
    const long long N = d->N, HW = d->HW;
    const int C = d->C, G = d->G, dtype = d->dtype, res_w = d->res_w;
    gn::Choice c = {};
    gn::pick_vec(C, a.D, dtype, (uintptr_t)x | (uintptr_t)dy | (uintptr_t)dx | (uintptr_t)dres, c.V, c.A);
    gn::set_groups(a, c);
    if (!gn::wide_slab(a, c.V)) {
        set_error("group_norm_bwd: groups of %d channels (vectors of %d) are wider than a workgroup takes", a.D, c.V);
        return M355_ERR_UNSUPPORTED;
    }
    const gn::Runner run = gn::runner(dtype);
    hipStream_t s = (hipStream_t)stream;
    const int es = gn::elem_bytes(dtype);
    a.gpart = (float2 *)ws;
    a.gsum = a.gpart + (size_t)N * gn::most_rows(N, HW, C) * G;
    float *cpart = (float *)(a.gsum + (size_t)N * G);
    a.cpart = dw || db ? cpart : nullptr;
    gn::set_items(a, res_w, res_w > 0);   // (the same order of additions whether or not dres is wanted)
    gn::set_ranges(a, 1, a.items);
    a.gnblk = 1;
    if (gn::one_pass(a, c.V, es, c)) {
        gn::by_samples(a, es, [&](const gn::Args &p) { run.bwd_one(p, c, s); });
        if (!a.per_sample && a.cpart) gn::affine_grad(a, s);
        return check_launch("group_norm_bwd");
    }
    gn::wide_slab(a, c.V);
    gn::take_ranges(a, gn::kReduce);
    a.gnblk = a.nblk;
    gn::Args p2 = a;
    gn::set_items(p2, 0, false);
    p2.dres = nullptr;
    gn::take_ranges(p2, gn::kDx);
    a.nt = p2.nt = gn::past_cache(d, 2 * es);
    a.finished = p2.finished = a.gnblk > gn::kJoin;
    gn::by_samples(a, es, [&](const gn::Args &p) { run.bwd_reduce(p, c.V, c.A, s); });
    if (a.cpart) gn::affine_grad(a, s);
    if (dx) {
        if (a.finished)
            gn::by_samples(a, es, [&](const gn::Args &p) { hipLaunchKernelGGL(gn::k_gn_bwd_finish, dim3(gn::wave_grid(p)), dim3(gn::kT), 0, s, p); });
        gn::by_samples(p2, es, [&](const gn::Args &p) { run.bwd_apply(p, c.V, c.A, s); });
    }
    return check_launch("group_norm_bwd");
}
