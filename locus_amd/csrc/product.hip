// Fused and grouped matrix products: the choice of kernel, the kernels around the products
// (joining a split sum, the gradient before the activation, column and row sums) and the C entry
// points locus_hip_product_* (include/locus_hip.h).
#include <algorithm>
#include <cmath>
#include <initializer_list>
#include <utility>

#include "product.h"

namespace locus {

namespace {

// v + x[0] + x[step] + .. + x[(count - 1) step] in this order, up to DEEP of them: all loads are under way before
// the first is needed, also where there are fewer (they read the last one again).
template <int DEEP, class T> __device__ __forceinline__ T add_up(T v, const T* x, long step, int count)
{
    T t[DEEP];
#pragma unroll
    for (int u = 0; u < DEEP; ++u) t[u] = x[(u < count ? u : count - 1) * step];
#pragma unroll
    for (int u = 0; u < DEEP; ++u) v += u < count ? t[u] : T(0);
    return v;
}
template <class T> __device__ __forceinline__ T sum_of(const T* x, long step, int count)
{
    T v = T(0);
    for (; count > 8; count -= 16, x += 16 * step) v = add_up<16>(v, x, step, count);
    return count > 0 ? add_up<8>(v, x, step, count) : v;
}

// C from the partial products of a split sum, added in the order of the slices (the same result
// every time).  Bound by reading them; one thread per element along the partials' contiguous index; in
// ROWS a lane looks its row's run up for the bias.  (A 64-bit division takes as many instructions as the rest.)
template <class T, int MODE>
__global__ void __launch_bounds__(256) product_join_kernel(const ProductDesc p)
{
    const long len = (long)p.m * p.n;
    const bool by_column = MODE == PRODUCT_DENSE && p.part_m == 1;
    const int fast = by_column ? p.m : p.n;              // the contiguous index's length
    for (long e = (long)blockIdx.x * 256 + threadIdx.x; e < (len + 63) / 64 * 64; e += (long)gridDim.x * 256) {
        const long at = e < len ? e : len - 1;           // whole waves stay together for the lookup
        const long slow = len >> 32 ? at / fast : (unsigned)at / (unsigned)fast;
        const long i = by_column ? at - slow * fast : slow;
        const long j = by_column ? slow : at - slow * fast;
        const int g = MODE == PRODUCT_ROWS ? find_runs(p.offsets, p.groups, p.m, (int)i) : 0;
        if (e < len && g >= 0)
            epi_store<T>(p.epi, g * p.sbias_g, i, j, sum_of(static_cast<const T*>(p.part) + at, p.part_z, p.nz));
    }
}

// G = dC act'(pre) and the sums of its columns, per run and part of a run: bound by reading dC and
// pre and writing G.  COLS columns x 1024 / COLS rows at a time; sums[part][groups][n], or the column sums
// themselves where there is one part.  Fewer columns, down to a line of memory, where there are few workgroups.
template <class T, int COLS>
__global__ void __launch_bounds__(1024) product_slope_kernel(const locus_hip_product_grad_args a, T* G,
                                                             int parts, T* sums)
{
    constexpr int ROWS = 1024 / COLS;
    __shared__ T red[ROWS][COLS];
    const int tx = threadIdx.x % COLS, ty = threadIdx.x / COLS;
    const long j = (long)blockIdx.x * COLS + tx;
    const int part = blockIdx.y, g = blockIdx.z;
    long lo = 0, hi = a.m;
    if (a.offsets) {
        const Run r = run_rows(a.offsets, (int)a.m, g);
        lo = r.lo;
        hi = r.hi;
    }
    const long len = hi - lo;
    hi = lo + len * (part + 1) / parts;
    lo = lo + len * part / parts;
    T sum = T(0);
    if (j < a.n) {
        const T* d = static_cast<const T*>(a.dC) + j * a.sd_n + (lo + ty) * a.sd_m;
        const T* z = static_cast<const T*>(a.pre) + j * a.sp_n + (lo + ty) * a.sp_m;
        T* out = G + j + (lo + ty) * a.n;
        const bool own = a.act != LOCUS_HIP_ACT_IDENTITY;
#pragma unroll 4
        for (long i = lo + ty; i < hi; i += ROWS) {
            T v = *d;
            if (own) {
                v *= act_slope<T>(a.act, *z);
                *out = v;
            }
            sum += v;
            d += ROWS * a.sd_m;
            z += ROWS * a.sp_m;
            out += ROWS * a.n;
        }
    }
    if (sums == nullptr) return;
    red[ty][tx] = sum;
    __syncthreads();
    if (ROWS > 16) {                                     // to 16 rows
        if (ty < 16) {
#pragma unroll
            for (int q = 16; q < ROWS; q += 16) sum += red[ty + q][tx];
            red[ty][tx] = sum;
        }
        __syncthreads();
    }
    if (ty == 0 && j < a.n) {
        T v = red[0][tx];
#pragma unroll
        for (int q = 1; q < 16; ++q) v += red[q][tx];
        sums[((long)part * gridDim.z + g) * a.n + j] = v;
    }
}

template <class T>
__global__ void __launch_bounds__(256) product_sums_join_kernel(const T* sums, int parts, long len,
                                                                T* out)
{
    const long e = (long)blockIdx.x * 256 + threadIdx.x;
    if (e >= len) return;
    out[e] = sum_of(sums + e, len, parts);
}

// Sums of G's rows (the gradient of a bias per row), one wave per row.
template <class T>
__global__ void __launch_bounds__(256) product_row_sums_kernel(const T* G, long s_m, long s_n, long m,
                                                               long n, T* out)
{
    for (long i = (long)blockIdx.x * 4 + (threadIdx.x >> 6); i < m; i += (long)gridDim.x * 4) {
        T v = T(0);
        for (long j = threadIdx.x & 63; j < n; j += 64) v += G[i * s_m + j * s_n];
#pragma unroll
        for (int s = 32; s > 0; s >>= 1) v += __shfl_xor(v, s);
        if ((threadIdx.x & 63) == 0) out[i] = v;
    }
}

// workgroups for `want` pieces of work, the rest in the kernels' own loops (2^32 threads to a launch)
unsigned grid_of(long want) { return (unsigned)std::max<long>(1, std::min<long>(want, 1 << 20)); }

struct Plan {
    bool rows = false;   // the kernel for few rows
    int tw = 4;          // else: tiles of 32 tw
    bool swap = false;   // C' = B' A' (n is the short side)
    int nz = 1;
    long kchunk = 0;
    double us = 0, join_us = 0;   // what it is expected to take, and the joining launch
};

// One product: its operands and what is asked of the plan.
struct Want {
    ProductDesc p;
    int mode;
    bool f64;
    int cfg[2];
    long cus, all_cus;   // CUs it may count on, and the device's
    bool tiles_only;     // not the kernel for few rows
    double host_us;      // what a call with a workspace and another launch takes on the host: no gain below that
};

// Which kernel, tile and split: the quickest by the estimates below, whose constants are fitted to measurements: 350
// products of 1 .. 4000 rows, 20 .. 20 000 covariates and 1 .. 10 000 columns, alone or in up to 100 runs, in 26
// geometries each, replayed from a graph.  On 200 others (profiles/products_plan.csv) its choice took 5 % longer than
// the best geometry for one pair, 8 for runs, 2 and 3 for gradients, where that one takes over 20 us.
//   Joining a split sum: 2.4 us, and the partials written and read at 4.2 TB/s.  Called one by one, a workspace and
// another launch cost the host more than that (host_us), so short calls are not split.  Replayed from a graph they
// would gain by it, 8 us against 14 at most (over all of those sizes 13, 10, 6 and 2 %): such a caller names a geometry.
//   Few rows: 5.1 us, 1.2 for every round of two workgroups a CU, C and what goes with it at 9 TB/s, and the longer of:
// a wave's blocks of k, 0.36 us each, times the workgroups a CU has; what they read through L2 at 7.6 TB/s (by the
// root of what the last round leaves idle longer).
//   Tiles: a CU holds 4 workgroups of tiles of 64, 2 of 128; the share of its rate that it reaches with 1, 2, .. of
// them (2000 x 500 x 20 000, both types within 3 %), at least 0.48 us for a K-tile; 3.5 us, 3.5 and 9 for every
// round of workgroups, C and what goes with it at 9 TB/s.
//   Runs: half a tile more for each of them than their rows fill, and for tiles of 64 and 128 a standard deviation
// or two of that sum (a tile more than there are places costs a round).
Plan plan_product(const Want& w)
{
    static const short splits[] = {1, 2, 3, 4, 5, 6, 7, 8, 10, 12, 14, 16, 20, 24, 28, 32, 40, 48, 64};
    Plan best;
    double best_call = 1e300;
    const ProductDesc& p = w.p;
    const long M = p.m, N = p.n, K = p.k, s = w.f64 ? 8 : 4;
    const bool runs = w.mode == PRODUCT_ROWS, sums = w.mode == PRODUCT_SUM;
    const long copies = sums ? p.groups : 1, len = sums ? (K + copies - 1) / copies : K;   // a sum's length
    auto offer = [&](Plan pl, double us) {
        if (pl.nz > 1) pl.join_us = 2.4 + 2.0 * pl.nz * M * N * copies * s / 4.2e6;
        pl.us = us + pl.join_us;
        const double call = std::max(pl.us, pl.nz > 1 ? w.host_us : 0.0);
        if (call < best_call || (call == best_call && pl.us < best.us)) {
            best = pl;
            best_call = call;
        }
    };
    auto each_split = [&](long most, auto take) {
        if (w.cfg[1]) return take(std::min<long>(w.cfg[1], 65535 / copies));     // runs x parts: a grid's third axis
        for (const long nz : splits) {
            if (nz > 1 && (nz > most || best_call <= w.host_us)) break;
            take(nz);
        }
    };

    // us a workgroup alone on its CU takes for a million elements of the activation
    const bool cdf = p.epi.act == LOCUS_HIP_ACT_PROBIT || p.epi.act == LOCUS_HIP_ACT_GELU;
    const double heavy = p.epi.act == LOCUS_HIP_ACT_IDENTITY ? 0.0 : (w.f64 ? (cdf ? 2200.0 : 1000.0) : 400.0);
    const double mn = 1e-6 * M * N * copies, outs = s * mn * (1 + !!p.epi.res + !!p.epi.pre + (p.epi.sb_m && p.epi.sb_n));
    const bool asked = w.cfg[0] == 16;
    const long side = runs ? M / p.groups : std::min(M, N);
    if (!sums && (asked || (!w.cfg[0] && !w.tiles_only && side <= 1024))) {
        const bool swap = !runs && N < M;
        const long m = swap ? N : M, n = swap ? M : N, kb = w.f64 ? 8 : 16;
        const double rt = runs ? std::max(1.0, std::min<double>(m, m / 16.0 + 0.5 * p.groups)) : (double)((m + 15) / 16);
        const double ct = (double)((n + 63) / 64), l2 = s * K * rt * (std::max(n, 16l) + 16 * ct) / 7.6e6;
        each_split(std::min<long>(64, K / (4 * kb)), [&](long nz) {
            Plan pl;
            pl.rows = true;
            pl.swap = swap;
            pl.kchunk = ((K + nz - 1) / nz + 4 * kb - 1) / (4 * kb) * (4 * kb);
            pl.nz = pl.kchunk > 0 ? (int)((K + pl.kchunk - 1) / pl.kchunk) : 1;
            const double wgs = rt * ct * pl.nz;
            const double even = std::ceil(wgs / w.cus) * w.cus / wgs;    // the CUs' share of the last round
            offer(pl, 5.1 + std::max(pl.kchunk / (4 * kb) * 0.36 * std::ceil(wgs / w.cus), l2 * std::sqrt(even)) +
                          1.2 * std::ceil(wgs / (2 * w.cus)) + outs / 9.0 +
                          (pl.nz == 1 ? mn * heavy / (2 * w.cus) : 0.0));
        });
    }
    if (asked && !sums) return best;

    // (the plan's own time, 1 to 2 us, counts in small calls: no tiles where they cannot be quicker)
    const long bk = w.f64 ? 16 : 32;
    if (!w.cfg[0] && best_call <= std::min(7.0 + 0.48 * len / bk, w.host_us)) return best;
    const double cu_rate = (w.f64 ? 75e6 : 150e6) / w.all_cus;   // flop per us
    for (int tw = 4; tw >= 2; tw -= 2) {
        if (w.cfg[0] >= 64 && w.cfg[0] != 32 * tw) continue;
        const long bm = 32 * tw;
        const long mt = runs ? (long)((double)M / bm + 0.5 * p.groups + 0.5 * std::sqrt((double)p.groups) + 0.5)
                             : (M + bm - 1) / bm;
        const long tiles = std::max<long>(mt, 1) * ((N + bm - 1) / bm) * copies;
        const long most = std::min<long>(std::min<long>(32, len / (4 * bk)), 65535 / copies);
        each_split(most, [&](long nz) {
            Plan pl;
            pl.tw = tw;
            pl.kchunk = ((len + nz - 1) / nz + bk - 1) / bk * bk;
            pl.nz = sums ? (int)nz : (int)(K > 0 ? (K + pl.kchunk - 1) / pl.kchunk : 1);
            const long wgs = tiles * pl.nz, load = (wgs + w.cus - 1) / w.cus, slots = tw == 4 ? 2 : 4;
            static const double share2[5] = {0, 0.67, 0.80, 0.86, 0.90}, share4[3] = {0, 0.86, 0.92};
            const double* share = tw == 4 ? share4 : share2;
            const double one = 2.0 * bm * bm * pl.kchunk / cu_rate;      // a workgroup's products on its CU
            const long rest = load % slots;
            const double rounds = (double)((load + slots - 1) / slots);
            double t = 3.5 + rounds * (tw == 4 ? 9.0 : 3.5) + outs / 9.0 +
                       std::max(one * ((load - rest) / share[slots] + (rest ? rest / share[rest] : 0.0)),
                                0.48 * pl.kchunk / bk * rounds);
            // the element function: in the epilogue by a CU's workgroups, after a split by all CUs
            const double f = 1e-6 * bm * bm * heavy;
            t += pl.nz == 1 ? f * std::max<double>(1.0, (double)wgs / w.cus / 2) : f * tiles / w.cus / 2;
            offer(pl, t);
        });
    }
    return best;
}

long plan_bytes(const Want& w, const Plan& pl)
{
    const long copies = w.mode == PRODUCT_SUM ? w.p.groups : 1;
    return pl.nz > 1 ? (long)pl.nz * w.p.m * w.p.n * copies * (w.f64 ? 8 : 4) : 0;
}

// The descriptor as the kernels take it: roles swapped, split sum in `part`.
ProductDesc planned(const Want& w, const Plan& pl, void* part)
{
    ProductDesc p = w.p;
    ProductEpi& e = p.epi;
    if (pl.swap) {
        std::swap(p.m, p.n);
        std::swap(p.A, p.B);
        const long am = p.sa_m, ak = p.sa_k;
        p.sa_m = p.sb_n; p.sa_k = p.sb_k;
        p.sb_n = am; p.sb_k = ak;
        std::swap(e.sc_m, e.sc_n);
        std::swap(e.sb_m, e.sb_n);
        std::swap(e.sr_m, e.sr_n);
        std::swap(e.sp_m, e.sp_n);
    }
    p.nz = std::max(1, pl.nz);
    p.kchunk = (int)pl.kchunk;
    if (pl.nz > 1) {
        p.part = part;
        p.part_z = (long)p.m * p.n * (w.mode == PRODUCT_SUM ? p.groups : 1);
        const bool mfast = w.mode == PRODUCT_DENSE && e.sc_n != 1 && e.sc_m == 1 && !pl.rows;
        p.part_m = mfast ? 1 : p.n;
        p.part_n = mfast ? p.m : 1;
    }
    return p;
}

template <class T> int join_product(ProductDesc p, int mode, hipStream_t st)
{
    if (p.nz <= 1) return 0;
    if (mode == PRODUCT_SUM) {                 // the runs' C lie one behind the other, as their partials do
        p.m *= p.groups;
        mode = PRODUCT_DENSE;
    }
    const dim3 grid(grid_of(((long)p.m * p.n + 255) / 256));
    if (mode == PRODUCT_DENSE) hipLaunchKernelGGL((product_join_kernel<T, PRODUCT_DENSE>), grid, dim3(256), 0, st, p);
    else hipLaunchKernelGGL((product_join_kernel<T, PRODUCT_ROWS>), grid, dim3(256), 0, st, p);
    LOCUS_HIP_CHECK(hipGetLastError());
    return 0;
}

template <class T> int run_product(const Want& w, const Plan& pl, void* part, hipStream_t st)
{
    if (w.p.m == 0 || w.p.n == 0) return 0;
    const ProductDesc p = planned(w, pl, part);
    const int rc = pl.rows ? launch_product_rows<T>(p, w.mode, st) : launch_product_tile<T>(p, w.mode, pl.tw, st);
    return rc ? rc : join_product<T>(p, w.mode, st);
}

int check_common(const char* what, int64_t m, int64_t n, int64_t k, int dtype, int act, int mode, const int32_t* cfg,
                 int64_t groups, const void* gather, int64_t a_rows)
{
    const std::string w(what);
    LOCUS_REQUIRE(dtype == LOCUS_HIP_F64 || dtype == LOCUS_HIP_F32, w + ": dtype");
    LOCUS_REQUIRE(act >= LOCUS_HIP_ACT_IDENTITY && act <= LOCUS_HIP_ACT_SILU, w + ": act");
    LOCUS_REQUIRE(mode == LOCUS_HIP_PRODUCT_DENSE || mode == LOCUS_HIP_PRODUCT_ROWS, w + ": mode");
    LOCUS_REQUIRE(m >= 0 && n >= 0 && k >= 0 && m < (1ll << 29) && n <= 65535 * 64 && k < (1ll << 29),
                  w + ": sizes (m, k < 2^29, n <= 4194240)");
    LOCUS_REQUIRE(cfg[0] == 0 || cfg[0] == 16 || cfg[0] == 64 || cfg[0] == 128, w + ": cfg[0] is 0, 16, 64 or 128");
    LOCUS_REQUIRE(cfg[1] >= 0 && cfg[1] <= 256, w + ": cfg[1] is 0..256");
    LOCUS_REQUIRE(cfg[0] != 16 || (mode == LOCUS_HIP_PRODUCT_DENSE ? std::min(m, n) <= 65535 * 16 : m < (1ll << 27)),
                  w + ": too many rows for the kernel for few");
    if (mode == LOCUS_HIP_PRODUCT_ROWS) {
        LOCUS_REQUIRE(groups >= 1 && groups <= 65535, w + ": groups (1..65535)");
        LOCUS_REQUIRE(!gather || (a_rows >= 0 && a_rows < (1ll << 31)), w + ": a_rows");
    }
    return 0;
}

// 0: there is enough; else what the entry point returns.
int64_t no_workspace(int64_t need, const void* ws, int64_t bytes, const char* fn)
{
    if (need == 0) return 0;
    if (!ws) return need;
    if (bytes >= need) return 0;
    set_error(std::string("workspace smaller than ") + fn);
    return LOCUS_HIP_EWORKSPACE;
}

int check_product(const locus_hip_product_args* a)
{
    LOCUS_REQUIRE(a, "product: no arguments");
    return check_common("product", a->m, a->n, a->k, a->dtype, a->act, a->mode, a->cfg, a->groups, a->gather, a->a_rows);
}

// The bytes that a strided array spans.
struct Span {
    const char *lo = nullptr, *hi = nullptr;
    const char* at = nullptr;
    long size = 0, n[3] = {1, 1, 1}, s[3] = {0, 0, 0};
    Span(const void* p, long bytes, std::initializer_list<std::pair<long, long>> dims)
    {
        if (!p) return;
        long back = 0, ahead = 0;
        int q = 0;
        for (auto [len, step] : dims) {
            if (len == 0) return;
            n[q] = len;
            s[q++] = step * bytes;
            (step < 0 ? back : ahead) += (len - 1) * step;
        }
        at = static_cast<const char*>(p);
        size = bytes;
        lo = at + back * bytes;
        hi = at + (ahead + 1) * bytes;
    }
    // [from, to): where the array's bytes lie within a period, counted from `at`; dimensions whose stride is a
    // whole number of periods do not count
    std::pair<long, long> within(long period) const
    {
        long from = 0, to = size;
        for (int q = 0; q < 3; ++q)
            if (s[q] % period) (s[q] < 0 ? from : to) += (n[q] - 1) * s[q];
        return {from, to};
    }
    // Blocks of columns of one matrix lie within each other's span and share nothing: with the matrix's row
    // as the period, one begins behind the other's end and ends before its next row.
    bool meets(const Span& o) const
    {
        if (!(lo < o.hi && o.lo < hi)) return false;
        for (const Span* x : {this, &o})
            for (int q = 0; q < 3; ++q) {
                const long period = x->s[q] < 0 ? -x->s[q] : x->s[q];
                if (x->n[q] < 2 || period <= size) continue;
                const auto [a0, a1] = within(period);
                const auto [b0, b1] = o.within(period);
                const long gap = (((long)(o.at - at) + b0 - a0) % period + period) % period;
                if (gap >= a1 - a0 && gap + (b1 - b0) <= period) return false;
            }
        return common(o);
    }
    // Whether two of their elements share a byte: o.at - at + sum (o's steps) - sum (own steps), one term for each
    // different stride, comes between -o.size and size.  The largest stride's multiples that the others can still
    // bring there are few where strides are nested, as in views of one matrix; more than 4096 tries count as shared.
    bool common(const Span& o) const
    {
        struct Term {
            long step, lo, hi;
        } t[6];
        int terms = 0;
        auto add = [&](long step, long lo, long hi) {
            if (step == 0 || lo == hi) return;
            if (step < 0) {
                step = -step;
                std::swap(lo, hi);
                lo = -lo;
                hi = -hi;
            }
            for (int q = 0; q < terms; ++q)
                if (t[q].step == step) {
                    t[q].lo += lo;
                    t[q].hi += hi;
                    return;
                }
            t[terms++] = {step, lo, hi};
        };
        for (int q = 0; q < 3; ++q) {
            add(o.s[q], 0, o.n[q] - 1);
            add(s[q], 1 - n[q], 0);
        }
        std::sort(t, t + terms, [](const Term& a, const Term& b) { return a.step > b.step; });
        long lo[7] = {}, hi[7] = {};                     // what the terms from q on can add
        for (int q = terms - 1; q >= 0; --q) {
            lo[q] = lo[q + 1] + t[q].lo * t[q].step;
            hi[q] = hi[q + 1] + t[q].hi * t[q].step;
        }
        auto floor_div = [](long a, long b) { return a >= 0 ? a / b : -((-a + b - 1) / b); };
        int tries = 0;
        auto search = [&](auto&& self, int q, long sum) -> bool {
            if (q == terms) return -o.size < sum && sum < size;
            long x = std::max(t[q].lo, -floor_div(sum + hi[q + 1] + o.size - 1, t[q].step));
            const long end = std::min(t[q].hi, floor_div(size - 1 - sum - lo[q + 1], t[q].step));
            for (; x <= end; ++x)
                if (++tries > 4096 || self(self, q + 1, sum + x * t[q].step)) return true;
            return false;
        };
        return search(search, 0, (long)(o.at - at));
    }
};

// Rows (or columns) that lie one behind the other: every element has memory of its own.
bool apart(long m, long sm, long n, long sn)
{
    sm = sm < 0 ? -sm : sm;
    sn = sn < 0 ? -sn : sn;
    if (m == 1) return n == 1 || sn >= 1;
    if (n == 1) return sm >= 1;
    return sm <= sn ? sm >= 1 && sn > sm * (m - 1) : sn >= 1 && sm > sn * (n - 1);
}

int check_spans(const locus_hip_product_args& a)
{
    const long s = a.dtype == LOCUS_HIP_F64 ? 8 : 4;
    const bool runs = a.mode == LOCUS_HIP_PRODUCT_ROWS;
    const long groups = runs ? a.groups : 1;
    const Span C(a.C, s, {{a.m, a.sc_m}, {a.n, a.sc_n}}), pre(a.pre, s, {{a.m, a.sp_m}, {a.n, a.sp_n}});
    const Span res(a.res, s, {{a.m, a.sr_m}, {a.n, a.sr_n}});
    const Span reads[] = {Span(a.A, s, {{runs && a.gather ? a.a_rows : a.m, a.sa_m}, {a.k, a.sa_k}}),
                          Span(a.B, s, {{groups, a.sb_g}, {a.k, a.sb_k}, {a.n, a.sb_n}}),
                          Span(a.bias, s, {{groups, a.sbias_g}, {a.m, a.sbias_m}, {a.n, a.sbias_n}}),
                          Span(runs ? a.offsets : nullptr, 8, {{groups + 1, 1}}),
                          Span(runs ? a.gather : nullptr, 8, {{a.m, 1}})};
    LOCUS_REQUIRE(apart(a.m, a.sc_m, a.n, a.sc_n), "product: elements of C share memory");
    LOCUS_REQUIRE(!a.pre || apart(a.m, a.sp_m, a.n, a.sp_n), "product: elements of pre share memory");
    for (const Span& r : reads)
        LOCUS_REQUIRE(!C.meets(r) && !pre.meets(r), "product: C or pre shares memory with what is read");
    LOCUS_REQUIRE(!C.meets(pre), "product: C shares memory with pre");
    LOCUS_REQUIRE(!pre.meets(res), "product: pre shares memory with the residual");
    // (one row's or column's stride says nothing)
    const bool same = a.C == a.res && (a.m == 1 || a.sc_m == a.sr_m) && (a.n == 1 || a.sc_n == a.sr_n);
    LOCUS_REQUIRE(same || !C.meets(res),
                  "product: C shares memory with the residual and is not it");
    return 0;
}

Want want_product(const locus_hip_product_args& a)
{
    Want w = {};
    ProductDesc& p = w.p;
    p.m = (int)a.m; p.n = (int)a.n; p.k = (int)a.k;
    p.A = a.A; p.sa_m = a.sa_m; p.sa_k = a.sa_k;
    p.B = a.B; p.sb_k = a.sb_k; p.sb_n = a.sb_n;
    ProductEpi& e = p.epi;
    e.C = a.C; e.sc_m = a.sc_m; e.sc_n = a.sc_n;
    e.bias = a.bias; e.sb_m = a.sbias_m; e.sb_n = a.sbias_n;
    e.res = a.res; e.sr_m = a.sr_m; e.sr_n = a.sr_n;
    e.pre = a.pre; e.sp_m = a.sp_m; e.sp_n = a.sp_n;
    e.alpha = a.alpha; e.beta = a.beta; e.act = a.act;
    if (a.mode == LOCUS_HIP_PRODUCT_ROWS) {
        p.groups = (int)a.groups;
        p.offsets = a.offsets;
        p.sb_g = a.sb_g; p.sbias_g = a.sbias_g;
        p.gather = a.gather;
        p.a_rows = a.a_rows;
        p.fill_rest = a.fill_rest;
    }
    w.mode = a.mode;
    w.f64 = a.dtype == LOCUS_HIP_F64;
    w.cfg[0] = a.cfg[0]; w.cfg[1] = a.cfg[1];
    w.cus = w.all_cus = real_cus();          // (LOCUS_HIP_MFMA_CUS is for the sweeps' launch plan)
    w.host_us = 14.5;
    return w;
}

// ---- gradient ------------------------------------------------------------------------------------

// How product_slope_kernel is cut.  Columns of a workgroup (of 16 waves): 64, or fewer, down to 128 bytes, while all
// workgroups run side by side, one on a CU in float64 (94 registers), two in float32.  Then parts of a run, up to two
// workgroups per CU.  A part has rows enough to be worth the launch that joins them: 16 waves do 256 rows of 64 columns without an
// activation, 64 with one (a 16-row turn of a float64 slope takes 2 to 3 us on a CU) in its time.
struct SlopeCut {
    int cols, parts;
};
SlopeCut slope_cut(const locus_hip_product_grad_args& a, long cus)
{
    const long groups = std::max<long>(1, a.groups), least_cols = a.dtype == LOCUS_HIP_F64 ? 16 : 32;
    SlopeCut c = {64, 1};
    auto blocks = [&] { return (a.n + c.cols - 1) / c.cols * groups; };
    const long room = a.dtype == LOCUS_HIP_F64 ? cus : 2 * cus;
    while (c.cols > least_cols && 2 * blocks() <= room && a.m * c.cols > groups * 1024) c.cols /= 2;
    const long least = (a.act == LOCUS_HIP_ACT_IDENTITY ? 256 : 64) * 64 / c.cols;
    const long want = std::min<long>(2 * cus / std::max<long>(1, blocks()), a.m / groups / least);
    c.parts = (int)std::max<long>(1, std::min<long>(want, 1024));
    return c;
}

int check_grad(const locus_hip_product_grad_args* a)
{
    LOCUS_REQUIRE(a, "product_grad: no arguments");
    int rc = check_common("product_grad", a->m, a->n, a->k, a->dtype, a->act, a->mode, a->cfg, a->groups, a->gather,
                          a->a_rows);
    if (rc) return rc;
    LOCUS_REQUIRE(a->k <= 65535 * 64, "product_grad: sizes (k <= 4194240)");
    LOCUS_REQUIRE(!(a->row_sums && a->mode == LOCUS_HIP_PRODUCT_ROWS), "product_grad: row sums are for one pair of matrices");
    LOCUS_REQUIRE(!(a->G && a->act == LOCUS_HIP_ACT_IDENTITY), "product_grad: with act = identity, G is dC: pass NULL");
    return 0;
}

int check_grad_spans(const locus_hip_product_grad_args& a)
{
    const long s = a.dtype == LOCUS_HIP_F64 ? 8 : 4, groups = std::max<long>(1, a.groups);
    const Span writes[] = {Span(a.G, s, {{a.m, a.n}, {a.n, 1}}), Span(a.dA, s, {{a.m, a.k}, {a.k, 1}}),
                           Span(a.dB, s, {{groups * a.k, a.n}, {a.n, 1}}), Span(a.col_sums, s, {{groups, a.n}, {a.n, 1}}),
                           Span(a.row_sums, s, {{a.m, 1}})};
    const Span reads[] = {Span(a.dC, s, {{a.m, a.sd_m}, {a.n, a.sd_n}}),
                          Span(a.act != LOCUS_HIP_ACT_IDENTITY ? a.pre : nullptr, s, {{a.m, a.sp_m}, {a.n, a.sp_n}}),
                          Span(a.dB ? a.A : nullptr, s, {{a.gather ? a.a_rows : a.m, a.sa_m}, {a.k, a.sa_k}}),
                          Span(a.dA ? a.B : nullptr, s, {{groups, a.sb_g}, {a.k, a.sb_k}, {a.n, a.sb_n}}),
                          Span(a.offsets, 8, {{groups + 1, 1}}), Span(a.gather, 8, {{a.m, 1}})};
    for (const Span& w : writes) {
        for (const Span& r : reads) LOCUS_REQUIRE(!w.meets(r), "product_grad: an output shares memory with what is read");
        for (const Span& o : writes) LOCUS_REQUIRE(&o == &w || !w.meets(o), "product_grad: two outputs share memory");
    }
    return 0;
}

// One pair of matrices has no runs, whatever those fields hold.
locus_hip_product_grad_args own_fields(locus_hip_product_grad_args a)
{
    if (a.mode == LOCUS_HIP_PRODUCT_DENSE) {
        a.groups = a.sb_g = a.a_rows = 0;
        a.offsets = a.gather = nullptr;
    }
    return a;
}

// What a gradient launches: workspace [G | column sums | partials of dA | partials of dB].
struct Grad {
    bool pair;                         // both products in one launch
    bool own_g, slope;                 // G in the workspace; G or sums are asked for
    SlopeCut cut;
    Want da, db;
    Plan pa, pb;
    long g_bytes, s_bytes, a_bytes, b_bytes;
    long all() const { return g_bytes + s_bytes + a_bytes + b_bytes; }
};

bool pairs(const ProductDesc& p, int mode, int tw, const ProductDesc& q, int qmode, int qtw, bool f64)
{
    return f64 ? product_pairs<double>(p, mode, tw, q, qmode, qtw) : product_pairs<float>(p, mode, tw, q, qmode, qtw);
}

Grad plan_grad(const locus_hip_product_grad_args& a)
{
    auto up = [](long v) { return (v + 255) / 256 * 256; };
    Grad r = {};
    const bool runs = a.mode == LOCUS_HIP_PRODUCT_ROWS, act = a.act != LOCUS_HIP_ACT_IDENTITY;
    const long s = a.dtype == LOCUS_HIP_F64 ? 8 : 4;
    r.own_g = act && !a.G;
    r.slope = act || a.col_sums;
    const long cus = real_cus();
    r.cut = slope_cut(a, cus);
    r.g_bytes = r.own_g ? up(a.m * a.n * s) : 0;
    r.s_bytes = a.col_sums && r.cut.parts > 1 ? up(r.cut.parts * std::max<long>(1, a.groups) * a.n * s) : 0;
    // G is row-major m x n, for the identity dC as it is
    const long g_m = act ? a.n : a.sd_m, g_n = act ? 1 : a.sd_n;
    Want w = {};
    w.f64 = a.dtype == LOCUS_HIP_F64;
    w.cfg[0] = a.cfg[0]; w.cfg[1] = a.cfg[1];
    w.cus = w.all_cus = cus;
    w.host_us = 16.0;
    w.p.epi.alpha = a.alpha;
    if (runs) {
        w.p.groups = (int)a.groups;
        w.p.offsets = a.offsets;
    }
    // dA = alpha G B'
    r.da = w;
    ProductDesc& p = r.da.p;
    r.da.mode = a.mode;
    p.m = (int)a.m; p.n = (int)a.k; p.k = (int)a.n;
    p.sa_m = g_m; p.sa_k = g_n;
    p.B = a.B; p.sb_k = a.sb_n; p.sb_n = a.sb_k; p.sb_g = a.sb_g;
    p.epi.C = a.dA; p.epi.sc_m = a.k; p.epi.sc_n = 1;
    p.fill_rest = runs;
    // dB = alpha A' G, per run
    r.db = w;
    ProductDesc& q = r.db.p;
    r.db.mode = runs ? PRODUCT_SUM : PRODUCT_DENSE;
    q.m = (int)a.k; q.n = (int)a.n; q.k = (int)a.m;
    q.A = a.A; q.sa_m = a.sa_k; q.sa_k = a.sa_m;
    q.sb_k = g_m; q.sb_n = g_n;
    q.epi.C = a.dB; q.epi.sc_m = a.n; q.epi.sc_n = 1;
    q.sc_g = a.k * a.n;
    if (runs) { q.gather = a.gather; q.a_rows = a.a_rows; }
    if (a.k * std::max<long>(1, a.groups) >= (1l << 31)) r.db.cfg[1] = 1;       // dB's rows are counted in 32 bits
    if (a.dA) r.pa = plan_product(r.da);
    if (a.dB) r.pb = plan_product(r.db);
    if (a.dA && a.dB && a.cfg[0] != 16) {
        // both in one launch, tiles of one size, each with half the CUs; or one after the other (the second
        // launch comes about 4 us cheaper than the estimate of one alone)
        Want da = r.da, db = r.db;
        da.cus = db.cus = std::max<long>(1, cus / 2);
        da.tiles_only = db.tiles_only = true;
        Plan pa = plan_product(da), pb = plan_product(db);
        if (pa.tw != pb.tw) {
            da.cfg[0] = db.cfg[0] = 64;
            pa = plan_product(da);
            pb = plan_product(db);
        }
        const double joins = pa.join_us + pb.join_us;
        void* const some = &r;         // (where partials lie does not matter here)
        if (std::max(pa.us - pa.join_us, pb.us - pb.join_us) + joins <= r.pa.us + r.pb.us - 4.0 &&
            pairs(planned(da, pa, some), da.mode, pa.tw, planned(db, pb, some), db.mode, pb.tw, w.f64)) {
            r.pair = true;
            r.pa = pa;
            r.pb = pb;
        }
    }
    if (a.dA) r.a_bytes = up(plan_bytes(r.da, r.pa));
    if (a.dB) r.b_bytes = up(plan_bytes(r.db, r.pb));
    return r;
}

template <class T> int run_grad(const locus_hip_product_grad_args& a, Grad& r, hipStream_t st)
{
    char* ws = static_cast<char*>(a.workspace);
    const bool act = a.act != LOCUS_HIP_ACT_IDENTITY;
    T* G = static_cast<T*>(r.own_g ? ws : a.G);
    T* sums = static_cast<T*>(r.s_bytes ? ws + r.g_bytes : a.col_sums);
    if (r.slope && a.n > 0) {
        const unsigned groups = (unsigned)std::max<long>(1, a.groups);
        const dim3 grid((unsigned)((a.n + r.cut.cols - 1) / r.cut.cols), (unsigned)r.cut.parts, groups);
        auto go = [&](auto kern) { hipLaunchKernelGGL(kern, grid, dim3(1024), 0, st, a, G, r.cut.parts, sums); };
        if (r.cut.cols == 64) go(product_slope_kernel<T, 64>);
        else if (r.cut.cols == 32) go(product_slope_kernel<T, 32>);
        else go(product_slope_kernel<T, 16>);
        LOCUS_HIP_CHECK(hipGetLastError());
        if (r.s_bytes) {
            const long len = (long)groups * a.n;
            hipLaunchKernelGGL(product_sums_join_kernel<T>, dim3((unsigned)((len + 255) / 256)), dim3(256), 0, st, sums,
                               r.cut.parts, len, static_cast<T*>(a.col_sums));
            LOCUS_HIP_CHECK(hipGetLastError());
        }
    }
    if (a.row_sums && a.m > 0) {
        hipLaunchKernelGGL(product_row_sums_kernel<T>, dim3(grid_of((a.m + 3) / 4)), dim3(256), 0, st,
                           act ? G : static_cast<const T*>(a.dC), act ? a.n : a.sd_m, act ? 1L : a.sd_n, a.m, a.n,
                           static_cast<T*>(a.row_sums));
        LOCUS_HIP_CHECK(hipGetLastError());
    }
    r.da.p.A = r.db.p.B = act ? G : a.dC;
    void* const pa = ws + r.g_bytes + r.s_bytes;
    void* const pb = ws + r.g_bytes + r.s_bytes + r.a_bytes;
    const bool da = a.dA && a.m > 0 && a.k > 0, db = a.dB && a.k > 0 && a.n > 0;
    if (da && db && r.pair) {
        const ProductDesc p = planned(r.da, r.pa, pa), q = planned(r.db, r.pb, pb);
        int rc = launch_product_pair<T>(p, r.da.mode, q, r.pa.tw, st);
        if (!rc) rc = join_product<T>(p, r.da.mode, st);
        return rc ? rc : join_product<T>(q, r.db.mode, st);
    }
    if (da) {
        const int rc = run_product<T>(r.da, r.pa, pa, st);
        if (rc) return rc;
    }
    return db ? run_product<T>(r.db, r.pb, pb, st) : 0;
}

}  // namespace
}  // namespace locus

using namespace locus;

extern "C" {

int64_t locus_hip_product_workspace_bytes(const locus_hip_product_args* args)
{
    const int rc = check_product(args);
    if (rc) return rc;
    const Want w = want_product(*args);
    return args->m == 0 || args->n == 0 ? 0 : plan_bytes(w, plan_product(w));
}

int64_t locus_hip_product_dev(const locus_hip_product_args* args, void* stream)
{
    int rc = check_product(args);
    if (rc) return rc;
    const locus_hip_product_args& a = *args;
    if (a.m == 0 || a.n == 0) return 0;
    LOCUS_REQUIRE(a.C && (a.k == 0 || (a.A && a.B)), "product: null pointer");
    LOCUS_REQUIRE(a.mode == LOCUS_HIP_PRODUCT_DENSE || a.offsets, "product: runs need offsets");
    LOCUS_REQUIRE(a.mode == LOCUS_HIP_PRODUCT_DENSE || !a.gather || a.a_rows > 0 || a.k == 0,
                  "product: rows gathered from an empty matrix");
    if ((rc = check_spans(a))) return rc;
    const Want w = want_product(a);
    const Plan pl = plan_product(w);
    const int64_t lack = no_workspace(plan_bytes(w, pl), a.workspace, a.workspace_bytes, "locus_hip_product_workspace_bytes()");
    if (lack) return lack;
    return w.f64 ? run_product<double>(w, pl, a.workspace, (hipStream_t)stream)
                 : run_product<float>(w, pl, a.workspace, (hipStream_t)stream);
}

int64_t locus_hip_product_grad_workspace_bytes(const locus_hip_product_grad_args* args)
{
    const int rc = check_grad(args);
    return rc ? rc : plan_grad(own_fields(*args)).all();
}

int64_t locus_hip_product_grad_dev(const locus_hip_product_grad_args* args, void* stream)
{
    int rc = check_grad(args);
    if (rc) return rc;
    const locus_hip_product_grad_args a = own_fields(*args);
    const bool act = a.act != LOCUS_HIP_ACT_IDENTITY;
    LOCUS_REQUIRE(a.m == 0 || a.n == 0 || (a.dC && (!act || a.pre)), "product_grad: null pointer");
    LOCUS_REQUIRE(!a.dA || a.B || a.k == 0 || a.n == 0 || a.m == 0, "product_grad: dA needs B");
    LOCUS_REQUIRE(!a.dB || a.A || a.k == 0 || a.n == 0 || a.m == 0, "product_grad: dB needs A");
    LOCUS_REQUIRE(a.mode == LOCUS_HIP_PRODUCT_DENSE || a.offsets, "product_grad: runs need offsets");
    LOCUS_REQUIRE(a.mode == LOCUS_HIP_PRODUCT_DENSE || !a.gather || a.a_rows > 0 || a.m == 0 || a.k == 0,
                  "product_grad: rows gathered from an empty matrix");
    if ((rc = check_grad_spans(a))) return rc;
    Grad r = plan_grad(a);
    const int64_t lack = no_workspace(r.all(), a.workspace, a.workspace_bytes, "locus_hip_product_grad_workspace_bytes()");
    if (lack) return lack;
    return a.dtype == LOCUS_HIP_F64 ? run_grad<double>(a, r, (hipStream_t)stream) : run_grad<float>(a, r, (hipStream_t)stream);
}

}  // extern "C"
