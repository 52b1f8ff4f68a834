// Fused and grouped matrix products: the choice of kernel, the kernels around the products
// (joining a split sum, the gradient before the activation, column and row sums) and the C entry
// points locus_hip_product_* (include/locus_hip.h).
#include <algorithm>

#include "product.h"

namespace locus {

namespace {

// C from the partial products of a split sum, added in the order of the slices (the same result
// every time).  Bound by reading them; DENSE: one thread per element along the partials' contiguous index;
// ROWS: a workgroup per row, which looks its run up for the bias.
template <class T, int MODE>
__global__ void __launch_bounds__(256) product_join_kernel(const ProductDesc p)
{
    auto join = [&](long bias0, long i, long j) {
        const T* x = static_cast<const T*>(p.part) + i * p.part_m + j * p.part_n;
        T v = T(0);
#pragma unroll 8
        for (int z = 0; z < p.nz; ++z) v += x[z * p.part_z];
        epi_store<T>(p.epi, bias0, i, j, v);
    };
    if constexpr (MODE == PRODUCT_DENSE) {
        const long len = (long)p.m * p.n;
        for (long e = (long)blockIdx.x * 256 + threadIdx.x; e < len; e += (long)gridDim.x * 256) {
            if (p.part_m == 1) join(0, e % p.m, e / p.m);
            else join(0, e / p.n, e % p.n);
        }
    } else {
        const long j = (long)blockIdx.y * 256 + threadIdx.x;
        for (long i = blockIdx.x; i < p.m; i += gridDim.x) {
            const Run r = find_run(p.offsets, p.groups, p.m, i, 0);
            if (r.g >= 0 && j < p.n) join(r.g * p.sbias_g, i, j);
        }
    }
}

// G = dC act'(pre) and the sums of its columns, per run and part of a run: bound by reading dC and
// pre and writing G.  64 columns x 4 rows at a time; sums[part][groups][n], or dbias where there is one part.
template <class T>
__global__ void __launch_bounds__(256) product_slope_kernel(const locus_hip_product_slope_args a,
                                                            int parts, T* sums)
{
    __shared__ T red[4][64];
    const int tx = threadIdx.x & 63, ty = threadIdx.x >> 6;
    const long j = (long)blockIdx.x * 64 + tx;
    const int part = blockIdx.y, g = blockIdx.z;
    long lo = 0, hi = a.m;
    if (a.offsets) {
        const Run r = run_rows(a.offsets, a.m, g);
        lo = r.lo;
        hi = r.hi;
    }
    const long len = hi - lo;
    hi = lo + len * (part + 1) / parts;
    lo = lo + len * part / parts;
    T sum = T(0);
    if (j < a.n) {
        const T* d = static_cast<const T*>(a.dC) + j * a.sd_n;
        const T* z = static_cast<const T*>(a.pre) + j * a.sp_n;
        T* out = static_cast<T*>(a.G) + j;
#pragma unroll 4
        for (long i = lo + ty; i < hi; i += 4) {
            T v = d[i * a.sd_m];
            if (a.act != LOCUS_HIP_ACT_IDENTITY) v *= act_slope<T>(a.act, z[i * a.sp_m]);
            if (a.G) out[i * a.n] = v;
            sum += v;
        }
    }
    if (sums == nullptr) return;
    red[ty][tx] = sum;
    __syncthreads();
    if (ty == 0 && j < a.n) {
        const long at = ((long)part * gridDim.z + g) * a.n + j;
        sums[at] = (red[0][tx] + red[1][tx]) + (red[2][tx] + red[3][tx]);
    }
}

template <class T>
__global__ void __launch_bounds__(256) product_sums_join_kernel(const T* sums, int parts, long len,
                                                                T* out)
{
    const long e = (long)blockIdx.x * 256 + threadIdx.x;
    if (e >= len) return;
    T v = T(0);
#pragma unroll 8
    for (int q = 0; q < parts; ++q) v += sums[q * len + e];
    out[e] = v;
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
    int rows_mt = 0;     // > 0: the kernel for few rows, with so many 16-row tiles
    int tw = 0;          // else: tiles of 32 tw
    bool swap = false;   // C' = B' A' (n is the short side)
    int nz = 1;
    long kchunk = 0;
};

// Which kernel, tile and split.  Times in microseconds from rates measured on this card (tiles:
// what a CU reaches with one and with several workgroups on it; joining: the partials written and
// read at 4.5 TB/s and one more launch).
Plan plan_product(const locus_hip_product_args& a)
{
    Plan pl;
    const bool f64 = a.dtype == LOCUS_HIP_F64;
    const long s = f64 ? 8 : 4;
    const long cus = device_cus();
    const bool runs = a.mode == LOCUS_HIP_PRODUCT_ROWS;
    const double avg = runs ? (double)a.m / a.groups : (double)a.m;
    const long bk = f64 ? 16 : 32;
    pl.kchunk = a.k;
    if (a.mode == LOCUS_HIP_PRODUCT_SUM) {
        const long t128 = ((a.m + 127) / 128) * ((a.n + 127) / 128) * a.groups;
        pl.tw = a.cfg[0] ? a.cfg[0] / 32 : (t128 >= 2 * cus && a.m > 64 && a.n > 64 ? 4 : 2);
        return pl;
    }
    const long shortside = runs ? (long)avg : std::min(a.m, a.n);
    const bool rows = a.cfg[0] ? a.cfg[0] <= 4 : shortside <= 64;
    if (rows) {
        pl.swap = !runs && a.n < a.m;
        const long m = pl.swap ? a.n : a.m, n = pl.swap ? a.m : a.n;
        const double per = runs ? avg : (double)m;
        pl.rows_mt = a.cfg[0] ? a.cfg[0] : (per <= 16 ? 1 : (per <= 32 ? 2 : 4));
        const long bm = 16 * pl.rows_mt, kb = f64 ? 8 : 16;
        const long rt = runs ? std::max<long>(1, std::min<long>(a.m, a.m / bm + a.groups)) : (m + bm - 1) / bm;
        const long wgs = rt * ((n + 63) / 64);
        long nz = std::min<long>(2 * cus / wgs, a.k / (16 * kb));
        nz = std::min<long>(nz, std::max<long>(1, (long)(0.1 * a.k / per)));
        if (a.cfg[1]) nz = a.cfg[1];
        nz = std::max<long>(1, std::min<long>(nz, 256));
        pl.kchunk = (a.k + nz - 1) / nz;
        pl.kchunk = std::max<long>((pl.kchunk + 4 * kb - 1) / (4 * kb) * (4 * kb), 4 * kb);
        pl.nz = (int)std::max<long>(1, (a.k + pl.kchunk - 1) / pl.kchunk);
        return pl;
    }
    const double cu_rate = (f64 ? 75e6 : 150e6) / cus;     // flop per us
    double best = 1e300;
    for (int tw = 4; tw >= 2; tw -= 2) {
        if (a.cfg[0] && a.cfg[0] != 32 * tw) continue;
        const long bm = 32 * tw;
        const long mt = runs ? (long)(a.groups * ((long)(avg + bm - 1) / bm)) : (a.m + bm - 1) / bm;
        const long tiles = std::max<long>(mt, 1) * ((a.n + bm - 1) / bm);
        for (long nz = 1; nz <= 32; ++nz) {
            if (a.cfg[1]) nz = a.cfg[1];
            const long chunk = ((a.k + nz - 1) / nz + bk - 1) / bk * bk;
            if (!a.cfg[1] && nz > 1 && chunk < 8 * bk) break;
            const long used = a.k > 0 ? (a.k + chunk - 1) / chunk : 1;
            const long wgs = tiles * used, load = (wgs + cus - 1) / cus;
            const double eff = tw == 4 ? (load == 1 ? 0.7 : 0.92) : (load == 1 ? 0.5 : (load == 2 ? 0.7 : 0.8));
            double t = load * 2.0 * bm * bm * chunk / (cu_rate * eff);
            if (used > 1) t += 4.0 + 2.0 * used * a.m * a.n * s / 4.5e6;
            if (t < best) {
                best = t;
                pl.tw = tw;
                pl.nz = (int)used;
                pl.kchunk = chunk;
            }
            if (a.cfg[1]) break;
        }
    }
    if (pl.tw == 0) pl.tw = 4;
    return pl;
}

long plan_bytes(const locus_hip_product_args& a, const Plan& pl)
{
    return pl.nz > 1 ? (long)pl.nz * a.m * a.n * (a.dtype == LOCUS_HIP_F64 ? 8 : 4) : 0;
}

int check_product(const locus_hip_product_args* a)
{
    LOCUS_REQUIRE(a, "product: no arguments");
    LOCUS_REQUIRE(a->dtype == LOCUS_HIP_F64 || a->dtype == LOCUS_HIP_F32, "product: dtype");
    LOCUS_REQUIRE(a->act >= LOCUS_HIP_ACT_IDENTITY && a->act <= LOCUS_HIP_ACT_SILU, "product: act");
    LOCUS_REQUIRE(a->mode >= LOCUS_HIP_PRODUCT_DENSE && a->mode <= LOCUS_HIP_PRODUCT_SUM, "product: mode");
    LOCUS_REQUIRE(a->m >= 0 && a->n >= 0 && a->k >= 0 && a->m < (1ll << 30) && a->n <= 65535 * 64 &&
                      a->k < (1ll << 30),
                  "product: sizes (m, k < 2^30, n <= 4194240)");
    LOCUS_REQUIRE(a->cfg[0] == 0 || a->cfg[0] == 64 || a->cfg[0] == 128 ||
                      (a->mode != LOCUS_HIP_PRODUCT_SUM &&
                       (a->cfg[0] == 1 || a->cfg[0] == 2 || a->cfg[0] == 4)),
                  "product: cfg[0] is 0, 1, 2, 4, 64 or 128 (64 or 128 for a sum over runs)");
    LOCUS_REQUIRE(a->cfg[1] >= 0 && a->cfg[1] <= 256 && (a->cfg[1] <= 1 || a->mode != LOCUS_HIP_PRODUCT_SUM),
                  "product: cfg[1] is 0..256 (0 or 1 for a sum over runs)");
    LOCUS_REQUIRE(a->cfg[0] == 0 || a->cfg[0] > 4 || a->mode != LOCUS_HIP_PRODUCT_DENSE ||
                      std::min(a->m, a->n) < (1ll << 20),
                  "product: the kernel for few rows takes fewer than 2^20 of them");
    if (a->mode != LOCUS_HIP_PRODUCT_DENSE) {
        LOCUS_REQUIRE(a->groups >= 1 && a->groups <= 65535, "product: groups (1..65535)");
        LOCUS_REQUIRE(!a->gather || a->a_rows >= 0, "product: a_rows");
    }
    return 0;
}

template <class T>
int run_product(const locus_hip_product_args& a, const Plan& pl, hipStream_t st)
{
    ProductDesc p = {};
    p.m = (int)a.m; p.n = (int)a.n; p.k = (int)a.k;
    p.A = a.A; p.sa_m = a.sa_m; p.sa_k = a.sa_k;
    p.B = a.B; p.sb_k = a.sb_k; p.sb_n = a.sb_n;
    ProductEpi& e = p.epi;
    e.C = a.C; e.sc_m = a.sc_m; e.sc_n = a.sc_n;
    e.bias = a.bias; e.sb_m = a.sbias_m; e.sb_n = a.sbias_n;
    e.res = a.res; e.sr_m = a.sr_m; e.sr_n = a.sr_n;
    e.pre = a.pre; e.sp_m = a.sp_m; e.sp_n = a.sp_n;
    e.alpha = a.alpha; e.beta = a.beta; e.act = a.act;
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
    const int mode = a.mode;
    if (mode != PRODUCT_DENSE) {
        p.groups = (int)a.groups;
        p.offsets = a.offsets;
        p.sb_g = a.sb_g; p.sbias_g = a.sbias_g; p.sc_g = a.sc_g;
        p.gather = a.gather;
        p.a_rows = a.a_rows;
        p.fill_rest = mode == PRODUCT_ROWS && a.fill_rest;
    }
    p.nz = pl.nz;
    p.kchunk = (int)pl.kchunk;
    if (pl.nz > 1) {
        p.part = a.workspace;
        p.part_z = (long)p.m * p.n;
        const bool mfast = mode == PRODUCT_DENSE && e.sc_n != 1 && e.sc_m == 1 && !pl.rows_mt;
        p.part_m = mfast ? 1 : p.n;
        p.part_n = mfast ? p.m : 1;
    }
    int rc = pl.rows_mt ? launch_product_rows<T>(p, mode, pl.rows_mt, st)
                        : launch_product_tile<T>(p, mode, pl.tw, st);
    if (rc) return rc;
    if (pl.nz > 1) {
        if (mode == PRODUCT_DENSE)
            hipLaunchKernelGGL((product_join_kernel<T, PRODUCT_DENSE>),
                               dim3(grid_of(((long)p.m * p.n + 255) / 256)), dim3(256), 0, st, p);
        else
            hipLaunchKernelGGL((product_join_kernel<T, PRODUCT_ROWS>),
                               dim3(grid_of(p.m), (unsigned)((p.n + 255) / 256)), dim3(256), 0, st, p);
        LOCUS_HIP_CHECK(hipGetLastError());
    }
    return 0;
}

// Parts of a run whose column sums are taken side by side: about four workgroups per CU, runs of at
// least 64 rows.
int slope_parts(const locus_hip_product_slope_args& a)
{
    const long blocks = ((a.n + 63) / 64) * std::max<long>(1, a.groups);
    const long per = a.m / std::max<long>(1, a.groups);
    const long want = std::min<long>(4L * device_cus() / std::max<long>(1, blocks), per / 32);
    return (int)std::max<long>(1, std::min<long>(want, 1024));
}

int check_slope(const locus_hip_product_slope_args* a)
{
    LOCUS_REQUIRE(a, "product_slope: no arguments");
    LOCUS_REQUIRE(a->dtype == LOCUS_HIP_F64 || a->dtype == LOCUS_HIP_F32, "product_slope: dtype");
    LOCUS_REQUIRE(a->act >= LOCUS_HIP_ACT_IDENTITY && a->act <= LOCUS_HIP_ACT_SILU, "product_slope: act");
    LOCUS_REQUIRE(a->m >= 0 && a->n >= 0 && a->m < (1ll << 30) && a->n <= 65535 * 64,
                  "product_slope: sizes (m < 2^30, n <= 4194240)");
    LOCUS_REQUIRE(a->offsets ? a->groups >= 1 && a->groups <= 65535 : a->groups == 0,
                  "product_slope: groups (1..65535 with offsets, else 0)");
    LOCUS_REQUIRE(!(a->row_sums && a->offsets), "product_slope: row sums are for one run");
    return 0;
}

template <class T>
int run_slope(const locus_hip_product_slope_args& a, hipStream_t st)
{
    const unsigned groups = (unsigned)std::max<long>(1, a.groups);
    if (a.G || a.col_sums) {
        const int parts = slope_parts(a);
        T* sums = a.col_sums ? (parts > 1 ? static_cast<T*>(a.workspace) : static_cast<T*>(a.col_sums)) : nullptr;
        hipLaunchKernelGGL(product_slope_kernel<T>, dim3((unsigned)((a.n + 63) / 64), (unsigned)parts, groups),
                           dim3(256), 0, st, a, parts, sums);
        LOCUS_HIP_CHECK(hipGetLastError());
        if (a.col_sums && parts > 1) {
            const long len = (long)groups * a.n;
            hipLaunchKernelGGL(product_sums_join_kernel<T>, dim3((unsigned)((len + 255) / 256)), dim3(256), 0, st,
                               sums, parts, len, static_cast<T*>(a.col_sums));
            LOCUS_HIP_CHECK(hipGetLastError());
        }
    }
    if (a.row_sums && a.m > 0) {
        const bool own = a.act != LOCUS_HIP_ACT_IDENTITY;
        hipLaunchKernelGGL(product_row_sums_kernel<T>, dim3(grid_of((a.m + 3) / 4)), dim3(256), 0, st,
                           static_cast<const T*>(own ? a.G : a.dC), own ? a.n : a.sd_m, own ? 1L : a.sd_n, a.m,
                           a.n, static_cast<T*>(a.row_sums));
        LOCUS_HIP_CHECK(hipGetLastError());
    }
    return 0;
}

}  // namespace
}  // namespace locus

using namespace locus;

extern "C" {

int64_t locus_hip_product_workspace_bytes(const locus_hip_product_args* args)
{
    const int rc = check_product(args);
    if (rc) return rc;
    if (args->m == 0 || args->n == 0) return 0;
    return plan_bytes(*args, plan_product(*args));
}

int locus_hip_product_dev(const locus_hip_product_args* args, void* stream)
{
    int rc = check_product(args);
    if (rc) return rc;
    const locus_hip_product_args& a = *args;
    if (a.m == 0 || a.n == 0) return 0;
    LOCUS_REQUIRE(a.C && (a.k == 0 || (a.A && a.B)), "product: null pointer");
    LOCUS_REQUIRE(a.mode == LOCUS_HIP_PRODUCT_DENSE || a.offsets, "product: runs need offsets");
    LOCUS_REQUIRE(a.pre != a.C, "product: pre and C are two buffers");
    LOCUS_REQUIRE(!a.gather || a.a_rows > 0 || a.k == 0, "product: rows gathered from an empty matrix");
    const Plan pl = plan_product(a);
    LOCUS_REQUIRE(plan_bytes(a, pl) <= (a.workspace ? a.workspace_bytes : 0),
                  "product: workspace smaller than locus_hip_product_workspace_bytes()");
    return a.dtype == LOCUS_HIP_F64 ? run_product<double>(a, pl, (hipStream_t)stream)
                                    : run_product<float>(a, pl, (hipStream_t)stream);
}

int64_t locus_hip_product_slope_workspace_bytes(const locus_hip_product_slope_args* args)
{
    const int rc = check_slope(args);
    if (rc) return rc;
    const int parts = slope_parts(*args);
    return parts > 1 ? (int64_t)parts * std::max<int64_t>(1, args->groups) * args->n *
                           (args->dtype == LOCUS_HIP_F64 ? 8 : 4)
                     : 0;
}

int locus_hip_product_slope_dev(const locus_hip_product_slope_args* args, void* stream)
{
    int rc = check_slope(args);
    if (rc) return rc;
    const locus_hip_product_slope_args& a = *args;
    if (a.n == 0) return 0;
    const bool identity = a.act == LOCUS_HIP_ACT_IDENTITY;
    LOCUS_REQUIRE(a.m == 0 || (a.dC && (identity || (a.pre && a.G))), "product_slope: null pointer");
    LOCUS_REQUIRE(!a.col_sums || locus_hip_product_slope_workspace_bytes(args) <=
                                     (a.workspace ? a.workspace_bytes : 0),
                  "product_slope: workspace smaller than locus_hip_product_slope_workspace_bytes()");
    return a.dtype == LOCUS_HIP_F64 ? run_slope<double>(a, (hipStream_t)stream)
                                    : run_slope<float>(a, (hipStream_t)stream);
}

}  // extern "C"
