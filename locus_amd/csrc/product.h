// Fused matrix products and ragged grouped products (float64, float32): what the kernels share.
//
//   Z = alpha A B + bias,   C = act(Z) + beta residual
//
// product_tile.h holds the tiled kernel, product_rows.h the one for few rows, product.hip the
// element-wise kernels, the choice between them and the C entry points.
#pragma once
#include "common.h"
#include "fastmath.h"

namespace locus {

// What one element of the result goes through once its sum is there.  Strides in elements; a
// stride of 0 broadcasts.
struct ProductEpi {
    void* C; long sc_m, sc_n;
    const void* bias; long sb_m, sb_n;
    const void* res; long sr_m, sr_n;
    void* pre; long sp_m, sp_n;
    double alpha, beta;
    int act;
};

// C = alpha sum and no more.
inline bool epi_plain(const ProductEpi& e) { return !e.bias && !e.res && !e.pre && e.act == LOCUS_HIP_ACT_IDENTITY; }

// Modes of a product: one pair of matrices; runs of rows with a B of their own; runs of the summed
// index with a C of their own (the gradient of the runs' B).
enum { PRODUCT_DENSE = 0, PRODUCT_ROWS = 1, PRODUCT_SUM = 2 };

struct ProductDesc {
    int m, n, k;                      // DENSE, ROWS: m = all rows; SUM: k = all rows
    const void* A; long sa_m, sa_k;
    const void* B; long sb_k, sb_n;
    ProductEpi epi;
    // runs: offsets[groups + 1] on the device, read as the largest of 0 and every earlier one and at
    // most the number of rows, so that runs never overlap whatever the array holds
    int groups;
    const int64_t* offsets;
    long sb_g, sbias_g, sc_g;         // B, bias (ROWS) and C (SUM) of the next run
    const int64_t* gather;            // row r reads A's row gather[r]; outside [0, a_rows): NaN
    long a_rows;
    int fill_rest;                    // ROWS: rows of no run become 0 in C and pre
    // a split sum: part [z][rows][n] (or [z][n][rows], following C) instead of C
    void* part;
    int nz, kchunk;
    long part_m, part_n, part_z;      // strides of the partial products, in elements
};

// ---- element functions -----------------------------------------------------------------------
// float64 goes through the branch-free helpers of fastmath.h: library exp, division and erfc (whose
// ranges all run where lanes differ) made the epilogue of 10 million probabilities cost 39 us.
// e = exp(-|z|) <= 1 carries both tails of the logistic function without overflow.
__device__ __forceinline__ double exp_of_minus(double x) { return exp_nonpos(-x); }      // x >= 0
__device__ __forceinline__ float exp_of_minus(float x) { return expf(-x); }
__device__ __forceinline__ double log_1_plus(double x) { return log1p(x); }
__device__ __forceinline__ float log_1_plus(float x) { return log1pf(x); }
__device__ __forceinline__ double part_of(double num, double den) { return div_1to2(num, den); }  // in [0, 1] / [1, 2]
__device__ __forceinline__ float part_of(float num, float den) { return num / den; }

template <class T> __device__ __forceinline__ T magnitude(T z) { return z < T(0) ? -z : z; }

template <class T> __device__ __forceinline__ T logistic(T z)
{
    const T e = exp_of_minus(magnitude(z));
    return part_of(z < T(0) ? e : T(1), T(1) + e);
}

// Phi(z).  The tail at a = |z| is exp(-a^2 / 2) erfcx(x) / 2 with x = a / sqrt 2, and (1 + 2 x) erfcx(x) is a
// polynomial in t = (x - 3.75) / (x + 3.75) (Shepherd and Laframboise, Math. Comp. 36, 1981): degree 23
// truncates at 5.1e-17; its coefficients were computed with 60 digits (scripts/microbench/cdf_poly.py).  a^2 / 2 is
// carried with its rounding error.  At most 8 units of rounding relative from -37.5 up; below, where results are no
// longer normal numbers, within one of the smallest positive number more; 0 from -38.6 down.
static __device__ const double kCdfPoly[24] = {
    0x1.3ccda0b5d5dc2p+0, -0x1.1f367683f89a5p-3, 0x1.d5f294816277ep-9, 0x1.510169d09665bp-4,
    -0x1.bda9309a35871p-4, 0x1.7a14188a9ce2ap-4, -0x1.e0d0fa6c16f3fp-5, 0x1.d0b0037d167adp-6,
    -0x1.3f603c7e65d24p-7, 0x1.cc3a0e7d2150cp-10, 0x1.33fb5a5e7ca14p-12, -0x1.303fa4966bc38p-12,
    0x1.b13e13fe20445p-15, 0x1.778b933adcce7p-16, -0x1.7fcc159f9a760p-17, -0x1.055686d42aa63p-20,
    0x1.d39c1a3875509p-20, -0x1.eb803840c0574p-25, -0x1.0ae6bf9452a1fp-22, 0x1.8fa9fe49c359bp-26,
    0x1.12b326b5668bfp-25, -0x1.014cd7201b5adp-28, -0x1.6884628ace07ap-29, 0x1.561b105822235p-32,
};
__device__ __forceinline__ double normal_cdf(double z)
{
    double a = magnitude(z);
    a = a > 40.0 ? 40.0 : a;                                  // a select: NaN stays
    const double x = a * 0.70710678118654752440, u = fma(2.0, x, 1.0), w = x + 3.75;
    const double r = rcp_pos_normal(u * w);
    const double t = (x - 3.75) * u * r, t2 = t * t, t4 = t2 * t2;
    double P = 0.0;
#pragma unroll
    for (int i = 20; i >= 0; i -= 4)
        P = fma(P, t4, fma(fma(kCdfPoly[i + 3], t, kCdfPoly[i + 2]), t2, fma(kCdfPoly[i + 1], t, kCdfPoly[i])));
    const double h = 0.5 * a, s = h * a, lost = fma(h, a, -s), e = exp_nonpos(-s);
    const double tail = 0.5 * P * (w * r) * fma(-lost, e, e);
    return z < 0.0 ? tail : 1.0 - tail;
}
// float32: the library's erfc.  Rounding its argument x alone cost up to 185 units in the left tail (2.9 like this), so what
// that lost comes back to first order: erfc(x + d) = erfc(x) (1 - d g(x)), g = 2 / (sqrt pi erfcx(x)) between
// x + sqrt(x^2 + 4 / pi) and x + sqrt(x^2 + 2), which differ by 0.4 units of rounding at most here.
__device__ __forceinline__ float normal_cdf(float z)
{
    constexpr double half = 0.70710678118654752440;
    constexpr float c = (float)half, c_lost = (float)(half - (double)c);
    const float a = z < -40.0f ? 40.0f : -z;                  // a select: NaN stays
    const float x = a * c, v = 0.5f * erfcf(x);
    const float d = fmaf(a, c, -x) + a * c_lost, g = x + __builtin_amdgcn_sqrtf(fmaf(x, x, 2.0f));
    return z < 0.0f ? fmaf(-d * g, v, v) : v;
}

// The rounding of z^2 / 2, which cost up to 511 (float32: 62) units of the density in its tails, is carried as in normal_cdf.
template <class T> __device__ __forceinline__ T normal_density(T z)
{
    T a = magnitude(z);
    a = a > T(40) ? T(40) : a;                                // a select: NaN stays
    const T h = T(0.5) * a, s = h * a, lost = fma(h, a, -s), e = exp_of_minus(s);
    return fma(-lost, e, e) * T(0.39894228040143267794);
}
// z * f where f -> 0 faster than z grows: 0 instead of inf * 0
template <class T> __device__ __forceinline__ T times_vanishing(T z, T f)
{
    return f == T(0) ? T(0) : z * f;
}

template <class T> __device__ __forceinline__ T act_value(int act, T z)
{
    switch (act) {
    case LOCUS_HIP_ACT_LOGISTIC: return logistic(z);
    case LOCUS_HIP_ACT_PROBIT: return normal_cdf(z);
    case LOCUS_HIP_ACT_SOFTPLUS:
        return (z > T(0) ? z : T(0)) + log_1_plus(exp_of_minus(magnitude(z)));
    case LOCUS_HIP_ACT_GELU: return times_vanishing(z, normal_cdf(z));
    case LOCUS_HIP_ACT_SILU: return times_vanishing(z, logistic(z));
    default: return z;
    }
}

template <class T> __device__ __forceinline__ T act_slope(int act, T z)
{
    switch (act) {
    case LOCUS_HIP_ACT_LOGISTIC: {
        const T e = exp_of_minus(magnitude(z)), r = part_of(T(1), T(1) + e);
        return e * r * r;
    }
    case LOCUS_HIP_ACT_PROBIT: return normal_density(z);
    case LOCUS_HIP_ACT_SOFTPLUS: return logistic(z);
    case LOCUS_HIP_ACT_GELU: return normal_cdf(z) + times_vanishing(z, normal_density(z));
    case LOCUS_HIP_ACT_SILU: {
        const T s = logistic(z);
        return s + times_vanishing(z, s * logistic(-z));
    }
    default: return T(1);
    }
}

// One element of the result: `sum` is the product's, i / j its row and column, bias0 an offset of
// the run's bias.  Reads the residual before it writes C, so that C may be the residual.
template <class T>
__device__ __forceinline__ void epi_store(const ProductEpi& e, long bias0, long i, long j, T sum)
{
    T z = T(e.alpha) * sum;
    if (e.bias) z += static_cast<const T*>(e.bias)[bias0 + i * e.sb_m + j * e.sb_n];
    if (e.pre) static_cast<T*>(e.pre)[i * e.sp_m + j * e.sp_n] = z;
    T v = act_value<T>(e.act, z);
    if (e.res) v += T(e.beta) * static_cast<const T*>(e.res)[i * e.sr_m + j * e.sr_n];
    static_cast<T*>(e.C)[i * e.sc_m + j * e.sc_n] = v;
}

// ---- runs --------------------------------------------------------------------------------------
struct Run {
    int g;            // which run (-1: none)
    int lo, hi;       // its rows (of the tile asked for)
};

__device__ __forceinline__ long uniform_long(long v)
{
    const int lo = __builtin_amdgcn_readfirstlane((int)(v & 0xffffffff));
    const int hi = __builtin_amdgcn_readfirstlane((int)(v >> 32));
    return ((long)hi << 32) | (unsigned)lo;
}

__device__ __forceinline__ int bounded(int64_t v, int rows) { return v < 0 ? 0 : (v > rows ? rows : (int)v); }

// 64 runs at a time, one per lane: the ordered offsets are a running maximum, the tiles of `bm` rows before
// a run a running sum.  Every wave does this for itself (no barrier); under 1 us for up to 64 runs, against
// a launch of its own for a tile map.
struct RunScan {
    const int64_t* offsets;
    int groups, rows, bm;
    int carry, before;       // the end of the runs so far, their tiles
    int lo, hi, excl, tiles; // this lane's run: its rows, the tiles before it, its own

    __device__ __forceinline__ RunScan(const int64_t* o, int g, int r, int b)
        : offsets(o), groups(g), rows(r), bm(b), carry(bounded(o[0], r)), before(0) {}
    __device__ __forceinline__ void next(int base)
    {
        const int lane = threadIdx.x & 63, g = base + lane;
        hi = g < groups ? bounded(offsets[g + 1], rows) : 0;
        hi = hi > carry ? hi : carry;
#pragma unroll
        for (int s = 1; s < 64; s <<= 1) {
            const int o = __shfl_up(hi, s);
            if (lane >= s && o > hi) hi = o;
        }
        const int up = __shfl_up(hi, 1);
        lo = lane == 0 ? carry : up;
        tiles = (hi - lo + bm - 1) / bm;
        int incl = tiles;
#pragma unroll
        for (int s = 1; s < 64; s <<= 1) {
            const int o = __shfl_up(incl, s);
            if (lane >= s) incl += o;
        }
        excl = before + incl - tiles;
        before += __builtin_amdgcn_readlane(incl, 63);
        carry = __builtin_amdgcn_readlane(hi, 63);
    }
    // the rows of `tile` if one of the lanes' runs holds it, else g = -1
    __device__ __forceinline__ Run pick(int base, int tile) const
    {
        const unsigned long long hit = __ballot(tile >= excl && tile < excl + tiles);
        if (hit == 0) return {-1, 0, 0};
        const int src = __ffsll((long long)hit) - 1;
        const int t0 = __builtin_amdgcn_readlane(lo, src) + (tile - __builtin_amdgcn_readlane(excl, src)) * bm;
        const int end = __builtin_amdgcn_readlane(hi, src);
        return {base + src, t0, end - t0 > bm ? t0 + bm : end};
    }
};

// The run and rows of `tile`, counted over all runs in order.  Where no run holds it: lo = the tiles there
// are, hi = the end of the last run.
__device__ __forceinline__ Run find_run(const int64_t* offsets, int groups, int rows, int tile, int bm)
{
    RunScan scan(offsets, groups, rows, bm);
    for (int base = 0; base < groups; base += 64) {
        scan.next(base);
        const Run r = scan.pick(base, tile);
        if (r.g >= 0) return r;
    }
    return {-1, scan.before, scan.carry};
}

// A workgroup's place: tile (bx, by) of slice bz.
struct Place {
    unsigned bx, by, bz;
};

// Workgroup `lin` of a grid of gx x gy x gz: its place in a list that is cut into a contiguous eighth per
// XCD (workgroups go to the XCDs in turn by their number).
struct XcdList {
    unsigned start, share, at;    // this XCD's part, the workgroup's number in it
    __device__ __forceinline__ XcdList(unsigned lin, unsigned total)
    {
        const unsigned xcd = lin & 7, rem = total & 7;
        start = xcd * (total >> 3) + (xcd < rem ? xcd : rem);
        share = (total >> 3) + (xcd < rem ? 1 : 0);
        at = lin >> 3;
    }
};

// The run, rows and place of workgroup `lin`, columns of tiles one after the other.  The grid has room for more
// tiles than runs of these lengths fill; up to 256 runs the workgroups without one come last in every
// XCD's list: where they lay between the others, the CUs that took them stayed behind (10 runs, 1000 x 5000 x 501
// float64 in four slices 165 us, 133 like this).  With more runs that count would cost longer than it saves.
__device__ __forceinline__ Run place_run(const int64_t* offsets, int groups, int rows, int bm, unsigned lin,
                                         unsigned gx, unsigned gy, unsigned gz, Place& at)
{
    const XcdList all(lin, gx * gy * gz);
    if (groups > 256) {
        const unsigned w = all.start + all.at, t = w % (gx * gy);
        at = {t % gx, t / gx, w / (gx * gy)};
        return find_run(offsets, groups, rows, at.bx, bm);
    }
    RunScan scan(offsets, groups, rows, bm);
    for (int base = 0; base < groups; base += 64) scan.next(base);
    const unsigned nx = scan.before;                   // tiles there are
    const XcdList list(lin, nx * gy * gz);
    if (list.at >= list.share) {
        const unsigned q = all.start - list.start + list.at - list.share, rest = gx - nx;
        at = {nx + q % rest, q / rest % gy, q / rest / gy};
        return {-1, (int)nx, scan.carry};
    }
    const unsigned w = list.start + list.at, t = w % (nx * gy);
    at = {t % nx, t / nx, w / (nx * gy)};
    if (groups <= 64) return scan.pick(0, at.bx);
    return find_run(offsets, groups, rows, at.bx, bm);
}

// Rows [lo, hi) of one run by its number (the same ordered offsets).
__device__ __forceinline__ Run run_rows(const int64_t* offsets, int rows, int g)
{
    const int lane = threadIdx.x & 63;
    const int64_t last = offsets[g + 1];
    int top = 0;                                       // largest of offsets[0 .. g]
    for (int i = lane; i <= g; i += 64) {
        const int v = bounded(offsets[i], rows);
        top = v > top ? v : top;
    }
#pragma unroll
    for (int s = 32; s > 0; s >>= 1) {
        const int o = __shfl_xor(top, s);
        top = o > top ? o : top;
    }
    const int hi = bounded(last, rows);
    Run r = {g, __builtin_amdgcn_readfirstlane(top), 0};
    r.hi = __builtin_amdgcn_readfirstlane(hi > top ? hi : top);
    return r;
}

// The run of each lane's own row (-1: none): the same scan, then every run of the 64 offered to all lanes.
__device__ __forceinline__ int find_runs(const int64_t* offsets, int groups, int rows, int row)
{
    const int lane = threadIdx.x & 63;
    int carry = bounded(offsets[0], rows), found = -1;
    for (int base = 0; base < groups; base += 64) {
        const int g = base + lane;
        int hi = g < groups ? bounded(offsets[g + 1], rows) : 0;
        hi = hi > carry ? hi : carry;
#pragma unroll
        for (int s = 1; s < 64; s <<= 1) {
            const int o = __shfl_up(hi, s);
            if (lane >= s && o > hi) hi = o;
        }
        const int here = groups - base < 64 ? groups - base : 64;
        int lo = carry;
        for (int s = 0; s < here; ++s) {
            const int top = __builtin_amdgcn_readlane(hi, s);
            if (row >= lo && row < top) found = base + s;
            lo = top;
        }
        carry = lo;
        if (__ballot(row >= carry) == 0) break;
    }
    return found;
}

// Tiles of bm rows that runs can have at most: full ones and one partial tile per run, none without a row;
// and one more, so that the tiles behind the last one cover the rows of no run (fill_rest_rows).
inline unsigned run_tiles(const ProductDesc& p, int bm)
{
    const long most = (long)p.m / bm + p.groups;
    return (unsigned)((most < p.m ? most : p.m) + (p.fill_rest ? 1 : 0));
}

// Rows of no run become 0: the workgroup behind the last tile takes the first bm of them, and so on.  There
// are enough of those: the grid has min(m / bm + groups, m) + 1 tiles, runs over all but R rows fill at
// most (m - R) / bm + groups and at most m - R of them.  r: what find_run said of the tile.
template <class T>
__device__ __forceinline__ void fill_rest_rows(const ProductDesc& p, const Run& r, int tile, int bm, int n0, int n1)
{
    const int head = bounded(p.offsets[0], p.m), rest = head + (p.m - r.hi), w = n1 - n0;
    const int q0 = (tile - r.lo) * bm, q1 = q0 + bm < rest ? q0 + bm : rest;
    for (int e = threadIdx.x; e < (q1 - q0) * w; e += blockDim.x) {
        const int q = q0 + e / w;
        const long j = n0 + e % w, i = q < head ? q : r.hi + (q - head);
        static_cast<T*>(p.epi.C)[i * p.epi.sc_m + j * p.epi.sc_n] = T(0);
        if (p.epi.pre) static_cast<T*>(p.epi.pre)[i * p.epi.sp_m + j * p.epi.sp_n] = T(0);
    }
}

template <class T> struct Mfma;
template <> struct Mfma<double> {
    typedef double acc_t __attribute__((ext_vector_type(4)));
    static __device__ __forceinline__ acc_t run(double a, double b, acc_t c)
    {
        return __builtin_amdgcn_mfma_f64_16x16x4f64(a, b, c, 0, 0, 0);
    }
    // row of register r in a lane (column = lane & 15)
    static __device__ __forceinline__ int row(int lane, int r) { return (lane >> 4) + 4 * r; }
};
template <> struct Mfma<float> {
    typedef float acc_t __attribute__((ext_vector_type(4)));
    static __device__ __forceinline__ acc_t run(float a, float b, acc_t c)
    {
        return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
    }
    static __device__ __forceinline__ int row(int lane, int r) { return 4 * (lane >> 4) + r; }
};

// Launchers, one translation unit per type (product_f64.hip, product_f32.hip).  tw: 4 = tiles of
// 128 x 128, 2 = 64 x 64.  A pair is two independent products in one launch; false: not this pair.
template <class T> int launch_product_tile(const ProductDesc& p, int mode, int tw, hipStream_t st);
template <class T> int launch_product_rows(const ProductDesc& p, int mode, hipStream_t st);
template <class T>
bool product_pairs(const ProductDesc& p, int mode, int tw, const ProductDesc& q, int qmode, int qtw);
template <class T>
int launch_product_pair(const ProductDesc& p, int mode, const ProductDesc& q, int tw, hipStream_t st);

}  // namespace locus
