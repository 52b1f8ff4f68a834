// Tiled matrix product with the epilogue of ProductEpi, on the matrix cores (16 x 16 x 4 tiles of
// float64 or float32).
//
// A workgroup of four waves (2 x 2) owns a BM x BN = (32 TW) x (32 TW) tile of C, a wave TW x TW
// matrix-core tiles of it.  K-tiles of BK travel global memory -> registers -> LDS, two buffers, one
// barrier per K-tile: tile t + 1 goes to LDS and tile t + 2 is requested before the products of
// tile t.  With TW = 4 a wave does 64 matrix instructions per K-tile (4096 cycles) against 32 LDS reads
// and 16 + 16 single-element moves, and two workgroups share a CU (74 KB of LDS each), so that one's
// barrier hides behind the other's products.  LDS rows are 17 elements longer than the tile: odd, so
// that the transposing stores of an operand whose contiguous index is k spread over the banks.
//
// The K loop does no vector address arithmetic: an element is a raw buffer load from a scalar base
// (advanced on the scalar unit) plus a loop-invariant 32-bit lane offset.  On gfx950 vector
// instructions take issue time from the matrix instructions of the same SIMD.  OFF32 = false is the
// same with 64-bit lane addresses, for tiles that reach over 2^31 bytes and for gathered rows.
//
// Rows and columns beyond the matrix read the tile's first one (they feed only elements that are
// never stored); only a last, partial K-tile checks k.
//
// Epilogue: the accumulators pass through LDS (the tile buffers are free then), half the tile's rows
// at a time, so that the element function is compiled once in a rolled loop and bias, residual, the
// kept Z and C are read and written along C's contiguous index, whichever it is.
#pragma once
#include <type_traits>

#include "product.h"

namespace locus {

template <class T, int TW, int BK> struct TileGeom {
    static constexpr int BM = 32 * TW, BN = 32 * TW, LD = BM + 17;
    static constexpr int NQ = BM * BK / 256;
    static constexpr int BUF = BK * LD;                       // one operand, one buffer
    static constexpr int ELEMS = 4 * BUF;
    static_assert(ELEMS >= (BM / 2) * (BN + 1), "half a tile fits into the buffers");
};

template <class T>
__device__ __forceinline__ T buffer_elem(const char* base, unsigned off)
{
    const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<char*>(base), 0, 0x7fffffff, 0x00020000 /* 32-bit data format, gfx9 */);
    if constexpr (sizeof(T) == 8)
        return __builtin_bit_cast(T, __builtin_amdgcn_raw_buffer_load_b64(r, off, 0, 0));
    else
        return __builtin_bit_cast(T, __builtin_amdgcn_raw_buffer_load_b32(r, off, 0, 0));
}

template <class T, int TW, int BK, int MODE, bool OFF32>
__global__ void __launch_bounds__(256, TW == 4 ? 2 : 3) product_tile_kernel(const ProductDesc p)
{
    typedef TileGeom<T, TW, BK> G;
    typedef typename Mfma<T>::acc_t acc_t;
    constexpr int BM = G::BM, BN = G::BN, LD = G::LD, NQ = G::NQ, BUF = G::BUF;
    __shared__ T lds[G::ELEMS];

    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int wm = wave >> 1, wn = wave & 1;

    // which tile
    int n0 = blockIdx.y * BN, nEnd = p.n;
    long m0, mEnd;                      // rows of C
    long kb = 0, kEnd = p.k;
    const T* A = static_cast<const T*>(p.A);
    const T* B = static_cast<const T*>(p.B);
    long bias0 = 0, c0 = 0;
    int z = 0;
    if constexpr (MODE == PRODUCT_DENSE) {
        m0 = (long)blockIdx.x * BM;
        mEnd = p.m;
    } else if constexpr (MODE == PRODUCT_ROWS) {
        if (p.fill_rest && blockIdx.x == gridDim.x - 1) {
            if (blockIdx.z == 0) fill_rest_rows<T>(p, n0, n0 + BN < p.n ? n0 + BN : p.n);
            return;
        }
        const Run r = find_run(p.offsets, p.groups, p.m, blockIdx.x, BM);
        if (r.g < 0) return;
        m0 = r.lo;
        mEnd = r.hi;
        B += r.g * p.sb_g;
        bias0 = r.g * p.sbias_g;
    } else {
        const Run r = run_rows(p.offsets, p.k, blockIdx.z);
        m0 = (long)blockIdx.x * BM;
        mEnd = p.m;
        kb = r.lo;
        kEnd = r.hi;
        c0 = r.g * p.sc_g;
    }
    if constexpr (MODE != PRODUCT_SUM) {
        if (p.part) {
            z = blockIdx.z;
            kb = (long)z * p.kchunk;
            kEnd = kb + p.kchunk < p.k ? kb + p.kchunk : p.k;
        }
    }

    // element -> (row, k) follows the contiguous index of each operand; gathered k rows are taken
    // one per wave at a time (row index on the scalar unit)
    const bool gk = MODE == PRODUCT_SUM && p.gather != nullptr;
    const bool a_kfast = p.sa_k == 1 && !gk;
    const bool b_kfast = p.sb_k == 1;
    const long mRows = mEnd - m0;
    typedef typename std::conditional<OFF32, unsigned, long>::type off_t;
    off_t oa[NQ], ob[NQ];
    int ak[NQ], bk[NQ];
    T* al[NQ];
    T* bl[NQ];
    bool bad[NQ];                       // gathered rows outside A (MODE ROWS)
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
        const int e = tid + q * 256;
        int am;
        if (a_kfast) { ak[q] = e % BK; am = e / BK; } else { am = e % BM; ak[q] = e / BM; }
        al[q] = lds + ak[q] * LD + am;
        const long i = am < mRows ? am : 0;
        long row = i;
        bad[q] = false;
        if constexpr (MODE == PRODUCT_ROWS && !OFF32) {
            row = m0 + i;
            if (p.gather) {
                row = p.gather[row];
                bad[q] = row < 0 || row >= p.a_rows;
                if (bad[q]) row = 0;
            }
        }
        oa[q] = (off_t)((row * p.sa_m + (gk ? 0 : ak[q] * p.sa_k)) * (long)sizeof(T));
        int bn;
        if (b_kfast) { bk[q] = e % BK; bn = e / BK; } else { bn = e % BN; bk[q] = e / BN; }
        bl[q] = lds + 2 * BUF + bk[q] * LD + bn;
        const long j = n0 + bn < nEnd ? bn : 0;
        ob[q] = (off_t)((j * p.sb_n + bk[q] * p.sb_k) * (long)sizeof(T));
    }
    const bool rows64 = MODE == PRODUCT_ROWS && !OFF32;
    const char* Ab = reinterpret_cast<const char*>(A + (rows64 ? 0 : m0 * p.sa_m) + (gk ? 0 : kb * p.sa_k));
    const char* Bb = reinterpret_cast<const char*>(B + (long)n0 * p.sb_n + kb * p.sb_k);
    const long da = (gk ? 0 : BK * p.sa_k) * (long)sizeof(T), db = BK * p.sb_k * (long)sizeof(T);

    acc_t acc[TW][TW];
#pragma unroll
    for (int i = 0; i < TW; ++i)
#pragma unroll
        for (int j = 0; j < TW; ++j) acc[i][j] = (acc_t){0, 0, 0, 0};

    const T qnan = T(__builtin_nan(""));
    auto get = [&](const char* base, off_t off) -> T {
        if constexpr (OFF32) return buffer_elem<T>(base, off);
        else return *reinterpret_cast<const T*>(base + off);
    };
    T ra[NQ], rb[NQ];
    auto get_a = [&](int q, long k) -> T {              // k: its place in the sum (gathered sums)
        if constexpr (MODE == PRODUCT_SUM) {
            if (gk) {
                const long row = uniform_long(p.gather[uniform_long(k)]);
                if (row < 0 || row >= p.a_rows) return qnan;
                return get(Ab + row * p.sa_k * (long)sizeof(T), oa[q]);
            }
        }
        if constexpr (MODE == PRODUCT_ROWS && !OFF32) {
            if (bad[q]) return qnan;
        }
        return get(Ab, oa[q]);
    };
    auto load_tile = [&](long k0) {
        if (k0 + BK <= kEnd) {
#pragma unroll
            for (int q = 0; q < NQ; ++q) ra[q] = get_a(q, k0 + ak[q]);
#pragma unroll
            for (int q = 0; q < NQ; ++q) rb[q] = get(Bb, ob[q]);
        } else {
#pragma unroll
            for (int q = 0; q < NQ; ++q) ra[q] = k0 + ak[q] < kEnd ? get_a(q, k0 + ak[q]) : T(0);
#pragma unroll
            for (int q = 0; q < NQ; ++q) rb[q] = k0 + bk[q] < kEnd ? get(Bb, ob[q]) : T(0);
        }
        Ab += da;
        Bb += db;
    };
    const T* ar = lds + (lane >> 4) * LD + wm * 16 * TW + (lane & 15);
    const T* br = lds + 2 * BUF + (lane >> 4) * LD + wn * 16 * TW + (lane & 15);
    auto k_tile = [&](auto bufc, long k0) {
        constexpr int buf = decltype(bufc)::value;
        if (k0 + BK < kEnd) {
#pragma unroll
            for (int q = 0; q < NQ; ++q) al[q][(buf ^ 1) * BUF] = ra[q];
#pragma unroll
            for (int q = 0; q < NQ; ++q) bl[q][(buf ^ 1) * BUF] = rb[q];
        }
        if (k0 + 2 * BK < kEnd) load_tile(k0 + 2 * BK);
#pragma unroll
        for (int s = 0; s < BK / 4; ++s) {
            T a[TW], b[TW];
#pragma unroll
            for (int i = 0; i < TW; ++i) a[i] = ar[buf * BUF + 4 * s * LD + i * 16];
#pragma unroll
            for (int j = 0; j < TW; ++j) b[j] = br[buf * BUF + 4 * s * LD + j * 16];
#pragma unroll
            for (int i = 0; i < TW; ++i)
#pragma unroll
                for (int j = 0; j < TW; ++j) acc[i][j] = Mfma<T>::run(a[i], b[j], acc[i][j]);
        }
        __syncthreads();
    };
    if (kb < kEnd) {
        load_tile(kb);
#pragma unroll
        for (int q = 0; q < NQ; ++q) al[q][0] = ra[q];
#pragma unroll
        for (int q = 0; q < NQ; ++q) bl[q][0] = rb[q];
        if (kb + BK < kEnd) load_tile(kb + BK);
        __syncthreads();
        for (long k0 = kb; k0 < kEnd; k0 += 2 * BK) {
            k_tile(std::integral_constant<int, 0>{}, k0);
            if (k0 + BK < kEnd) k_tile(std::integral_constant<int, 1>{}, k0 + BK);
        }
    }

    // Through LDS, half the rows at a time.
    constexpr int HM = BM / 2, EL = BN + 1;
    const bool mfast = p.part ? p.part_m == 1 : (p.epi.sc_n != 1 && p.epi.sc_m == 1);
    ProductEpi epi = p.epi;
    epi.C = static_cast<T*>(p.epi.C) + c0;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        if (wm == h) {
#pragma unroll
            for (int i = 0; i < TW; ++i)
#pragma unroll
                for (int j = 0; j < TW; ++j)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        lds[(i * 16 + Mfma<T>::row(lane, r)) * EL + wn * 16 * TW + j * 16 +
                            (lane & 15)] = acc[i][j][r];
        }
        __syncthreads();
#pragma unroll 1
        for (int e = tid; e < HM * BN; e += 256) {
            const int i = mfast ? e % HM : e / BN, j = mfast ? e / HM : e % BN;
            const long gi = m0 + h * HM + i;
            const int gj = n0 + j;
            if (gi < mEnd && gj < nEnd) {
                const T v = lds[i * EL + j];
                if (p.part)
                    static_cast<T*>(p.part)[z * p.part_z + gi * p.part_m + gj * p.part_n] = v;
                else
                    epi_store<T>(epi, bias0, gi, gj, v);
            }
        }
        __syncthreads();
    }
}

template <class T>
int launch_product_tile(const ProductDesc& p, int mode, int tw, hipStream_t st)
{
    constexpr int BK = sizeof(T) == 8 ? 16 : 32;
    const int bm = 32 * tw;
    const long lim = ((1L << 31) - 1) / (long)sizeof(T);
    const bool off32 = p.gather == nullptr && p.sa_m >= 0 && p.sa_k >= 0 && p.sb_n >= 0 &&
                       p.sb_k >= 0 && (bm - 1) * p.sa_m + (BK - 1) * p.sa_k <= lim &&
                       (bm - 1) * p.sb_n + (BK - 1) * p.sb_k <= lim;
    const unsigned gy = (unsigned)((p.n + bm - 1) / bm);
    unsigned gx = (unsigned)((p.m + bm - 1) / bm), gz = p.part ? (unsigned)p.nz : 1u;
    // runs of rows: at most m / bm full tiles and one partial tile per run
    if (mode == PRODUCT_ROWS) gx = (unsigned)(p.m / bm + p.groups + (p.fill_rest ? 1 : 0));
    if (mode == PRODUCT_SUM) gz = (unsigned)p.groups;
    auto go = [&](auto kern) {
        hipLaunchKernelGGL(kern, dim3(gx, gy, gz), dim3(256), 0, st, p);
        return 0;
    };
    auto pick = [&](auto twc) {
        constexpr int TW = decltype(twc)::value;
        if (mode == PRODUCT_DENSE)
            return off32 ? go(product_tile_kernel<T, TW, BK, PRODUCT_DENSE, true>)
                         : go(product_tile_kernel<T, TW, BK, PRODUCT_DENSE, false>);
        if (mode == PRODUCT_ROWS)
            return off32 ? go(product_tile_kernel<T, TW, BK, PRODUCT_ROWS, true>)
                         : go(product_tile_kernel<T, TW, BK, PRODUCT_ROWS, false>);
        return off32 ? go(product_tile_kernel<T, TW, BK, PRODUCT_SUM, true>)
                     : go(product_tile_kernel<T, TW, BK, PRODUCT_SUM, false>);
    };
    const int rc = tw == 4 ? pick(std::integral_constant<int, 4>{}) : pick(std::integral_constant<int, 2>{});
    if (rc) return rc;
    LOCUS_HIP_CHECK(hipGetLastError());
    return 0;
}

}  // namespace locus
