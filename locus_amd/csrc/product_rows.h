// Matrix product of few rows (tiles of 16) with the epilogue of ProductEpi: one new sample against all
// effects, a served batch, runs of a few rows each, and whatever is small.  B is read once (per tile of rows) and
// bounds the time: one row x 20 000 x 1000 float64 28 us (160 MB, 5.6 TB/s), 70 rows in 64 runs x 2000 x 200 float32
// 22 us (102 MB, 4.7 TB/s).  The matrix cores take the products whatever the number of rows.  (Tiles of 32 and 64
// rows that load B once for all of them are no faster: 33 samples x 20 011 x 1000 float32 33 us with three tiles of
// 16, whose second and third reading of B comes from L2, 37 and 35 with the larger ones.)
//
// A workgroup of four waves owns 16 rows x 64 columns and a slice of k; its waves take a quarter
// of the slice each and are added through LDS, the slices by product_join_kernel (or, where there is
// one slice, the epilogue runs here).  Nothing of B passes through LDS: a lane loads 16 bytes at a time
// straight into operand registers, DEPTH blocks ahead (16 loads of a wave in flight; two workgroups a
// CU then hold ~64 KB of reads open, what ~5 TB/s times the latency asks for).
//
// A matrix instruction sums four k; which four does not matter as long as A and B agree.  Lane group
// g = lane >> 4 takes the V = 16 bytes / sizeof(T) consecutive k = 4 V block + V g + u, instruction u
// of the block its u-th: so A's loads are 16 bytes wide where A is contiguous in k, and
//   BK_N  (B contiguous in n): a load holds V columns of one k, a column tile is every V-th column;
//   BK_K  (B contiguous in k): a load holds the V k of one column;
//   BK_ANY: element loads, any strides.
// A load at the right edge is moved left so that it ends with the row; the lane's columns move with
// it, and columns below its first own one are another lane's to store.
#pragma once
#include <type_traits>

#include "product.h"

namespace locus {

enum { ROWS_BK_N = 0, ROWS_BK_K = 1, ROWS_BK_ANY = 2 };

template <class T> struct Vec16 {
    static constexpr int V = 16 / sizeof(T);
    // element alignment only: a row may start anywhere
    typedef T type __attribute__((ext_vector_type(16 / sizeof(T)), aligned(sizeof(T))));
};

// PLAIN: partial products, or C = alpha sum and no more.
template <class T, int BKIND, int MODE, bool PLAIN>
__global__ void __launch_bounds__(256) product_rows_kernel(const ProductDesc p)
{
    constexpr int V = Vec16<T>::V;
    typedef typename Vec16<T>::type vec_t;
    typedef typename Mfma<T>::acc_t acc_t;
    constexpr int NT = 4;                   // column tiles of 16
    constexpr int UN = NT / V;              // loads side by side over the 64 columns
    constexpr int KB = 4 * V;               // k per block
    constexpr int DEPTH = 4;                // blocks in flight
    constexpr int BM = 16;
    constexpr int EL = 65;
    __shared__ T lds[4 * 16 * EL];

    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int c = lane & 15, g = lane >> 4;
    // runs: their tiles on the grid's long axis; one matrix: its (possibly many) columns there
    const int n0 = (MODE == PRODUCT_DENSE ? blockIdx.x : blockIdx.y) * 64;
    const unsigned tile = MODE == PRODUCT_DENSE ? blockIdx.y : blockIdx.x;
    long m0, mEnd;
    const T* A = static_cast<const T*>(p.A);
    const T* B = static_cast<const T*>(p.B);
    long bias0 = 0;
    if constexpr (MODE == PRODUCT_DENSE) {
        m0 = (long)tile * BM;
        mEnd = p.m;
    } else {
        const Run r = find_run(p.offsets, p.groups, p.m, tile, BM);
        if (r.g < 0) {
            if (p.fill_rest && blockIdx.z == 0) fill_rest_rows<T>(p, r, tile, BM, n0, n0 + 64 < p.n ? n0 + 64 : p.n);
            return;
        }
        m0 = r.lo;
        mEnd = r.hi;
        B += r.g * p.sb_g;
        bias0 = r.g * p.sbias_g;
    }

    // this wave's k
    const int kz = blockIdx.z * p.kchunk;
    const int kzEnd = kz + p.kchunk < p.k ? kz + p.kchunk : p.k;
    const int per = ((kzEnd - kz + 3) / 4 + KB - 1) / KB * KB;
    const int kb = kz + wave * per;
    const int kEnd = kb + per < kzEnd ? kb + per : kzEnd;

    // lane's rows of A (beyond the last row: the last one, never stored) and columns of B
    long row = m0 + c < mEnd ? m0 + c : mEnd - 1;
    if (MODE == PRODUCT_ROWS && p.gather) {
        row = p.gather[row];
        if (row < 0 || row >= p.a_rows) row = 0;         // the epilogue makes it NaN
    }
    const T* ap = A + row * p.sa_m;
    const bool a_vec = p.sa_k == 1;
    int first[UN];                              // BK_N: first column of the lane's load
    const T* bp[BKIND == ROWS_BK_N ? UN : NT];
    if constexpr (BKIND == ROWS_BK_N) {
#pragma unroll
        for (int u = 0; u < UN; ++u) {
            const int own = n0 + 16 * V * u + V * c;
            first[u] = own + V <= p.n ? own : p.n - V;
            bp[u] = B + first[u];
        }
    } else {
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            const int col = n0 + 16 * j + c;
            bp[j] = B + (long)(col < p.n ? col : p.n - 1) * p.sb_n;
        }
    }

    acc_t acc[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[j] = (acc_t){0, 0, 0, 0};

    T a[DEPTH][V], b[DEPTH][NT][V];             // b[..][j][u]: column tile j, instruction u
    auto load = [&](int s, int k0) {            // a whole block
        const int k = k0 + V * g;
        if constexpr (BKIND == ROWS_BK_N) {
#pragma unroll
            for (int u = 0; u < V; ++u)
#pragma unroll
                for (int w = 0; w < UN; ++w) {
                    const vec_t x = *reinterpret_cast<const vec_t*>(bp[w] + (long)(k + u) * p.sb_k);
#pragma unroll
                    for (int j = 0; j < V; ++j) b[s][w * V + j][u] = x[j];
                }
        } else if constexpr (BKIND == ROWS_BK_K) {
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                const vec_t x = *reinterpret_cast<const vec_t*>(bp[j] + k);
#pragma unroll
                for (int u = 0; u < V; ++u) b[s][j][u] = x[u];
            }
        } else {
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int u = 0; u < V; ++u) b[s][j][u] = bp[j][(long)(k + u) * p.sb_k];
        }
        if (a_vec) {
            const vec_t x = *reinterpret_cast<const vec_t*>(ap + k);
#pragma unroll
            for (int u = 0; u < V; ++u) a[s][u] = x[u];
        } else {
#pragma unroll
            for (int u = 0; u < V; ++u) a[s][u] = ap[(long)(k + u) * p.sa_k];
        }
    };
    auto load_part = [&](int s, int k0) {       // the last, partial block: k beyond the end are 0
#pragma unroll
        for (int u = 0; u < V; ++u) {
            const int k = k0 + V * g + u;
            const bool in = k < kEnd;
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                T x = T(0);
                if (in) {
                    if constexpr (BKIND == ROWS_BK_N) x = bp[j / V][(long)k * p.sb_k + j % V];
                    else x = bp[j][(long)k * p.sb_k];
                }
                b[s][j][u] = x;
            }
            a[s][u] = in ? ap[(long)k * p.sa_k] : T(0);
        }
    };
    auto use = [&](int s) {
#pragma unroll
        for (int u = 0; u < V; ++u)
#pragma unroll
            for (int j = 0; j < NT; ++j) acc[j] = Mfma<T>::run(a[s][u], b[s][j][u], acc[j]);
    };
    const int blocks = kb < kEnd ? (kEnd - kb) / KB : 0;    // whole ones
#pragma unroll
    for (int s = 0; s < DEPTH; ++s)
        if (s < blocks) load(s, kb + s * KB);
    // Bias and residual of this thread's four elements are asked for before the products, not after them
    // (1008 x 99 x 23 float32 6.5 -> 5.8 us).
    constexpr int OWN = 16 * 64 / 256;
    T eb[OWN], er[OWN];
    if (!PLAIN) {
#pragma unroll
        for (int q = 0; q < OWN; ++q) {
            const long gi = m0 + wave + 4 * q;
            const int gj = n0 + lane;
            const bool in = gi < mEnd && gj < p.n;
            eb[q] = in && p.epi.bias ? static_cast<const T*>(p.epi.bias)[bias0 + gi * p.epi.sb_m + gj * p.epi.sb_n] : T(0);
            er[q] = in && p.epi.res ? static_cast<const T*>(p.epi.res)[gi * p.epi.sr_m + gj * p.epi.sr_n] : T(0);
        }
    }
    if (kb < kEnd) {
        int i = 0;
        for (; i + 2 * DEPTH <= blocks; i += DEPTH) {
#pragma unroll
            for (int s = 0; s < DEPTH; ++s) {
                use(s);
                load(s, kb + (i + DEPTH + s) * KB);
            }
        }
        // at most 2 DEPTH - 1 blocks left, the first DEPTH of them loaded
#pragma unroll
        for (int s = 0; s < DEPTH; ++s) {
            if (i + s < blocks) {
                use(s);
                if (i + DEPTH + s < blocks) load(s, kb + (i + DEPTH + s) * KB);
            }
        }
#pragma unroll
        for (int s = 0; s < DEPTH; ++s)
            if (i + DEPTH + s < blocks) use(s);
        if (kb + blocks * KB < kEnd) {
            load_part(0, kb + blocks * KB);
            use(0);
        }
    }

    // the four waves' sums
    constexpr int WS = 16 * EL;
#pragma unroll
    for (int j = 0; j < NT; ++j) {
        int col;                                         // in the tile
        bool own = true;
        if constexpr (BKIND == ROWS_BK_N) {
            col = first[j / V] + j % V - n0;
            own = col >= 16 * V * (j / V) + V * c;
        } else {
            col = 16 * j + c;
        }
        if (own)
#pragma unroll
            for (int r = 0; r < 4; ++r) lds[wave * WS + Mfma<T>::row(lane, r) * EL + col] = acc[j][r];
    }
    __syncthreads();
#pragma unroll 1
    for (int q = 0; q < OWN; ++q) {
        const int i = wave + 4 * q, j = lane;
        const long gi = m0 + i;
        const int gj = n0 + j;
        if (gi < mEnd && gj < p.n) {
            const T* x = lds + i * EL + j;
            T v = (x[0] + x[WS]) + (x[2 * WS] + x[3 * WS]);
            if (MODE == PRODUCT_ROWS && p.gather && p.k > 0) {
                const long at = p.gather[gi];
                if (at < 0 || at >= p.a_rows) v = T(__builtin_nan(""));
            }
            T* const c = static_cast<T*>(p.epi.C) + gi * p.epi.sc_m + gj * p.epi.sc_n;
            if (p.part) {
                static_cast<T*>(p.part)[blockIdx.z * p.part_z + gi * p.part_m + gj * p.part_n] = v;
            } else if (PLAIN) {
                *c = T(p.epi.alpha) * v;
            } else {
                const T z = T(p.epi.alpha) * v + eb[0];
                if (p.epi.pre) static_cast<T*>(p.epi.pre)[gi * p.epi.sp_m + gj * p.epi.sp_n] = z;
                const T y = act_value<T>(p.epi.act, z);
                *c = p.epi.res ? y + T(p.epi.beta) * er[0] : y;
            }
        }
        if (!PLAIN) {                                    // (the next ones: an index would take memory)
#pragma unroll
            for (int u = 0; u + 1 < OWN; ++u) {
                eb[u] = eb[u + 1];
                er[u] = er[u + 1];
            }
        }
    }
}

template <class T>
int launch_product_rows(const ProductDesc& p, int mode, hipStream_t st)
{
    constexpr int V = Vec16<T>::V;
    const unsigned gx = (unsigned)((p.n + 63) / 64);
    const unsigned gy = mode == PRODUCT_DENSE ? (unsigned)((p.m + 15) / 16)
                                              : run_tiles(p, 16);
    const int kind = p.sb_n == 1 && p.n >= V ? ROWS_BK_N : (p.sb_k == 1 ? ROWS_BK_K : ROWS_BK_ANY);
    const bool dense = mode == PRODUCT_DENSE;
    const bool plain = p.part || epi_plain(p.epi);
    const dim3 grid(dense ? gx : gy, dense ? gy : gx, (unsigned)p.nz);
    auto go = [&](auto kern) { hipLaunchKernelGGL(kern, grid, dim3(256), 0, st, p); };
    auto pick = [&](auto kc) {
        constexpr int KIND = decltype(kc)::value;
        if (dense && plain) go(product_rows_kernel<T, KIND, PRODUCT_DENSE, true>);
        else if (dense) go(product_rows_kernel<T, KIND, PRODUCT_DENSE, false>);
        else if (plain) go(product_rows_kernel<T, KIND, PRODUCT_ROWS, true>);
        else go(product_rows_kernel<T, KIND, PRODUCT_ROWS, false>);
    };
    if (kind == ROWS_BK_N) pick(std::integral_constant<int, ROWS_BK_N>{});
    else if (kind == ROWS_BK_K) pick(std::integral_constant<int, ROWS_BK_K>{});
    else pick(std::integral_constant<int, ROWS_BK_ANY>{});
    LOCUS_HIP_CHECK(hipGetLastError());
    return 0;
}

}  // namespace locus
