// Tiled matrix product with the epilogue of ProductEpi, on the matrix cores (16 x 16 x 4 tiles of
// float64 or float32).
//
// A workgroup of four waves (2 x 2) owns a BM x BN = (32 TW) x (32 TW) tile of C, a wave TW x TW
// matrix-core tiles of it.  K-tiles of BK = 16 (float64) or 32 travel global memory -> registers -> LDS, two
// buffers, one barrier per K-tile.  The work is cut into steps of four k: a step first reads the operands
// of the next one, then moves its share of the coming K-tiles (t + 1 to LDS, t + 1 + PF from memory), then
// does its TW x TW matrix instructions, so that they wait for no read just issued.  LDS rows are 15 elements
// longer than the tile: odd, so that the transposing stores of an operand whose contiguous index is k spread
// over the banks, and small enough that tiles of 64 (40 KB) fit a CU four times, tiles of 128 (74 KB) twice.
// Those four keep its matrix cores 90 % busy (2000 x 20 000 x 500 float64; 84 % in the two products of a gradient,
// 1999 x 5000 x 1000 float32); one alone reaches 67 % of the rate.  Tiles of 128 read half as much and are chosen
// where the sums are long and the tiles fill the chip evenly.
//
// The K loop does no vector address arithmetic: an element is a raw buffer load from a scalar base
// (advanced on the scalar unit) plus a loop-invariant 32-bit lane offset, one instruction for any alignment.
// On gfx950 vector instructions take issue time from the matrix instructions of the same SIMD.  LAY_ANY is the
// same with 64-bit lane addresses, for tiles that reach over 2^31 bytes, negative strides and layouts that no
// caller of weight has.
//
// Rows and columns beyond the matrix read the tile's first one (they feed only elements that are
// never stored); only the last K-tiles check k, and steps beyond the end are skipped.
//
// Epilogue: the accumulators pass through LDS (the tile buffers are free then), all the tile's rows at a time or
// half of them, so that the element function is compiled once in a rolled loop and bias, residual, the
// kept Z and C are read and written along C's contiguous index, whichever it is.  Bound by memory where sums are
// short: 1000 x 63 x 10 000 float64 with its residual, 166 MB, takes 56 us (3.0 TB/s; it was 120 with an address
// computed for each element).
#pragma once
#include <type_traits>

#include "product.h"

namespace locus {

template <class T, int TW, int BK> struct TileGeom {
    static constexpr int BM = 32 * TW, BN = 32 * TW, LD = BM + 15;
    static constexpr int NQ = BM * BK / 256;
    static constexpr int BUF = BK * LD;                       // one operand, one buffer
    static constexpr int ELEMS = 4 * BUF;
    static_assert(ELEMS >= (BM / 2) * (BN + 1), "half a tile fits into the buffers");
};

template <class T>
__device__ __forceinline__ T buffer_elem(const char* base, unsigned off, unsigned soff)
{
    const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<char*>(base), 0, 0x7fffffff, 0x00020000 /* 32-bit data format, gfx9 */);
    if constexpr (sizeof(T) == 8)
        return __builtin_bit_cast(T, __builtin_amdgcn_raw_buffer_load_b64(r, off, soff, 0));
    else
        return __builtin_bit_cast(T, __builtin_amdgcn_raw_buffer_load_b32(r, off, soff, 0));
}

// A block of HM x BN sums in LDS (row stride EL) to where it belongs, by 256 threads: VE = 16 bytes of
// elements along C's contiguous index per thread and turn, addresses stepped, not multiplied out (a
// 64-bit product per element and matrix made short sums cost 26 us where writing C takes 8).  Partial
// products and act = identity go U turns at a time, their residuals loaded first; the other functions
// take long enough to hide one load.  PLAIN: C = alpha sum and no more (gradients: half the code).
template <class T, int HM, int BN, int EL, bool PLAIN>
__device__ __forceinline__ void store_block(const ProductDesc& p, const T* lds, bool mfast, long m0, int n0,
                                            int rows, int cols, long bias0, long c0, unsigned bz, bool gr,
                                            bool outside)
{
    constexpr int VE = 16 / (int)sizeof(T), TURNS = HM * BN / VE / 256, U = TURNS < 4 ? TURNS : 4;
    typedef T vec_t __attribute__((ext_vector_type(16 / sizeof(T)), aligned(sizeof(T))));
    const int fg = (mfast ? HM : BN) / VE, sp = 256 / fg;  // threads along the fast index, slow ones per turn
    const int f0 = (int)threadIdx.x % fg * VE, s0 = (int)threadIdx.x / fg;
    const int cnt = (mfast ? rows : cols) - f0;            // elements of this thread's group that are there
    const int sEnd = mfast ? cols : rows;
    if (cnt <= 0 || s0 >= sEnd) return;
    const bool whole = cnt >= VE;
    const ProductEpi& e = p.epi;
    const bool raw = p.part != nullptr;
    const int act = PLAIN || raw ? LOCUS_HIP_ACT_IDENTITY : e.act;
    const bool has_res = !PLAIN && !raw && e.res, has_pre = !PLAIN && !raw && e.pre, has_bias = !PLAIN && !raw && e.bias;
    const long gi = m0 + (mfast ? f0 : s0), gj = n0 + (mfast ? s0 : f0);
    auto walk = [&](const void* base, long off, long sm, long sn) {
        return static_cast<T*>(const_cast<void*>(base)) + off + gi * sm + gj * sn;
    };
    const long c_m = raw ? p.part_m : e.sc_m, c_n = raw ? p.part_n : e.sc_n;
    T* c = walk(raw ? p.part : e.C, raw ? bz * p.part_z + c0 : c0, c_m, c_n);
    const long c_f = mfast ? c_m : c_n, c_s = sp * (mfast ? c_n : c_m);
    const T* res = walk(e.res, 0, e.sr_m, e.sr_n);
    const long r_f = mfast ? e.sr_m : e.sr_n, r_s = sp * (mfast ? e.sr_n : e.sr_m);
    const T* bias = walk(e.bias, bias0, e.sb_m, e.sb_n);
    const long b_f = mfast ? e.sb_m : e.sb_n, b_s = sp * (mfast ? e.sb_n : e.sb_m);
    T* pre = walk(e.pre, 0, e.sp_m, e.sp_n);
    const long p_f = mfast ? e.sp_m : e.sp_n, p_s = sp * (mfast ? e.sp_n : e.sp_m);
    auto get = [&](const T* at, long fs, T* x) {
        if (whole && fs == 1) {
            const vec_t v = *reinterpret_cast<const vec_t*>(at);
#pragma unroll
            for (int q = 0; q < VE; ++q) x[q] = v[q];
        } else {
#pragma unroll
            for (int q = 0; q < VE; ++q) x[q] = q < cnt ? at[q * fs] : T(0);
        }
    };
    auto put = [&](T* at, long fs, const T* x) {
        if (whole && fs == 1) {
            vec_t v;
#pragma unroll
            for (int q = 0; q < VE; ++q) v[q] = x[q];
            *reinterpret_cast<vec_t*>(at) = v;
        } else {
#pragma unroll
            for (int q = 0; q < VE; ++q)
                if (q < cnt) at[q * fs] = x[q];
        }
    };
    const T* at = lds + (mfast ? f0 * EL + s0 : s0 * EL + f0);
    const int l_f = mfast ? EL : 1, l_s = mfast ? sp : sp * EL;
    auto sum = [&](int t, T* x) {
#pragma unroll
        for (int q = 0; q < VE; ++q) x[q] = outside ? T(__builtin_nan("")) : at[t * l_s + q * l_f];
        if (gr && p.k > 0) {
#pragma unroll
            for (int q = 0; q < VE; ++q)
                if (q < cnt) {
                    const long row = p.gather[gi + (mfast ? q : t * sp)];
                    if (row < 0 || row >= p.a_rows) x[q] = T(__builtin_nan(""));
                }
        }
    };
    const T alpha = raw ? T(1) : T(e.alpha), beta = T(e.beta);
    T b[VE];
#pragma unroll
    for (int q = 0; q < VE; ++q) b[q] = T(0);
    if (has_bias) get(bias, b_f, b);
    const bool bias_each = has_bias && b_s != 0;           // else: one bias for all turns
    const int turns = (sEnd - s0 + sp - 1) / sp;           // of this thread, at most TURNS
    if (act == LOCUS_HIP_ACT_IDENTITY) {
#pragma unroll 1
        for (int t0 = 0; t0 < turns; t0 += U) {
            T r[U][VE];
            if (has_res) {
#pragma unroll
                for (int u = 0; u < U; ++u)
                    if (t0 + u < turns) get(res + (t0 + u) * r_s, r_f, r[u]);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int t = t0 + u;
                if (t >= turns) break;
                T x[VE];
                sum(t, x);
                if (bias_each) get(bias + t * b_s, b_f, b);
#pragma unroll
                for (int q = 0; q < VE; ++q) x[q] = alpha * x[q] + b[q];
                if (has_pre) put(pre + t * p_s, p_f, x);
                if (has_res)
#pragma unroll
                    for (int q = 0; q < VE; ++q) x[q] += beta * r[u][q];
                put(c + t * c_s, c_f, x);
            }
        }
        return;
    }
#pragma unroll 1
    for (int t = 0; t < turns; ++t) {
        T x[VE], r[VE];
        if (has_res) get(res + t * r_s, r_f, r);
        sum(t, x);
        if (bias_each) get(bias + t * b_s, b_f, b);
#pragma unroll
        for (int q = 0; q < VE; ++q) x[q] = alpha * x[q] + b[q];
        if (has_pre) put(pre + t * p_s, p_f, x);
#pragma unroll
        for (int q = 0; q < VE; ++q) x[q] = act_value<T>(act, x[q]);
        if (has_res)
#pragma unroll
            for (int q = 0; q < VE; ++q) x[q] += beta * r[q];
        put(c + t * c_s, c_f, x);
    }
}

// How a kernel is compiled for the operands: FAST with each operand's contiguous index (k or not),
// or the general form: run-time layouts and 64-bit lane addresses.
enum { LAY_ANY = 0, LAY_FAST = 1, LAY_A_K = 2, LAY_B_K = 4, LAY_GATHER = 8 /* a fast sum's gathered A */,
       LAY_PLAIN = 16 /* with FAST: nothing but alpha in the epilogue */ };

// Workgroup `lin` of a grid of gx x gy x gz.
template <class T, int TW, int BK, int PF, int MODE, int LAY>
__device__ __forceinline__ void product_tile(const ProductDesc& p, T* lds, unsigned lin, unsigned gx,
                                             unsigned gy, unsigned gz)
{
    typedef TileGeom<T, TW, BK> G;
    typedef typename Mfma<T>::acc_t acc_t;
    constexpr int BM = G::BM, BN = G::BN, LD = G::LD, NQ = G::NQ, BUF = G::BUF;
    constexpr bool FAST = LAY & LAY_FAST, AKF = LAY & LAY_A_K, BKF = LAY & LAY_B_K;

    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int wm = wave >> 1, wn = wave & 1;

    // Which tile.  A pair of matrices: each XCD takes a contiguous eighth of the list below, in which 64
    // neighbours (what an XCD holds at once) are 8 x 8 tiles of one slice of k, so that strips of A and B are
    // read from its L2 by the others.  Sums over runs, whose lengths differ: every XCD takes an eighth of every
    // run's tiles, each eighth one in such a list (with contiguous eighths, runs that is, the XCDs were done at
    // different times: both products of ten runs' gradient, 1000 x 2000 x 500 float64, 120 us, 109 like this).
    Place at;
    Run run = {};
    if (MODE == PRODUCT_ROWS) {
        run = place_run(p.offsets, p.groups, p.m, BM, lin, gx, gy, gz, at);
    } else {
        constexpr unsigned HIGH = MODE == PRODUCT_SUM ? 64 : 8;
        const unsigned each = gx * gy;
        unsigned w = lin;
        if (MODE == PRODUCT_DENSE) {
            const XcdList list(lin, each * gz);
            w = list.start + list.at;
        }
        at.bz = w / each;
        const unsigned t = w - at.bz * each, panel = t / (HIGH * gy), r = t - panel * HIGH * gy;
        const unsigned high = gx - panel * HIGH < HIGH ? gx - panel * HIGH : HIGH;
        at.by = r / high;
        at.bx = panel * HIGH + r - at.by * high;
    }
    const unsigned bx = at.bx, by = at.by;
    unsigned bz = at.bz;
    const int n0 = by * BN, nEnd = p.n;
    long m0, mEnd;                      // rows of C
    int kb = 0, kEnd = p.k;
    const T* A = static_cast<const T*>(p.A);
    const T* B = static_cast<const T*>(p.B);
    long bias0 = 0, c0 = 0;
    if constexpr (MODE == PRODUCT_DENSE) {
        m0 = (long)bx * BM;
        mEnd = p.m;
    } else if constexpr (MODE == PRODUCT_ROWS) {
        if (run.g < 0) {
            if (p.fill_rest && bz == 0) fill_rest_rows<T>(p, run, bx, BM, n0, n0 + BN < p.n ? n0 + BN : p.n);
            return;
        }
        m0 = run.lo;
        mEnd = run.hi;
        B += run.g * p.sb_g;
        bias0 = run.g * p.sbias_g;
    } else {
        // a run's rows in nz parts of whole K-tiles
        const unsigned g = bz / (unsigned)p.nz;
        bz -= g * p.nz;
        const Run r = run_rows(p.offsets, p.k, g);
        const int len = r.hi - r.lo, chunk = (len + p.nz * BK - 1) / (p.nz * BK) * BK;
        m0 = (long)bx * BM;
        mEnd = p.m;
        kb = r.lo + (int)bz * chunk;
        kEnd = kb + chunk < r.hi ? kb + chunk : r.hi;
        c0 = g * p.sc_g;
        if (kb >= kEnd) {               // no rows: 0
            const int w = nEnd - n0 < BN ? nEnd - n0 : BN;
            T* C = static_cast<T*>(p.part ? p.part : p.epi.C) + (p.part ? bz * p.part_z : 0) + c0 + m0 * p.epi.sc_m + n0;
            const int h = (int)(mEnd - m0 < BM ? mEnd - m0 : BM);
            if (w == p.epi.sc_m) {      // whole rows: one piece of memory
                for (int e = tid; e < h * w; e += 256) C[e] = T(0);
            } else {
                for (int i = tid / BN; i < h; i += 256 / BN)
                    if (tid % BN < w) C[i * p.epi.sc_m + tid % BN] = T(0);
            }
            return;
        }
    }
    if constexpr (MODE != PRODUCT_SUM) {
        if (p.part) {
            kb = bz * p.kchunk;
            kEnd = kb + p.kchunk < p.k ? kb + p.kchunk : p.k;
        }
    }

    // Element q of a thread: k-fast operands (k contiguous) k = tid % BK, row = tid / BK + q 256 / BK;
    // else row = tid % BM, k = tid / BM + q 256 / BM (the same k for a whole wave).
    constexpr int QK = 256 / BK, QM = 256 / BM;
    constexpr int sz = (int)sizeof(T);
    const bool akf = FAST ? AKF : (p.sa_k == 1 && !(MODE == PRODUCT_SUM && p.gather));
    const bool bkf = FAST ? BKF : p.sb_k == 1;
    const int ak0 = akf ? tid % BK : __builtin_amdgcn_readfirstlane(tid / BM);
    const int bk0 = bkf ? tid % BK : __builtin_amdgcn_readfirstlane(tid / BM);
    const int mRows = (int)(mEnd - m0 < BM ? mEnd - m0 : BM), nCols = nEnd - n0 < BN ? nEnd - n0 : BN;
    T* const al = lds + (akf ? (tid % BK) * LD + tid / BK : (tid / BM) * LD + tid % BM);
    T* const bl = lds + 2 * BUF + (bkf ? (tid % BK) * LD + tid / BK : (tid / BM) * LD + tid % BM);
    const int aq = akf ? QK : QM * LD, bq = bkf ? QK : QM * LD;      // LDS step of q

    // Row of A behind row i of the tile; gathered indexes outside A count as 0 here (they never reach
    // a result: the epilogue makes it NaN).  Base: the tile's first row, gathered: A's first.
    const bool gr = MODE == PRODUCT_ROWS && p.gather;
    const bool gs = MODE == PRODUCT_SUM && (FAST ? (LAY & LAY_GATHER) != 0 : p.gather != nullptr);
    auto in_a = [&](long row) { return row >= 0 && row < p.a_rows ? row : 0; };
    auto a_row = [&](int i) -> long {
        const int c = i < mRows ? i : 0;
        return gr ? in_a(p.gather[m0 + c]) : c;
    };
    // (readfirstlane: the compiler does not see that a run's base is the same for all lanes, and would
    // ask lane by lane for each load of the K loop)
    auto base = [&](const T* at) { return reinterpret_cast<const char*>(uniform_long(reinterpret_cast<long>(at))); };
    const char* Ab = base(A + (gr ? 0 : m0 * p.sa_m) + (gs ? 0 : kb * p.sa_k));
    const char* Bb = base(B + (long)n0 * p.sb_n + kb * p.sb_k);
    const long da = (gs ? 0 : BK * p.sa_k) * sz, db = BK * p.sb_k * sz;
    // Lane offsets in bytes: one per element where k is contiguous (rows are clamped one by one), else one, and
    // the step of q on the scalar unit.
    typedef typename std::conditional<FAST, unsigned, long>::type off_t;
    constexpr int NA = FAST && !AKF ? 1 : NQ, NB = FAST && !BKF ? 1 : NQ;
    off_t oa[NA], ob[NB];
#pragma unroll
    for (int q = 0; q < NA; ++q)
        oa[q] = (off_t)((akf ? a_row(tid / BK + q * QK) * p.sa_m + ak0 * p.sa_k
                             : a_row(tid % BM) * p.sa_m + (gs ? 0 : (ak0 + q * QM) * p.sa_k)) * sz);
#pragma unroll
    for (int q = 0; q < NB; ++q) {
        const int j = bkf ? tid / BK + q * QK : tid % BM;
        ob[q] = (off_t)(((j < nCols ? j : 0) * p.sb_n + (bkf ? bk0 : bk0 + q * QM) * p.sb_k) * sz);
    }

    acc_t acc[TW][TW];
#pragma unroll
    for (int i = 0; i < TW; ++i)
#pragma unroll
        for (int j = 0; j < TW; ++j) acc[i][j] = (acc_t){0, 0, 0, 0};

    const int tiles = kEnd > kb ? (kEnd - kb + BK - 1) / BK : 0;   // K-tiles
    T ra[PF][NQ], rb[PF][NQ];           // [stage]: K-tiles on their way
    // Element q of the K-tile that starts at k0; `in`: k is not beyond the end.  An element beyond it is 0: FAST
    // asks for an offset outside the buffer resource, which the hardware answers with 0 (no branches in
    // short sums).  Gathered sums: one row of A per wave and element; lane q holds the q-th one of the
    // K-tile (rows), read a K-tile ahead.
    bool outside = false;               // a gathered row outside A: the run's C is NaN
    auto gathered = [&](int k0) -> int {
        if (MODE != PRODUCT_SUM || !gs) return 0;
        const int k = k0 + ak0 + lane % NQ * QM;
        const long row = p.gather[k < kEnd ? k : kb];
        outside |= row < 0 || row >= p.a_rows;
        return (int)in_a(row);
    };
    auto get_a = [&](int q, int rows, bool in) -> T {
        if (MODE == PRODUCT_SUM && gs) {
            const long row = (long)__builtin_amdgcn_readlane(rows, q) * p.sa_k * sz;
            if constexpr (FAST) return buffer_elem<T>(Ab, in ? oa[0] : 0x80000000u, (unsigned)row);
            else return in ? *reinterpret_cast<const T*>(Ab + row + oa[q]) : T(0);
        }
        if constexpr (FAST)
            return buffer_elem<T>(Ab, in ? oa[AKF ? q : 0] : 0x80000000u, AKF ? 0u : (unsigned)(q * QM * p.sa_k * sz));
        else
            return in ? *reinterpret_cast<const T*>(Ab + oa[q]) : T(0);
    };
    auto get_b = [&](int q, bool in) -> T {
        if constexpr (FAST)
            return buffer_elem<T>(Bb, in ? ob[BKF ? q : 0] : 0x80000000u, BKF ? 0u : (unsigned)(q * QM * p.sb_k * sz));
        else
            return in ? *reinterpret_cast<const T*>(Bb + ob[q]) : T(0);
    };
    // The K-tile whose first k is k0, elements [q0, q1) of each operand, to registers (stage st).
    auto load_part = [&](auto stc, auto wholec, int k0, int rows, int q0, int q1) {
        constexpr int st = decltype(stc)::value % PF;
        constexpr bool whole = decltype(wholec)::value;
#pragma unroll
        for (int q = q0; q < q1; ++q) {
            ra[st][q] = get_a(q, rows, whole || k0 + ak0 + (akf ? 0 : q * QM) < kEnd);
            rb[st][q] = get_b(q, whole || k0 + bk0 + (bkf ? 0 : q * QM) < kEnd);
        }
    };
    int rows = gathered(kb);            // of the K-tile to be asked for next
    auto advance = [&]() {
        Ab += da;
        Bb += db;
    };
    auto write_part = [&](auto tc, int q0, int q1) {
        constexpr int buf = decltype(tc)::value, st = buf % PF;
#pragma unroll
        for (int q = q0; q < q1; ++q) {
            al[buf * BUF + q * aq] = ra[st][q];
            bl[buf * BUF + q * bq] = rb[st][q];
        }
    };
    const T* ar = lds + (lane >> 4) * LD + wm * 16 * TW + (lane & 15);
    const T* br = lds + 2 * BUF + (lane >> 4) * LD + wn * 16 * TW + (lane & 15);
    T fa[2][TW], fb[2][TW];             // operands of this and of the next step
    auto read_step = [&](auto bufc, auto sc) {
        constexpr int buf = decltype(bufc)::value, s = decltype(sc)::value;
#pragma unroll
        for (int i = 0; i < TW; ++i) fa[s & 1][i] = ar[buf * BUF + 4 * s * LD + i * 16];
#pragma unroll
        for (int j = 0; j < TW; ++j) fb[s & 1][j] = br[buf * BUF + 4 * s * LD + j * 16];
    };
    constexpr int S = BK / 4;           // steps of a K-tile
    constexpr int MS = S / 2;           // the first MS of them move the coming K-tiles
    static_assert(S % 2 == 0 && NQ % MS == 0, "steps and elements");
    // K-tile t, its step 0 already in fa[0], fb[0].  Every step first reads the operands of the next
    // one (the last step those of the next K-tile, behind the barrier that publishes it), so that a
    // wave's matrix instructions never wait for an LDS read just issued; tile t + 1 goes to LDS and
    // tile t + 1 + PF is requested in pieces between them.  CHECK: the last tiles, which ask what is left.
    auto k_tile = [&](auto bufc, auto checkc, int t) {
        constexpr bool CHECK = decltype(checkc)::value;
        constexpr auto nextc = std::integral_constant<int, (decltype(bufc)::value ^ 1)>{};
        const bool more = !CHECK || t + 1 < tiles;
        const int kl = kb + (t + 1 + PF) * BK;
        const bool ask = !CHECK || t + 1 + PF < tiles;
        auto step = [&](auto sc) {
            constexpr int s = decltype(sc)::value;
            if constexpr (s + 1 < S) {
                read_step(bufc, std::integral_constant<int, s + 1>{});
            } else {
                __syncthreads();
                if (more) read_step(nextc, std::integral_constant<int, 0>{});
            }
            if constexpr (s < MS) {
                constexpr int q0 = s * (NQ / MS), q1 = q0 + NQ / MS;
                if (more) write_part(nextc, q0, q1);
                if (ask) {
                    load_part(nextc, std::bool_constant<!CHECK>{}, kl, rows, q0, q1);
                    if (s == MS - 1) {
                        advance();
                        rows = gathered(kl + BK);
                    }
                }
            }
            __builtin_amdgcn_sched_barrier(0);
            if (!CHECK || 4 * s < kEnd - (kb + t * BK)) {       // steps beyond the end have nothing to add
#pragma unroll
                for (int i = 0; i < TW; ++i)
#pragma unroll
                    for (int j = 0; j < TW; ++j) acc[i][j] = Mfma<T>::run(fa[s & 1][i], fb[s & 1][j], acc[i][j]);
            }
            __builtin_amdgcn_sched_barrier(0);
        };
        step(std::integral_constant<int, 0>{});
        step(std::integral_constant<int, 1>{});
        step(std::integral_constant<int, 2>{});
        step(std::integral_constant<int, 3>{});
        if constexpr (S == 8) {
            step(std::integral_constant<int, 4>{});
            step(std::integral_constant<int, 5>{});
            step(std::integral_constant<int, 6>{});
            step(std::integral_constant<int, 7>{});
        }
    };
    // The residual's lines (128 bytes) of this tile, one a thread, into L2 while the products run: 1000 x 63 x 10 000
    // float64 with inputs from memory 62.7 -> 56.1 us (with all of them in the last cache already 49 -> 54).
    T line = T(0);
    auto touch = [&]() {
        if constexpr (TW == 2 && MODE != PRODUCT_SUM && !(LAY & LAY_PLAIN)) {
            if (p.part || !p.epi.res) return;
            constexpr int LE = 128 / (int)sizeof(T);
            const bool by_column = p.epi.sr_n != 1 && p.epi.sr_m == 1;
            const int f = tid % (BM / LE) * LE, o = tid / (BM / LE), i = by_column ? f : o, j = by_column ? o : f;
            if (i < mRows && j < nCols) line = static_cast<const T*>(p.epi.res)[(m0 + i) * p.epi.sr_m + (n0 + j) * p.epi.sr_n];
        }
    };
    if (tiles > 0) {
        constexpr auto b0 = std::integral_constant<int, 0>{};
        constexpr auto b1 = std::integral_constant<int, 1>{};
        const int rows1 = gathered(kb + BK), rows2 = gathered(kb + PF * BK);
        load_part(b0, std::false_type{}, kb, rows, 0, NQ);
        advance();
        rows = gathered(kb + (PF + 1) * BK);
        if (PF == 2 && tiles > 1) {
            load_part(b1, std::false_type{}, kb + BK, rows1, 0, NQ);
            advance();
        }
        write_part(b0, 0, NQ);
        if (tiles > PF) {
            load_part(std::integral_constant<int, PF>{}, std::false_type{}, kb + PF * BK, rows2, 0, NQ);
            advance();
        }
        touch();
        __syncthreads();
        read_step(b0, b0);
        const int full = (kEnd - kb) / BK;
        int t = 0;
        for (; t + 2 + PF < full; t += 2) {
            k_tile(b0, std::false_type{}, t);
            k_tile(b1, std::false_type{}, t + 1);
        }
        for (; t < tiles; t += 2) {
            k_tile(b0, std::true_type{}, t);
            if (t + 1 < tiles) k_tile(b1, std::true_type{}, t + 1);
        }
    }

    asm volatile("" ::"v"(line));        // (or the load would go)
    if (gs) outside = __syncthreads_or(outside);

    constexpr bool PLAIN = MODE == PRODUCT_SUM || (LAY & LAY_PLAIN) != 0;
    // Through LDS, all rows at a time or half of them, then along C's contiguous index.
    constexpr int HALVES = BM * (BN + 1) <= G::ELEMS ? 1 : 2, HM = BM / HALVES, EL = BN + 1;
    const bool mfast = p.part ? p.part_m == 1 : (p.epi.sc_n != 1 && p.epi.sc_m == 1);
#pragma unroll
    for (int h = 0; h < HALVES; ++h) {
        if (HALVES == 1 || wm == h) {
            T* at = lds + (HALVES == 1 ? wm * 16 * TW * EL : 0) + wn * 16 * TW + (lane & 15);
#pragma unroll
            for (int i = 0; i < TW; ++i)
#pragma unroll
                for (int j = 0; j < TW; ++j)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        at[(i * 16 + Mfma<T>::row(lane, r)) * EL + j * 16] = acc[i][j][r];
        }
        __syncthreads();
        const int rows = (int)(mEnd - m0 - h * HM < HM ? mEnd - m0 - h * HM : HM);
        store_block<T, HM, BN, EL, PLAIN>(p, lds, mfast, m0 + h * HM, n0, rows, nCols, bias0, c0, bz, gr, outside);
        if (h + 1 < HALVES) __syncthreads();
    }
}

template <class T> constexpr int tile_bk() { return sizeof(T) == 8 ? 16 : 32; }
template <class T, int TW> constexpr int tile_elems() { return TileGeom<T, TW, tile_bk<T>()>::ELEMS; }

template <class T, int TW, int PF, int MODE, int LAY>
__global__ void __launch_bounds__(256, TW == 4 ? 2 : 4) product_tile_kernel(const ProductDesc p)
{
    __shared__ T lds[tile_elems<T, TW>()];
    product_tile<T, TW, tile_bk<T>(), PF, MODE, LAY>(
        p, lds, blockIdx.x + gridDim.x * (blockIdx.y + gridDim.y * blockIdx.z), gridDim.x, gridDim.y, gridDim.z);
}

struct TileGrid {
    unsigned x, y, z;
    __host__ __device__ unsigned all() const { return (x * y * z + 7) / 8 * 8; }    // whole turns over the XCDs
};
struct ProductPair {
    ProductDesc p, q;
    TileGrid gp, gq;
    int q_first;
};

// Two products that do not wait for each other (the two of a gradient) in one launch: the second one's
// workgroups fill the CUs that the first one's last ones leave.  The one with the longer sums is the first, so that
// short workgroups end the launch (12 runs, 3306 x 2096 x 30 float64 76 -> 54 us).
template <class T, int TW, int MODE0, int LAY0, int MODE1, int LAY1>
__global__ void __launch_bounds__(256, TW == 4 ? 2 : 4) product_pair_kernel(const ProductPair d)
{
    __shared__ T lds[tile_elems<T, TW>()];
    constexpr int PF = TW == 2 ? 2 : 1;
    const unsigned first = d.q_first ? d.gq.all() : d.gp.all();
    const bool second = blockIdx.x >= first;
    const unsigned lin = second ? blockIdx.x - first : blockIdx.x;
    if (second == (d.q_first != 0)) {
        if (lin < d.gp.x * d.gp.y * d.gp.z)
            product_tile<T, TW, tile_bk<T>(), PF, MODE0, LAY0>(d.p, lds, lin, d.gp.x, d.gp.y, d.gp.z);
    } else if (lin < d.gq.x * d.gq.y * d.gq.z) {
        product_tile<T, TW, tile_bk<T>(), PF, MODE1, LAY1>(d.q, lds, lin, d.gq.x, d.gq.y, d.gq.z);
    }
}

// The form a product takes: FAST and its layout, or LAY_ANY.  Compiled fast: every layout of one matrix pair and of
// runs of rows; sums over runs with B contiguous along a row, and a gathered A, too.
template <class T> int tile_layout(const ProductDesc& p, int mode, int tw)
{
    constexpr int BK = tile_bk<T>();
    const int bm = 32 * tw;
    // 32-bit lane offsets: a K-tile's elements lie, whole, within the 2^31 - 1 bytes of buffer_elem's window behind its
    // first one (a gathered A: all of A does); of one that ended at 2^31 the hardware would make a 0
    const long lim = ((1L << 31) - 1) / (long)sizeof(T) - 1;
    const long a_m = mode == PRODUCT_ROWS && p.gather ? p.a_rows : bm;
    const long a_k = mode == PRODUCT_SUM && p.gather ? p.a_rows : BK;
    const bool off32 = p.sa_m >= 0 && p.sa_k >= 0 && p.sb_n >= 0 && p.sb_k >= 0 &&
                       (a_m - 1) * p.sa_m + (a_k - 1) * p.sa_k <= lim &&
                       (bm - 1) * p.sb_n + (BK - 1) * p.sb_k <= lim;
    // (one column has no stride of its own: it goes with the layout of a pair and of sums over runs)
    const bool ak = p.sa_k == 1, bk = p.sb_k == 1 && !(p.n == 1 && mode != PRODUCT_ROWS && !ak);
    if (!off32 || (mode == PRODUCT_SUM && bk)) return LAY_ANY;
    if (mode == PRODUCT_SUM && p.gather) return LAY_FAST | LAY_GATHER;
    return LAY_FAST | (ak ? LAY_A_K : 0) | (bk ? LAY_B_K : 0);
}

inline TileGrid tile_grid(const ProductDesc& p, int mode, int bm)
{
    TileGrid g = {(unsigned)((p.m + bm - 1) / bm), (unsigned)((p.n + bm - 1) / bm), p.part ? (unsigned)p.nz : 1u};
    if (mode == PRODUCT_ROWS) g.x = run_tiles(p, bm);
    if (mode == PRODUCT_SUM) g.z = (unsigned)p.groups * (unsigned)p.nz;
    return g;
}

template <class T>
int launch_product_tile(const ProductDesc& p, int mode, int tw, hipStream_t st)
{
    // partial products and plain ones by kernels without the rest of the epilogue
    const bool plain = mode == PRODUCT_SUM || p.part || epi_plain(p.epi);
    const int form = tile_layout<T>(p, mode, tw), lay = form && plain ? form | LAY_PLAIN : form;
    const TileGrid g = tile_grid(p, mode, lay ? 32 * tw : 64);
    auto go = [&](auto kern) { hipLaunchKernelGGL(kern, dim3(g.x, g.y, g.z), dim3(256), 0, st, p); };
    auto pick = [&](auto twc, auto plc) {
        constexpr int TW = decltype(twc)::value, PF = TW == 2 ? 2 : 1, PL = decltype(plc)::value;
        constexpr int AK = LAY_FAST | LAY_A_K | PL, BK = LAY_FAST | LAY_B_K | PL, NONE = LAY_FAST | PL;
        if (mode == PRODUCT_DENSE) {
            if (lay == (AK | BK)) go(product_tile_kernel<T, TW, PF, PRODUCT_DENSE, AK | BK>);
            else if (lay == AK) go(product_tile_kernel<T, TW, PF, PRODUCT_DENSE, AK>);
            else if (lay == BK) go(product_tile_kernel<T, TW, PF, PRODUCT_DENSE, BK>);
            else go(product_tile_kernel<T, TW, PF, PRODUCT_DENSE, NONE>);
        } else if (mode == PRODUCT_ROWS) {
            if (lay == (AK | BK)) go(product_tile_kernel<T, TW, PF, PRODUCT_ROWS, AK | BK>);
            else if (lay == AK) go(product_tile_kernel<T, TW, PF, PRODUCT_ROWS, AK>);
            else if (lay == BK) go(product_tile_kernel<T, TW, PF, PRODUCT_ROWS, BK>);
            else go(product_tile_kernel<T, TW, PF, PRODUCT_ROWS, NONE>);
        } else if constexpr (PL != 0) {
            constexpr int AK = LAY_FAST | LAY_A_K;
            if (p.gather) go(product_tile_kernel<T, TW, PF, PRODUCT_SUM, LAY_FAST | LAY_GATHER>);
            else if (form == AK) go(product_tile_kernel<T, TW, PF, PRODUCT_SUM, AK>);
            else go(product_tile_kernel<T, TW, PF, PRODUCT_SUM, LAY_FAST>);
        }
    };
    if (lay == LAY_ANY) {                       // tiles of 64 only
        if (mode == PRODUCT_DENSE) go(product_tile_kernel<T, 2, 1, PRODUCT_DENSE, LAY_ANY>);
        else if (mode == PRODUCT_ROWS) go(product_tile_kernel<T, 2, 1, PRODUCT_ROWS, LAY_ANY>);
        else go(product_tile_kernel<T, 2, 1, PRODUCT_SUM, LAY_ANY>);
    } else {
        const auto pl = std::integral_constant<int, LAY_PLAIN>{};
        const auto full = std::integral_constant<int, 0>{};
        if (tw == 4 && plain) pick(std::integral_constant<int, 4>{}, pl);
        else if (tw == 4) pick(std::integral_constant<int, 4>{}, full);
        else if (plain) pick(std::integral_constant<int, 2>{}, pl);
        else pick(std::integral_constant<int, 2>{}, full);
    }
    LOCUS_HIP_CHECK(hipGetLastError());
    return 0;
}

// Pairs that are compiled: a gradient's two products of row-major G and B, dA = G B' and dB = A' G, with A row-major,
// column-major or gathered by rows.
template <class T>
bool product_pairs(const ProductDesc& p, int mode, int tw, const ProductDesc& q, int qmode, int qtw)
{
    constexpr int ABK = LAY_FAST | LAY_A_K | LAY_B_K;
    const TileGrid g = tile_grid(p, mode, 32 * tw), h = tile_grid(q, qmode, 32 * tw);
    const double all = (double)g.x * g.y * g.z + (double)h.x * h.y * h.z;
    return tw == qtw && all < (1 << 23) && (mode == PRODUCT_DENSE ? qmode == PRODUCT_DENSE : mode == PRODUCT_ROWS && qmode == PRODUCT_SUM) &&
           tile_layout<T>(p, mode, tw) == ABK && (tile_layout<T>(q, qmode, tw) & ~LAY_GATHER & ~LAY_A_K) == LAY_FAST;
}

template <class T>
int launch_product_pair(const ProductDesc& p, int mode, const ProductDesc& q, int tw, hipStream_t st)
{
    constexpr int ABK = LAY_FAST | LAY_A_K | LAY_B_K;
    const int qmode = mode == PRODUCT_DENSE ? PRODUCT_DENSE : PRODUCT_SUM;
    const long p_sum = p.k / p.nz, q_sum = q.k / (qmode == PRODUCT_SUM ? q.groups : 1) / q.nz;   // lengths of the sums
    const ProductPair d = {p, q, tile_grid(p, mode, 32 * tw), tile_grid(q, qmode, 32 * tw), q_sum > p_sum};
    const dim3 grid(d.gp.all() + d.gq.all());
    auto go = [&](auto kern) { hipLaunchKernelGGL(kern, grid, dim3(256), 0, st, d); };
    auto pick = [&](auto twc) {
        constexpr int TW = decltype(twc)::value;
        constexpr int PL = LAY_PLAIN, AK = LAY_FAST | LAY_A_K;
        const bool by_column = tile_layout<T>(q, qmode, tw) & LAY_A_K;
        if (mode == PRODUCT_DENSE && by_column) go(product_pair_kernel<T, TW, PRODUCT_DENSE, ABK | PL, PRODUCT_DENSE, AK | PL>);
        else if (mode == PRODUCT_DENSE) go(product_pair_kernel<T, TW, PRODUCT_DENSE, ABK | PL, PRODUCT_DENSE, LAY_FAST | PL>);
        else if (by_column) go(product_pair_kernel<T, TW, PRODUCT_ROWS, ABK | PL, PRODUCT_SUM, AK>);
        else if (q.gather) go(product_pair_kernel<T, TW, PRODUCT_ROWS, ABK | PL, PRODUCT_SUM, LAY_FAST | LAY_GATHER>);
        else go(product_pair_kernel<T, TW, PRODUCT_ROWS, ABK | PL, PRODUCT_SUM, LAY_FAST>);
    };
    if (tw == 2) pick(std::integral_constant<int, 2>{});
    else pick(std::integral_constant<int, 4>{});
    LOCUS_HIP_CHECK(hipGetLastError());
    return 0;
}

}  // namespace locus
