// Orthogonalised matrix updates (gfx950): the Newton-Schulz iteration and the momentum step that uses it (Muon).
//
//   X0 = U / (|U|_F + eps), transposed so that it has m <= n;      five times:  S = X X^T,  P = b S + c S S,  X <- a X + P X
//   momentum step:  M <- mu M + g;  U = g + mu M (nesterov) or M;  p <- p (1 - lr wd) - lr s X
//
// (a, b, c) = (3.4445, -4.7750, 2.0315): every singular value s in (0, 1] runs through s <- a s + b s^3 + c s^5 and lands near 1.
//
// Bound by the matrix pipe: m^2 n + m^3 + 2 m^2 n flops per iteration (S and S S are symmetric: only the tiles on and below the diagonal
// are computed and stored twice).  X X^T and S S take both operands row by row; P X takes X along its rows, turned by the transposing LDS read.
//
// Precision.  The iteration multiplies a small singular value -- and every rounding error next to it -- by a^5 = 485, so 8 bits (bf16
// storage) leave 1e-2 of error in the result and 11 bits (half) 1e-3, 1e-2 where a few directions dominate the matrix.  Numbers are
// therefore kept as a PAIR of halves, value + rest (22 bits; scaled by 2^13, so that neither leaves half's range: |X| <= 1.2, |S| <=
// 1.5, |P + a| <= 3.5), and a product is value value + value rest + rest value with fp32 sums: the result agrees with fp32 arithmetic to its
// own rounding (2.1e-6 of error against 3.1e-6 of the fp32 form on a 1024^2 Gaussian), and a 16-bit result is off by its one rounding.  Values alone in
// the last two iterations would save a seventh of the time (16 x [1280, 1280]: 1859 against 2159 us) and leave 1e-3 of error, as much again as
// the rounding to bf16 and far more than an fp32 parameter's: not taken for any type.
// (Taking the polynomials of S = X X^T alone and multiplying X0 once saves half the products of a wide matrix, but S holds squared singular
// values: on the gradients of a small ControlNet, which a few directions dominate, the result was 1e-3 to 1e-2 off where this form is 3e-5.)
// Pairs are stored as 128-byte blocks, 32 values then their 32 rests: a K step loads whole lines.
#include <algorithm>
#include <new>
#include <vector>

#include "dm_common.h"
#include "dm_elem.h"

namespace {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

[[maybe_unused]] constexpr float kA = 3.4445f, kB = -4.7750f, kC = 2.0315f;
[[maybe_unused]] constexpr float kScale = 8192.f, kInv = 1.f / 8192.f;        // 2^13, see above
constexpr int kGroup = 16;                                   // matrices of one launch
constexpr int kNormParts = 512;                              // most partial sums of a squared norm

// One matrix [rows, cols] (row-major, contiguous).  The iteration takes it as m x n, m <= n (transposed if rows > cols); mp, np: padded to
// multiples of 64.
struct Mat {
    const void* g;
    float* mom;              // momentum, or NULL
    float* p;                // parameter, or NULL
    void* out;               // orthogonalised matrix, or NULL
    _Float16* work;          // pairs: X [mp][np] twice (ping-pong), S [mp][mp], P [mp][mp]
    int rows, cols;
    float step;
    short parts;             // workgroups of the norm pass
    short whole;             // rows and pointers of the norm pass are whole 16-byte chunks
    __host__ __device__ int m() const { return rows < cols ? rows : cols; }
    __host__ __device__ int n() const { return rows < cols ? cols : rows; }
    __host__ __device__ int mp() const { return (m() + 63) & ~63; }
    __host__ __device__ int np() const { return (n() + 63) & ~63; }
    __device__ bool flip() const { return rows > cols; }
    __device__ _Float16* x(int k) const { return work + (long long)k * mp() * 2 * np(); }
    __device__ _Float16* s() const { return x(2); }
    __device__ _Float16* pm() const { return x(2) + (long long)mp() * 2 * mp(); }
};

struct NsArgs {
    Mat t[kGroup];           // same-shaped ones side by side
    double* norm;            // [count][kNormParts]
    float mu, eps, decay;
    int nesterov;
};

// position of element (r, c) in a pair matrix of padded width w; its rest is 32 further
__device__ __forceinline__ long long pair_at(long long r, int c, int w) { return r * 2 * w + (c >> 5) * 64 + (c & 31); }

__device__ __forceinline__ void split(float v, _Float16& hi, _Float16& lo) {
    hi = (_Float16)v;
    lo = (_Float16)(v - (float)hi);
}

// the update direction of element i
template <typename T>
__device__ __forceinline__ float direction(const NsArgs& a, const Mat& t, long long i) {
    const float g = (float)reinterpret_cast<const T*>(t.g)[i];
    if (!t.mom) return g;
    const float m = t.mom[i];
    return a.nesterov ? g + a.mu * m : m;
}

// momentum update and the squared norm of the direction: parts workgroups per matrix, four elements per thread, sums in 64 bits.  Bound by HBM:
// 47 M elements (gradient read, momentum read and written) in 94 us, 5.9 TB/s.
template <typename T>
__global__ __launch_bounds__(256) void k_ns_norm(NsArgs a) {
    __shared__ double red[4];
    const int b = blockIdx.y;
    const Mat& t = a.t[b];
    if ((int)blockIdx.x >= t.parts) return;
    const long long total = (long long)t.rows * t.cols;
    const T* g = reinterpret_cast<const T*>(t.g);
    float* mom = t.mom;
    double s = 0.0;
    auto add = [&](float u) { s += (double)u * (double)u; };
    if (t.whole) {
        typedef T vec __attribute__((ext_vector_type(4)));
        for (long long i = ((long long)blockIdx.x * 256 + threadIdx.x) * 4; i < total; i += 1024LL * t.parts) {
            const vec gv = *reinterpret_cast<const vec*>(g + i);
            if (mom) {
                float4 m = *reinterpret_cast<const float4*>(mom + i);
                m.x = a.mu * m.x + (float)gv[0]; m.y = a.mu * m.y + (float)gv[1]; m.z = a.mu * m.z + (float)gv[2]; m.w = a.mu * m.w + (float)gv[3];
                *reinterpret_cast<float4*>(mom + i) = m;
                add(a.nesterov ? (float)gv[0] + a.mu * m.x : m.x);
                add(a.nesterov ? (float)gv[1] + a.mu * m.y : m.y);
                add(a.nesterov ? (float)gv[2] + a.mu * m.z : m.z);
                add(a.nesterov ? (float)gv[3] + a.mu * m.w : m.w);
            } else {
#pragma unroll
                for (int k = 0; k < 4; ++k) add((float)gv[k]);
            }
        }
    } else {
        for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total; i += 256LL * t.parts) {
            if (mom) mom[i] = a.mu * mom[i] + (float)g[i];
            add(direction<T>(a, t, i));
        }
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) a.norm[(long long)b * kNormParts + blockIdx.x] = red[0] + red[1] + red[2] + red[3];
}

// X0 as pairs, zero past m and n; a 64 x 64 tile through LDS per workgroup (a matrix with rows > cols is turned there).  Bound by HBM: 47 M
// elements in 124 us, 4.5 TB/s.
template <typename T>
__global__ __launch_bounds__(256) void k_ns_pack(NsArgs a) {
    __shared__ float tile[64][65];
    __shared__ double red[4];
    const int b = blockIdx.z, i0 = blockIdx.y * 64, j0 = blockIdx.x * 64;       // rows / columns of X
    const int tx = threadIdx.x & 63, ty = threadIdx.x >> 6;
    const Mat& t = a.t[b];
    const int m = t.m(), n = t.n(), mp = t.mp(), np = t.np();
    const bool flip = t.flip();
    if (i0 >= mp || j0 >= np) return;
    float v[16];
#pragma unroll
    for (int q = 0; q < 16; ++q) {                                              // read along the rows as given
        const int r = ty + 4 * q, i = flip ? i0 + tx : i0 + r, j = flip ? j0 + r : j0 + tx;
        v[q] = i < m && j < n ? direction<T>(a, t, flip ? (long long)j * t.cols + i : (long long)i * t.cols + j) : 0.f;
    }
    double s = 0.0;
    for (int k = threadIdx.x; k < t.parts; k += 256) s += a.norm[(long long)b * kNormParts + k];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
    if (tx == 0) red[ty] = s;
    __syncthreads();
    const float inv = (float)((double)kScale / (sqrt(red[0] + red[1] + red[2] + red[3]) + (double)a.eps));
#pragma unroll
    for (int q = 0; q < 16; ++q) {
        const int r = ty + 4 * q;
        if (flip) tile[tx][r] = v[q] * inv;
        else tile[r][tx] = v[q] * inv;
    }
    __syncthreads();
    _Float16* x = t.x(0);
#pragma unroll
    for (int q = 0; q < 2; ++q) {                                               // eight entries of a row per thread: 16-byte stores
        const int r = (threadIdx.x >> 3) + 32 * q, c = (threadIdx.x & 7) * 8;
        half8 h, l;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            _Float16 p, w;
            split(tile[r][c + k], p, w);
            h[k] = p;
            l[k] = w;
        }
        const long long at = pair_at(i0 + r, j0 + c, np);
        *reinterpret_cast<half8*>(x + at) = h;
        *reinterpret_cast<half8*>(x + at + 32) = l;
    }
}

constexpr int threads_of(int T) { return T == 256 ? 512 : 256; }

template <int T>
__device__ __forceinline__ int tile_at(int row, int blk, int chunk) {
    return (row * (T / 32) + (blk ^ ((row >> 3) & 1))) * 128 + ((chunk ^ (row & 7)) << 4);
}

// The products of the iteration over pair matrices:
//   GRAM  S = X X^T
//   POLY  P = a + b S + c S S^T (a on the diagonal, so that X is not read again for a X)
//   STEP  X' = P X, from one copy of X into the other
//   LAST  the same, into the parameter or the output
enum { NS_GRAM = 0, NS_POLY = 1, NS_STEP = 2, NS_LAST = 3 };

// One launch over a group: same-shaped matrices are a class; a class's units are tiles, each split into `splits` shares of K
struct Class {
    int first;               // its first workgroup, a multiple of 8
    int mat, count;          // matrices mat .. mat + count
    int tiles_i, tiles_j, per_mat;
    int splits, part;        // shares per tile (1: none); its first share among all shares
};
struct Launch {
    Class c[kGroup];
    float* part;             // fp32 partial sums [share][T * T]
    int classes, in;         // which copy of X is read
};

// block -> class, unit.  Block b runs on XCD b % 8: every XCD gets an eighth of each class's units, neighbours of a matrix together; the odd
// units go to other XCDs class by class.  False: nothing to do.
__device__ __forceinline__ bool locate(const Launch& l, int bid, Class& c, int& id) {
    int k = 0;
    if (l.classes > 1) {
        while (k + 1 < l.classes && bid >= l.c[k + 1].first) ++k;
        c = l.c[k];
    }
    const int units = c.per_mat * c.count * c.splits, local = bid - c.first, x = ((local & 7) + 3 * k) & 7;
    id = (int)((long long)units * x / 8) + (local >> 3);
    return id < (int)((long long)units * (x + 1) / 8);
}

// tile of a matrix: SYM: on or below the diagonal
template <bool SYM>
__device__ __forceinline__ void tile_of(const Class& c, int rem, int& ti, int& tj) {
    if constexpr (SYM) {
        ti = (int)((sqrtf(8.f * (float)rem + 1.f) - 1.f) * 0.5f);
        while ((ti + 1) * (ti + 2) / 2 <= rem) ++ti;
        while (ti * (ti + 1) / 2 > rem) --ti;
        tj = rem - ti * (ti + 1) / 2;
    } else {
        ti = rem % c.tiles_i;                   // the row tiles of one panel of B side by side
        tj = rem / c.tiles_i;
    }
}

// Tile T x T, two rows of WJ waves of T/2 x T/WJ.  K goes in steps of 32 pairs (three products), through a ring of
// NST LDS stages filled by buffer_load ... lds, NST - 1 of them in flight.  A stage holds T rows of the left operand, 128 bytes of K each
// (chunks XOR-swizzled by (row >> 1) & 7), and of the right one, S or X^T, the same -- or, in P X, the 32 rows of X along K,
// T columns each, which the transposing LDS read turns (chunks XOR-swizzled by 4 (row & 3): its four rows meet different banks).
// GRAM and POLY are symmetric: tiles i >= j, stored twice.
// The epilogue goes through LDS: the tile of S arrives as whole lines (POLY), every lane replaces its own entries, and whole lines leave (GRAM,
// POLY: in both orientations, the transposed one by the transposing read); a 256 tile does that half by half.  A share of a split
// contraction leaves its fp32 sums in l.part instead, for k_ns_join.
// Bound by feeding the matrix pipe (busy 51 to 57 % of the cycles of a 256 tile), by the rounds and by the epilogue, which one workgroup per CU
// does not overlap.  16 x [1280, 1280], 256 tiles, in TF/s of half products: X X^T 116 us = 1040, S S^T 127 us = 950, P X 206 us = 980 (1.56 tiles per CU in two rounds).
// One [320, 320]: 7 to 8 us each, all latency.
template <int KIND, int T, int NST, typename OT>
__global__ __launch_bounds__(threads_of(T)) void k_ns_gemm(NsArgs a, Launch l) {
    [[maybe_unused]] constexpr int NT = threads_of(T), NW = NT / 64, WJ = NW / 2, ROWB = 128, STAGE = 2 * T * ROWB, TI = T / 2, TJ = T / WJ, FI = TI / 32, FJ = TJ / 32,
                                   PIECES = T / 8 / NW, H = T == 256 ? 2 : 1, TR = T / H;       // TR rows per epilogue pass
    [[maybe_unused]] constexpr bool SYM = KIND <= NS_POLY, LAST = KIND == NS_LAST, POLY = KIND == NS_POLY;
    // the result in units of 2^13 (LAST: 1) from products in units of 2^26
    [[maybe_unused]] constexpr float ACC = LAST ? kInv * kInv : POLY ? kC * kInv : kInv;
    // A 64 tile has LDS to spare for its tile of S: requested before the products instead of waited for behind them
    [[maybe_unused]] constexpr bool EARLY = POLY && T == 64;
    extern __shared__ __attribute__((aligned(16))) char smem[];      // EARLY: NST * STAGE + 4 TR T, else the larger of the two
#if defined(__HIP_DEVICE_COMPILE__)
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, hi = lane >> 5, l31 = lane & 31;
    const int wi = wave / WJ, wj = wave % WJ;
    // the arguments come from memory: the first class and matrix are requested at once, so that one matrix waits for them once, not three times
    Mat t = a.t[0];
    Class c = l.c[0];
    int id;
    if (!locate(l, blockIdx.x, c, id)) return;
    const int tiles = c.per_mat * c.count, z = id / tiles, tile = id - z * tiles, rel = tile / c.per_mat, splits = c.splits;
    int ti, tj;
    tile_of<SYM>(c, tile - rel * c.per_mat, ti, tj);
    if (c.mat + rel) t = a.t[c.mat + rel];
    const int mp = t.mp(), np = t.np();
    const int i0 = ti * T, j0 = tj * T;
    const int kw = KIND == NS_GRAM ? np : mp, ow = SYM ? mp : np, oh = mp;      // contraction; the result's columns and rows
    // bytes of a row of X in a stage (P X) and its 16-byte chunks; the swizzle of row's chunks
    [[maybe_unused]] constexpr int RB = 4 * T, CPR = RB / 16;
    [[maybe_unused]] auto turn = [](int row) __attribute__((always_inline)) { return (row & 3) << 2; };
    char* const pane = smem + (EARLY ? NST * STAGE : 0);
    [[maybe_unused]] auto source = [&](int r0) __attribute__((always_inline)) {         // rows r0 .. r0 + TR of the tile of S
        constexpr int P = TR * T / 256 / NW;                           // 1 KB = 8 blocks per wave and request
        const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc((void*)(t.s() + (long long)r0 * 2 * ow), 0, min(TR, oh - r0) * ow * 4, 0x00020000);
#pragma unroll
        for (int p = 0; p < P; ++p) {
            const int q = (wave * P + p) * 8 + (lane >> 3), row = q / (T / 32), blk = (q % (T / 32)) ^ ((row >> 3) & 1);
            const int chunk = (lane & 7) ^ (row & 7);
            const unsigned o = (unsigned)row * (unsigned)ow * 4u + (unsigned)((j0 / 32 + blk) * 128 + (chunk << 4));
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (__attribute__((address_space(3))) void*)(pane + (wave * P + p) * 1024), 16, (int)o, 0, 0, 0);
        }
    };
    if constexpr (EARLY) source(i0);
    f32x16 acc[FI][FJ];
    {
        const _Float16* A = KIND == NS_GRAM ? t.x(l.in) : KIND == NS_POLY ? t.s() : t.pm();
        const int arows = min(T, oh - i0), brows = min(T, ow - j0);
        const __amdgpu_buffer_rsrc_t ars = __builtin_amdgcn_make_buffer_rsrc((void*)(A + (long long)i0 * 2 * kw), 0, arows * kw * 4, 0x00020000);
        const __amdgpu_buffer_rsrc_t brs = __builtin_amdgcn_make_buffer_rsrc((void*)(A + (long long)j0 * 2 * kw), 0, brows * kw * 4, 0x00020000);      // (SYM)
        unsigned off[PIECES];                                      // rows past the matrix lie past the descriptor: zeros
#pragma unroll
        for (int p = 0; p < PIECES; ++p) {
            const int row = wave * (T / NW) + 8 * p + (lane >> 3);
            off[p] = (unsigned)row * (unsigned)kw * 4u + (unsigned)(((lane & 7) ^ ((row >> 1) & 7)) * 16);
        }
        [[maybe_unused]] unsigned xoff[PIECES];                    // P X: rows along K of X, columns past it out of range
        if constexpr (!SYM) {
#pragma unroll
            for (int p = 0; p < PIECES; ++p) {
                const int q = (wave * PIECES + p) * 64 + lane, row = q / CPR, chunk = (q % CPR) ^ turn(row), blk = chunk >> 3;
                xoff[p] = j0 + 32 * blk < ow ? (unsigned)row * (unsigned)ow * 4u + (unsigned)((j0 / 32 + blk) * 128 + (chunk & 7) * 16) : 0x80000000u;
            }
        }
        auto issue = [&](int s, int stage) __attribute__((always_inline)) {
            char* base = smem + stage * STAGE;
#pragma unroll
            for (int p = 0; p < PIECES; ++p)
                __builtin_amdgcn_raw_ptr_buffer_load_lds(ars, (__attribute__((address_space(3))) void*)(base + (wave * (T / NW) + 8 * p) * ROWB), 16, (int)off[p], s * 128, 0, 0);
            if constexpr (SYM) {
#pragma unroll
                for (int p = 0; p < PIECES; ++p)
                    __builtin_amdgcn_raw_ptr_buffer_load_lds(brs, (__attribute__((address_space(3))) void*)(base + T * ROWB + (wave * (T / NW) + 8 * p) * ROWB), 16, (int)off[p], s * 128, 0, 0);
            } else {
                const __amdgpu_buffer_rsrc_t xrs = __builtin_amdgcn_make_buffer_rsrc((void*)(t.x(l.in) + (long long)s * 64 * ow), 0, 32 * ow * 4, 0x00020000);
#pragma unroll
                for (int p = 0; p < PIECES; ++p)
                    __builtin_amdgcn_raw_ptr_buffer_load_lds(xrs, (__attribute__((address_space(3))) void*)(base + T * ROWB + (wave * PIECES + p) * 1024), 16, (int)xoff[p], 0, 0, 0);
            }
        };
#pragma unroll
        for (int i = 0; i < FI; ++i)
#pragma unroll
            for (int j = 0; j < FJ; ++j)
#pragma unroll
                for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;
        auto frag = [&](const char* base, int row, int chunk) __attribute__((always_inline)) {
            return *reinterpret_cast<const half8*>(base + row * ROWB + ((chunk ^ ((row >> 1) & 7)) << 4));
        };
        // eight k of one column of X per lane: two transposing reads of four rows each
        [[maybe_unused]] const int l15 = lane & 15, col = 16 * ((lane >> 4) & 1) + 4 * (l15 & 3), first = 8 * hi + (l15 >> 2);
        [[maybe_unused]] int at[FJ][2];                            // (turn has period 4: the steps along K are constants)
        if constexpr (!SYM) {
#pragma unroll
            for (int j = 0; j < FJ; ++j)
#pragma unroll
                for (int part = 0; part < 2; ++part) {
                    const int chunk = 8 * (TJ / 32 * wj + j) + 4 * part + (col >> 3);
                    at[j][part] = T * ROWB + first * RB + ((chunk ^ turn(first)) << 4) + ((col & 4) << 1);
                }
        }
        // All of a stage's fragments of X before the next stage is requested: the compiler lets a transposing read wait for every request in flight,
        // which costs nothing while there is none.  The deeper ring of 64 tiles always has some: there the reads bring their own wait.
        [[maybe_unused]] half8 xt[2][FJ][2];
        auto turned = [&](const char* base) __attribute__((always_inline)) {
            elem4 q[2][FJ][2][2];
            if constexpr (T == 64) {
                const unsigned p0 = (unsigned)(uintptr_t)(base + at[0][0]), p1 = (unsigned)(uintptr_t)(base + at[0][1]);
                asm volatile("ds_read_b64_tr_b16 %0, %8\n\tds_read_b64_tr_b16 %1, %8 offset:%10\n\t"
                             "ds_read_b64_tr_b16 %2, %9\n\tds_read_b64_tr_b16 %3, %9 offset:%10\n\t"
                             "ds_read_b64_tr_b16 %4, %8 offset:%11\n\tds_read_b64_tr_b16 %5, %8 offset:%12\n\t"
                             "ds_read_b64_tr_b16 %6, %9 offset:%11\n\tds_read_b64_tr_b16 %7, %9 offset:%12\n\ts_waitcnt lgkmcnt(0)"
                             : "=&v"(q[0][0][0][0]), "=&v"(q[0][0][0][1]), "=&v"(q[0][0][1][0]), "=&v"(q[0][0][1][1]), "=&v"(q[1][0][0][0]),
                               "=&v"(q[1][0][0][1]), "=&v"(q[1][0][1][0]), "=&v"(q[1][0][1][1])
                             : "v"(p0), "v"(p1), "n"(4 * RB), "n"(16 * RB), "n"(20 * RB) : "memory");
            } else {
#pragma unroll
                for (int kk = 0; kk < 2; ++kk)
#pragma unroll
                    for (int j = 0; j < FJ; ++j)
#pragma unroll
                        for (int part = 0; part < 2; ++part) {
                            q[kk][j][part][0] = dm_ds_read_tr16_b64(base + at[j][part] + 16 * kk * RB);
                            q[kk][j][part][1] = dm_ds_read_tr16_b64(base + at[j][part] + (16 * kk + 4) * RB);
                        }
            }
#pragma unroll
            for (int kk = 0; kk < 2; ++kk)
#pragma unroll
                for (int j = 0; j < FJ; ++j)
#pragma unroll
                    for (int part = 0; part < 2; ++part) {
                        const elem4 u = q[kk][j][part][0], v = q[kk][j][part][1];
                        xt[kk][j][part] = __builtin_bit_cast(half8, elem8{u[0], u[1], u[2], u[3], v[0], v[1], v[2], v[3]});
                    }
        };
        const int all = kw / 32;
        const int s_lo = (int)((long long)all * z / splits), s_hi = (int)((long long)all * (z + 1) / splits);
#pragma unroll
        for (int q = 0; q < NST - 1; ++q)
            if (s_lo + q < s_hi) issue(s_lo + q, q);
        int st = 0;
        for (int s = s_lo; s < s_hi; ++s) {
            // this wave's pieces of stage s have landed when at most the younger stages' (2 PIECES each) are outstanding
            if (s + NST - 2 < s_hi) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((NST - 2) * 2 * PIECES) : "memory");
            else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
            const char* ab = smem + st * STAGE;
            if constexpr (!SYM) turned(ab);
            const int fill = st == 0 ? NST - 1 : st - 1;           // the stage read one step ago
            if (s + NST - 1 < s_hi) issue(s + NST - 1, fill);
            const char* bb = ab + T * ROWB;
#pragma unroll
            for (int kk = 0; kk < 2; ++kk) {
                half8 ah[FI], al[FI], bh[FJ], bl[FJ];
#pragma unroll
                for (int i = 0; i < FI; ++i) {
                    const int row = TI * wi + 32 * i + l31;
                    ah[i] = frag(ab, row, 2 * kk + hi);
                    al[i] = frag(ab, row, 4 + 2 * kk + hi);
                }
#pragma unroll
                for (int j = 0; j < FJ; ++j) {
                    if constexpr (SYM) {
                        const int row = TJ * wj + 32 * j + l31;
                        bh[j] = frag(bb, row, 2 * kk + hi);
                        bl[j] = frag(bb, row, 4 + 2 * kk + hi);
                    } else {
                        bh[j] = xt[kk][j][0];
                        bl[j] = xt[kk][j][1];
                    }
                }
                // B as the matrix instruction's first operand: a lane holds one row i and four consecutive columns j per group
#pragma unroll
                for (int i = 0; i < FI; ++i)
#pragma unroll
                    for (int j = 0; j < FJ; ++j) {
                        acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(bl[j], ah[i], acc[i][j], 0, 0, 0);
                        acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(bh[j], al[i], acc[i][j], 0, 0, 0);
                        acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(bh[j], ah[i], acc[i][j], 0, 0, 0);
                    }
            }
            st = st + 1 == NST ? 0 : st + 1;
        }
        if (KIND == NS_GRAM && splits > 1) {
            float4* part = reinterpret_cast<float4*>(l.part) + (long long)(c.part + tile * splits + z) * (T * T / 4);
#pragma unroll
            for (int i = 0; i < FI; ++i)
#pragma unroll
                for (int j = 0; j < FJ; ++j)
#pragma unroll
                    for (int q = 0; q < 4; ++q)
                        part[((wave * FI + i) * FJ + j) * 256 + 64 * q + lane] =
                            make_float4(acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]);
            return;
        }
    }

    // ---- epilogue.  lane: row i = l31 of the fragment, registers 4 g + r: columns 8 g + 4 hi + r
    typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
    for (int h = 0; h < H; ++h) {
        const int r0 = i0 + h * TR;                                    // first row of this pass
        if (h && r0 >= oh) break;
        __syncthreads();                                               // every wave has read its last fragments (its share of the last pass)
        if constexpr (POLY && !EARLY) {
            source(r0);
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __syncthreads();
        }
        if (H == 1 || wi == h) {
#pragma unroll
            for (int fi = 0; fi < FI; ++fi)
#pragma unroll
                for (int fj = 0; fj < FJ; ++fj)
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const int row = (H == 1 ? TI * wi : 0) + 32 * fi + l31, blk = (TJ * wj) / 32 + fj;
                        half4* vp = reinterpret_cast<half4*>(pane + tile_at<T>(row, blk, q) + 8 * hi);
                        half4* rp = reinterpret_cast<half4*>(pane + tile_at<T>(row, blk, 4 + q) + 8 * hi);
                        float v[4];
#pragma unroll
                        for (int r = 0; r < 4; ++r) v[r] = acc[fi][fj][4 * q + r] * ACC;
                        if constexpr (POLY) {
                            const half4 hv = *vp, lv = *rp;
#pragma unroll
                            for (int r = 0; r < 4; ++r)
                                v[r] += kB * ((float)hv[r] + (float)lv[r]) + (r0 + row == j0 + 32 * blk + 8 * q + 4 * hi + r ? kA * kScale : 0.f);
                        }
                        if constexpr (LAST) {                          // fp32 in the pair's place: columns 0, 1 | 2, 3 of the four
                            *reinterpret_cast<float2*>(vp) = make_float2(v[0], v[1]);
                            *reinterpret_cast<float2*>(rp) = make_float2(v[2], v[3]);
                        } else {
                            half4 hv, lv;
#pragma unroll
                            for (int r = 0; r < 4; ++r) {
                                _Float16 x, y;
                                split(v[r], x, y);
                                hv[r] = x;
                                lv[r] = y;
                            }
                            *vp = hv;
                            *rp = lv;
                        }
                    }
        }
        __syncthreads();
        if constexpr (LAST) {
            const bool flip = t.flip();
            float* p = t.p;
            OT* out = reinterpret_cast<OT*>(t.out);
            // four entries per thread along the fast axis of the matrix as given, a batch of loads in flight
            constexpr int Q = TR * T / 4 / NT, U = T == 256 ? 4 : Q < 8 ? Q : 8;
            static_assert(Q % U == 0, "whole batches");
            const bool four = (flip ? t.m() : t.n()) % 4 == 0 && !((uintptr_t)(p ? (void*)p : (void*)out) & 15);
            for (int k0 = 0; k0 < Q; k0 += U) {
                float4 old[U];
                long long to[U];
                int ok[U];
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int k = tid + (k0 + u) * NT;
                    const int row = flip ? k % (TR / 4) * 4 : k / (T / 4), col = flip ? k / (TR / 4) : k % (T / 4) * 4, i = r0 + row, j = j0 + col;
                    const int fast = flip ? t.m() - i : t.n() - j, slow = flip ? t.n() - j : t.m() - i;
                    ok[u] = slow > 0 ? max(0, min(4, fast)) : 0;
                    to[u] = flip ? (long long)j * t.cols + i : (long long)i * t.cols + j;
                    if (p && ok[u]) {
                        if (four) old[u] = *reinterpret_cast<const float4*>(p + to[u]);
                        else {
                            old[u].x = p[to[u]];
                            old[u].y = ok[u] > 1 ? p[to[u] + 1] : 0.f;
                            old[u].z = ok[u] > 2 ? p[to[u] + 2] : 0.f;
                            old[u].w = ok[u] > 3 ? p[to[u] + 3] : 0.f;
                        }
                    }
                }
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    if (!ok[u]) continue;
                    const int k = tid + (k0 + u) * NT;
                    const int row = flip ? k % (TR / 4) * 4 : k / (T / 4), col = flip ? k / (TR / 4) : k % (T / 4) * 4;
                    float o[4];
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const int rr = flip ? row + r : row, cc = flip ? col : col + r;
                        o[r] = *reinterpret_cast<const float*>(pane + tile_at<T>(rr, cc >> 5, ((cc & 31) >> 3) + ((cc & 2) << 1)) + ((cc & 4) << 1) + ((cc & 1) << 2));
                    }
                    if (p) {
                        const float w[4] = {old[u].x * a.decay - t.step * o[0], old[u].y * a.decay - t.step * o[1], old[u].z * a.decay - t.step * o[2],
                                            old[u].w * a.decay - t.step * o[3]};
                        if (four) *reinterpret_cast<float4*>(p + to[u]) = make_float4(w[0], w[1], w[2], w[3]);
                        else
                            for (int r = 0; r < ok[u]; ++r) p[to[u] + r] = w[r];
                    } else if (four) {
                        typedef OT vec __attribute__((ext_vector_type(4)));
                        *reinterpret_cast<vec*>(out + to[u]) = vec{(OT)o[0], (OT)o[1], (OT)o[2], (OT)o[3]};
                    } else {
                        for (int r = 0; r < ok[u]; ++r) out[to[u] + r] = (OT)o[r];
                    }
                }
            }
        } else {
            _Float16* D = KIND == NS_GRAM ? t.s() : KIND == NS_POLY ? t.pm() : t.x(l.in ^ 1);
#pragma unroll 4
            for (int q = tid; q < TR * T / 4; q += NT) {               // 16-byte chunks, whole rows of blocks
                const int chunk = q & 7, blk = (q >> 3) % (T / 32), row = (q >> 3) / (T / 32);
                if (r0 + row < oh && j0 + 32 * blk < ow)
                    *reinterpret_cast<u32x4*>(D + (long long)(r0 + row) * 2 * ow + (j0 / 32 + blk) * 64 + chunk * 8) =
                        *reinterpret_cast<const u32x4*>(pane + tile_at<T>(row, blk, chunk));
            }
            if (SYM && ti != tj) {                                     // the other half: rows j, blocks of 32 i
                const int l15 = lane & 15, grp = lane >> 4;
                for (int u = wave; u < (T / 16) * (TR / 32) * 2; u += NW) {
                    const int part = u & 1, v = u >> 1, ib = v % (TR / 32), c0 = v / (TR / 32) * 16;
                    const int row = 32 * ib + 8 * grp + (l15 >> 2), cc = (c0 & 31) + 4 * (l15 & 3);
                    const char* p0 = pane + tile_at<T>(row, c0 >> 5, (cc >> 3) + 4 * part) + ((cc & 4) << 1);
                    const char* p1 = pane + tile_at<T>(row + 4, c0 >> 5, (cc >> 3) + 4 * part) + ((cc & 4) << 1);
                    const elem4 q0 = dm_ds_read_tr16_b64(p0), q1 = dm_ds_read_tr16_b64(p1);
                    const elem8 o = {q0[0], q0[1], q0[2], q0[3], q1[0], q1[1], q1[2], q1[3]};
                    const int j = j0 + c0 + l15, i = r0 + 32 * ib;
                    if (j < ow && i < oh) *reinterpret_cast<elem8*>(D + pair_at(j, i, oh) + 8 * grp + 32 * part) = o;
                }
            }
        }
    }
#endif
}

// S from the shares of a split Gram contraction, in both orientations: a wave per 32 x 32 block of a tile, summed in the shares' order.
// Bound by the read of the shares: 195 shares of 256 tiles in 14 us, 3.6 TB/s.
template <int T>
__global__ __launch_bounds__(256) void k_ns_join(NsArgs a, Launch l) {
    __shared__ float sums[4][32][33];
    constexpr int FI = T / 64, FJ = T == 256 ? 2 : T / 64, WJ = threads_of(T) / 128, BLOCKS = (T / 32) * (T / 32) / 4;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, hi = lane >> 5, l31 = lane & 31;
    int cls = 0;
    while (cls + 1 < l.classes && (int)blockIdx.x >= l.c[cls + 1].first) ++cls;
    const Class& c = l.c[cls];
    const int local = blockIdx.x - c.first, tile = local / BLOCKS, f = (local - tile * BLOCKS) * 4 + wave;      // f = (wave of the product, i, j)
    const int rel = tile / c.per_mat;
    int ti, tj;
    tile_of<true>(c, tile - rel * c.per_mat, ti, tj);
    const Mat& t = a.t[c.mat + rel];
    const int mp = t.mp(), w = f / (FI * FJ), i = f / FJ % FI, j = f % FJ;
    const int i0 = ti * T + T / 2 * (w / WJ) + 32 * i, j0 = tj * T + T / WJ * (w % WJ) + 32 * j;
    const float4* part = reinterpret_cast<const float4*>(l.part) + (long long)(c.part + tile * c.splits) * (T * T / 4) + f * 256 + lane;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        float4 v = part[64 * q];
        for (int z = 1; z < c.splits; ++z) {
            const float4 o = part[(long long)z * (T * T / 4) + 64 * q];
            v.x += o.x; v.y += o.y; v.z += o.z; v.w += o.w;
        }
        float* d = &sums[wave][l31][8 * q + 4 * hi];
        d[0] = v.x * kInv; d[1] = v.y * kInv; d[2] = v.z * kInv; d[3] = v.w * kInv;
    }
    __syncthreads();
    if (i0 >= mp || j0 >= mp) return;                                  // (mp is a multiple of 64)
    const int r = lane >> 1, c0 = (lane & 1) * 16;
    auto store = [&](int row0, int col0, bool turned) {
        _Float16* to = t.s() + pair_at(row0 + r, col0 + c0, mp);
#pragma unroll
        for (int o = 0; o < 16; o += 8) {
            half8 h, e;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                _Float16 x, y;
                split(turned ? sums[wave][c0 + o + k][r] : sums[wave][r][c0 + o + k], x, y);
                h[k] = x;
                e[k] = y;
            }
            *reinterpret_cast<half8*>(to + o) = h;
            *reinterpret_cast<half8*>(to + 32 + o) = e;
        }
    };
    store(i0, j0, false);
    if (ti != tj) store(j0, i0, true);
}

// A launch of one kind over a group, and what it should take, in K steps of 32 pairs on one CU with a 256 tile (2.8 us).
// Measured on 1280^2: a 256 tile needs a third of a 128 tile's LDS and request traffic per product; 128 tiles run two per CU and a
// round of 512 costs 1.15, half a round 0.6; 64 tiles 0.3 per 512, 0.18 where a CU gets one (then with a ring as deep as LDS allows: its
// loads have nothing else to hide behind).  Rounds: of equal units, whole ones; of unequal ones (longest first) the longest, or a tenth more
// than their mean over the CUs.
struct Plan {
    Launch l;
    int tile, blocks, units, shares;
    double cost;
};

constexpr int kShareBytes = 128 << 20;          // most memory of partial sums

// length > 0: the contraction is split into shares of at most so many steps (and no fewer than 16)
Plan plan_tile(const Mat* t, int count, int kind, int T, int length) {
    Plan p{};
    p.tile = T;
    struct Item { Class c; int steps; } items[kGroup];
    int n = 0, longest = 0, shortest = 1 << 30, top = 0;
    double work = 0;
    for (int at = 0, end; at < count; at = end) {
        for (end = at + 1; end < count && t[end].mp() == t[at].mp() && t[end].np() == t[at].np();) ++end;
        Item& q = items[n++];
        const int mp = t[at].mp(), np = t[at].np(), all = (kind == NS_GRAM ? np : mp) / 32;
        q.c = {};
        q.c.mat = at;
        q.c.count = end - at;
        q.c.tiles_i = (mp + T - 1) / T;
        q.c.tiles_j = ((kind <= NS_POLY ? mp : np) + T - 1) / T;
        q.c.per_mat = kind <= NS_POLY ? q.c.tiles_i * (q.c.tiles_i + 1) / 2 : q.c.tiles_i * q.c.tiles_j;
        q.c.splits = length > 0 ? std::max(1, std::min((all + length - 1) / length, all / 16)) : 1;
        q.steps = (all + q.c.splits - 1) / q.c.splits;
        const int units = q.c.per_mat * q.c.count * q.c.splits;
        if (q.c.splits > 1) {
            q.c.part = p.shares;
            p.shares += units;
        }
        p.units += units;
        work += (double)units * q.steps;
        longest = std::max(longest, q.steps);
        shortest = std::min(shortest, q.steps);
        top = std::max(top, mp);
    }
    std::stable_sort(items, items + n, [](const Item& x, const Item& y) { return x.steps > y.steps; });
    for (int i = 0; i < n; ++i) {
        p.l.c[i] = items[i].c;
        p.l.c[i].first = p.blocks;
        p.blocks += (items[i].c.per_mat * items[i].c.count * items[i].c.splits + 7) / 8 * 8;
    }
    p.l.classes = n;
    auto rounds = [&](int slots) {
        return longest == shortest ? (double)longest * ((p.units + slots - 1) / slots) : std::max((double)longest, 1.1 * work / slots);
    };
    if (T == 256) p.cost = rounds(256);
    else if (T == 128) p.cost = std::max(0.6 * longest, 1.15 * work / 512);
    else p.cost = p.units <= 256 ? 0.18 * longest : 0.3 * rounds(512);
    if (p.shares) p.cost += 2 + 0.05 * p.shares * (T * T) / 65536;       // the join: a launch, 256 KB written and read per share of a 256 tile
    if (top < T || (long long)p.shares * T * T * 4 > kShareBytes) p.cost = 1e30;
    return p;
}

Plan plan(const Mat* t, int count, int kind) {
    Plan best{};
    best.cost = 2e30;
    int most = 0;
    for (int i = 0; i < count; ++i) most = std::max(most, t[i].np() / 32);
    for (int T = 64; T <= 256; T *= 2)
        for (int d = 0; d <= (kind == NS_GRAM ? 16 : 0); ++d) {          // shares of a d-th of the longest contraction
            if (d && most / d < 16) break;
            const Plan p = plan_tile(t, count, kind, T, d ? (most + d - 1) / d : 0);
            if (p.cost < best.cost) best = p;
        }
    return best;
}

template <int KIND, int T, int NST, typename OT>
int launch_tile(const NsArgs& a, const Plan& p, int in, float* part, hipStream_t stream) {
    constexpr int RING = NST * 2 * T * 128, TILE = T == 256 ? 2 * T * T : 4 * T * T, LDS = T == 64 && KIND == NS_POLY ? RING + TILE : std::max(RING, TILE);
    static unsigned long long devices = 0;
    DM_HIP(dm_dynamic_lds(reinterpret_cast<const void*>(&k_ns_gemm<KIND, T, NST, OT>), LDS, devices));
    Launch l = p.l;
    l.in = in;
    l.part = part;
    hipLaunchKernelGGL((k_ns_gemm<KIND, T, NST, OT>), dim3(p.blocks), dim3(threads_of(T)), LDS, stream, a, l);
    DM_LAUNCH_CHECK();
    if constexpr (KIND == NS_GRAM) {
        if (!p.shares) return DM_OK;
        int n = 0, blocks = 0;
        for (int c = 0; c < p.l.classes; ++c) {
            if (p.l.c[c].splits < 2) continue;
            l.c[n] = p.l.c[c];
            l.c[n++].first = blocks;
            blocks += p.l.c[c].per_mat * p.l.c[c].count * ((T / 32) * (T / 32) / 4);
        }
        l.classes = n;
        hipLaunchKernelGGL((k_ns_join<T>), dim3(blocks), dim3(256), 0, stream, a, l);
        DM_LAUNCH_CHECK();
    }
    return DM_OK;
}

template <int KIND, typename OT>
int launch_gemm(const NsArgs& a, const Plan& p, int in, float* part, hipStream_t stream) {
    if (p.tile == 256) return launch_tile<KIND, 256, 2, OT>(a, p, in, part, stream);
    if (p.tile == 128) return launch_tile<KIND, 128, 2, OT>(a, p, in, part, stream);
    if (p.units <= 256) return launch_tile<KIND, 64, 8, OT>(a, p, in, part, stream);
    return launch_tile<KIND, 64, 4, OT>(a, p, in, part, stream);
}

#define NS_TRY(call) do { if (int rc_ = (call)) return rc_; } while (0)

template <typename T>
int run_group(const NsArgs& a, int count, int steps, float* part, hipStream_t stream) {
    int parts = 1, mp = 0, np = 0;
    for (int i = 0; i < count; ++i) {
        parts = std::max<int>(parts, a.t[i].parts);
        mp = std::max(mp, a.t[i].mp());
        np = std::max(np, a.t[i].np());
    }
    hipLaunchKernelGGL((k_ns_norm<T>), dim3(parts, count), dim3(256), 0, stream, a);
    hipLaunchKernelGGL((k_ns_pack<T>), dim3(np / 64, mp / 64, count), dim3(256), 0, stream, a);
    DM_LAUNCH_CHECK();
    const Plan gram = plan(a.t, count, NS_GRAM), poly = plan(a.t, count, NS_POLY), step = plan(a.t, count, NS_STEP);
    for (int k = 0; k < steps; ++k) {
        NS_TRY((launch_gemm<NS_GRAM, float>(a, gram, k & 1, part, stream)));
        NS_TRY((launch_gemm<NS_POLY, float>(a, poly, 0, part, stream)));
        if (k + 1 < steps) NS_TRY((launch_gemm<NS_STEP, float>(a, step, k & 1, part, stream)));
        else NS_TRY((launch_gemm<NS_LAST, T>(a, step, k & 1, part, stream)));
    }
    return DM_OK;
}

// workspace of one matrix (X twice, S, P, norm) and of a group
long long mat_bytes(const Mat& t) { return 4LL * t.mp() * (2LL * t.np() + 2LL * t.mp()) + 8 * kNormParts; }
long long group_bytes(const Mat* t, int count) {
    const Plan gram = plan(t, count, NS_GRAM);
    long long b = 4LL * gram.shares * gram.tile * gram.tile;
    for (int i = 0; i < count; ++i) b += mat_bytes(t[i]);
    return b;
}
// the most that groups of `fit` need
long long need_bytes(const std::vector<Mat>& t, int fit) {
    long long b = 0;
    for (size_t at = 0; at < t.size(); at += fit) b = std::max(b, group_bytes(t.data() + at, (int)std::min<size_t>(fit, t.size() - at)));
    return b;
}

bool sizes_ok(int rows, int cols) { return (long long)rows * cols <= (1LL << 31) && std::min(rows, cols) <= 32768 && std::max(rows, cols) <= (1 << 20); }

// largest first, equal shapes side by side
void order(std::vector<Mat>& t) {
    std::stable_sort(t.begin(), t.end(), [](const Mat& x, const Mat& y) {
        const long long a = (long long)x.mp() * x.np(), b = (long long)y.mp() * y.np();
        return a != b ? a > b : x.mp() > y.mp();
    });
}

// dtype of the gradients / outputs: 0 bf16, 1 half, 2 fp32
int run(std::vector<Mat>& t, NsArgs& a, int dtype, int steps, void* ws, size_t ws_bytes, hipStream_t stream) {
    if (steps < 1 || steps > 64 || dtype < 0 || dtype > 2 || !ws || ((uintptr_t)ws & 255)) return DM_ERR_ARG;
    for (Mat& m : t) {
        if (!m.g || (m.p ? !m.mom : !m.out) || m.rows <= 0 || m.cols <= 0) return DM_ERR_ARG;
        if (!sizes_ok(m.rows, m.cols)) return DM_ERR_UNSUPPORTED;
        m.parts = (short)std::max<long long>(1, std::min<long long>(kNormParts, (long long)m.rows * m.cols / (256 * 8)));
        m.whole = m.cols % 4 == 0 && !(((uintptr_t)m.g | (uintptr_t)m.mom) & 15);      // rows of 16-byte (8-byte) chunks in every operand of the norm pass
    }
    order(t);
    int fit = kGroup;
    while (fit && need_bytes(t, fit) > (long long)ws_bytes) --fit;
    if (!fit) return DM_ERR_WORKSPACE;
    DM_ENTER();
    for (size_t at = 0; at < t.size(); at += fit) {
        const int c = (int)std::min<size_t>(fit, t.size() - at);
        char* w = (char*)ws;
        a.norm = (double*)w;
        w += 8LL * kNormParts * c;
        for (int i = 0; i < c; ++i) {
            a.t[i] = t[at + i];
            a.t[i].work = (_Float16*)w;
            w += mat_bytes(a.t[i]) - 8 * kNormParts;
        }
        float* part = (float*)w;
        const int rc = dtype == 0 ? run_group<__bf16>(a, c, steps, part, stream) : dtype == 1 ? run_group<_Float16>(a, c, steps, part, stream) : run_group<float>(a, c, steps, part, stream);
        if (rc) return rc;
    }
    return DM_OK;
}

// host memory for the matrices' list: an allocation that fails is an error code, not an exception
template <typename F>
int with_mats(int count, F f) {
    try {
        std::vector<Mat> t((size_t)count);
        return f(t);
    } catch (const std::bad_alloc&) {
        return DM_ERR_WORKSPACE;
    }
}

}  // namespace

extern "C" {

// workspace bytes that take `count` [rows, cols] matrices in groups of 16 (less memory, down to one matrix's: smaller groups); 0: sizes out of range
size_t dm_orthogonalize_workspace_bytes(int count, int rows, int cols) {
    if (count <= 0 || rows <= 0 || cols <= 0 || !sizes_ok(rows, cols)) return 0;
    Mat t[kGroup] = {};
    for (Mat& m : t) { m.rows = rows; m.cols = cols; }
    return (size_t)std::max(group_bytes(t, std::min(count, kGroup)), count > kGroup && count % kGroup ? group_bytes(t, count % kGroup) : 0);
}

// the same for matrices of their own sizes
size_t dm_muon_step_workspace_bytes(const int* rows_host, const int* cols_host, int count) {
    if (count <= 0 || !rows_host || !cols_host) return 0;
    size_t bytes = 0;
    with_mats(count, [&](std::vector<Mat>& t) {
        for (int i = 0; i < count; ++i) {
            t[i].rows = rows_host[i];
            t[i].cols = cols_host[i];
            if (rows_host[i] <= 0 || cols_host[i] <= 0 || !sizes_ok(rows_host[i], cols_host[i])) return DM_ERR_ARG;
        }
        order(t);
        bytes = (size_t)need_bytes(t, kGroup);
        return DM_OK;
    });
    return bytes;
}

// out[i] = Newton-Schulz of g[i]: `count` same-shaped matrices [rows, cols] behind HOST arrays of device pointers; dtype 0 bf16 |
// 1 half | 2 fp32 of both; ws 256-byte aligned
int dm_orthogonalize(const void* const* g_host, void* const* out_host, int count, int rows, int cols, int dtype, int steps, float eps, void* ws,
                     size_t ws_bytes, hipStream_t stream) {
    if (count < 0 || rows <= 0 || cols <= 0 || (count && (!g_host || !out_host))) return DM_ERR_ARG;
    return with_mats(count, [&](std::vector<Mat>& t) {
        for (int i = 0; i < count; ++i) {
            t[i].g = g_host[i];
            t[i].out = out_host[i];
            t[i].rows = rows;
            t[i].cols = cols;
        }
        NsArgs a{};
        a.eps = eps;
        return run(t, a, dtype, steps, ws, ws_bytes, stream);
    });
}

// momentum step on fp32 masters of their own sizes: mom <- mu mom + g;  u = g + mu mom or mom;  p <- p decay - step[i] orth(u).  g of `dtype`,
// mom / p fp32; all arrays on the HOST
int dm_muon_step(const void* const* g_host, float* const* mom_host, float* const* p_host, const int* rows_host, const int* cols_host,
                 const float* step_host, int count, int dtype, int steps, float mu, int nesterov, float eps, float decay, void* ws, size_t ws_bytes,
                 hipStream_t stream) {
    if (count < 0 || (count && (!g_host || !mom_host || !p_host || !rows_host || !cols_host || !step_host))) return DM_ERR_ARG;
    return with_mats(count, [&](std::vector<Mat>& t) {
        for (int i = 0; i < count; ++i) {
            t[i].g = g_host[i];
            t[i].mom = mom_host[i];
            t[i].p = p_host[i];
            t[i].rows = rows_host[i];
            t[i].cols = cols_host[i];
            t[i].step = step_host[i];
        }
        NsArgs a{};
        a.mu = mu; a.nesterov = nesterov; a.eps = eps; a.decay = decay;
        return run(t, a, dtype, steps, ws, ws_bytes, stream);
    });
}

}  // extern "C"
