// Low-rank adapters of many requests at once beside a frozen projection (gfx950, bf16 and -- with -DDM_F16 -- IEEE half).
//
//   y[m, :] = x[m, :] W^T + bias + u[m, :] B_e^T (+ residual[m, :])        u[m, :] = s x[m, :] A_e^T        e = adapter of row m
//
// W [N, K] is shared and frozen, A [E, R, K] and B [E, N, R] are the adapters.  Row m belongs to request i (rows of equal count, or
// offsets[i] <= m < offsets[i + 1]) and request i to adapter ids[i]; rows of no request and ids outside [0, E) have no adapter.
//
// Three kernels:
//   shrink  u = s x A_e^T, one pass over x; u is kept as a PAIR of 16-bit numbers (value and remainder: 16-22 significant bits), so
//           the second product loses nothing against fp32 and still runs on the 16-bit matrix pipe.  In half precision a row is
//           scaled by the power of two that brings its largest entry to [2^13, 2^14): half's exponent range must not bound u, and
//           entries down to 2^-22 of the largest keep 16 bits (2^-27: 11), so that a small rank beside a large one keeps its gradient.
//           Infinities come out as the formula has them: an infinite u has a zero rest, and where the other factor is infinite the
//           rest takes no part (the value's product decides; the rest's would turn it into NaN).
//   expand  the big product, its K loop extended by [u_value | u_rest] [B | B]^T: the low-rank product costs 2 ceil(R/16) 16
//           columns of K and no pass over y.  Rows of a tile that belong to another adapter are left out by selection (never by
//           a multiplication with zero: 0 * inf of another request's adapter would reach them).
//   wgrad   dA_e = du^T x and dB_e = dy^T u over the rows of e, rows gathered in adapter order, split over row ranges and joined in
//           a fixed order (no atomics).
// The data gradient is the same pair of kernels on (dy, W^T, B^T, A^T): dx = dy W + (s dy B_e) A_e.
#include <algorithm>
#include <type_traits>

#include "dm_common.h"
#include "dm_elem.h"

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

constexpr int kMaxRank = 128;
constexpr int kNone = -1;

__host__ __device__ inline int rank_pad(int R) { return R <= 16 ? 16 : R <= 32 ? 32 : R <= 64 ? 64 : 128; }

// which adapter a row belongs to
struct Rows {
    const int* ids;        // [n]
    const int* offsets;    // [n + 1] or NULL: n requests of `each` rows
    long long M, each;
    int n, E;
};

__device__ __forceinline__ int checked(int id, int E) { return (unsigned)id < (unsigned)E ? id : kNone; }

__device__ __forceinline__ int adapter_of(const Rows& r, long long m) {
    if (m >= r.M) return kNone;
    if (!r.offsets) return checked(r.ids[m / r.each], r.E);
    int lo = 0, hi = r.n;                                   // the last request that starts at or before m
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (r.offsets[mid + 1] <= m) lo = mid + 1;
        else hi = mid;
    }
    return lo < r.n && r.offsets[lo] <= m ? checked(r.ids[lo], r.E) : kNone;
}

__device__ __forceinline__ float pow2_scale(float biggest) {
#if defined(DM_F16)
    // 2^k that brings the row's largest entry to [2^13, 2^14); 1 for a row of zeros.  k >= -60, because the big product divides
    // x W^T (below 2^52) by it in fp32: an even smaller u has fewer bits, and adds less than the smallest half.
    if (!(biggest > 0.f)) return 1.f;
    int e;
    frexpf(biggest, &e);
    return ldexpf(1.f, max(e - 14, -60));
#else
    return 1.f;
#endif
}

// ------------------------------------------------------------------------------------------------ shrink
// u rows are stored [value: Rp | rest: Rp] elem_t (Rp = rank_pad(R), columns past R zero) with us[m] = the row's power of two and who[m] = the
// row's adapter, which the big product then reads instead of searching for it.
__device__ __forceinline__ elem_t rest_of(float v, elem_t hi) {
    const float h = (float)hi;
    return fabsf(h) <= 3.4028235e38f ? (elem_t)(v - h) : (elem_t)0.f;
}

__device__ __forceinline__ void store_pair(elem_t* u, int Rp, int r, float v) {
    const elem_t hi = (elem_t)v;
    u[r] = hi;
    u[Rp + r] = rest_of(v, hi);
}

// |v| where v is finite, for the largest entry of a row
__device__ __forceinline__ float finite_abs(float v) { return fabsf(v) <= 3.4028235e38f ? fabsf(v) : 0.f; }

// the entries with infinities and NaN as zeros (an exponent of ones), two to a dword
__device__ __forceinline__ elem8 finite_only(elem8 v) {
    typedef unsigned short u16x8 __attribute__((ext_vector_type(8)));
#if defined(DM_F16)
    constexpr unsigned short biggest = 0x7bff;
#else
    constexpr unsigned short biggest = 0x7f7f;
#endif
    const u16x8 bits = __builtin_bit_cast(u16x8, v), one = 1;
    const u16x8 over = __builtin_elementwise_sub_sat(bits & (unsigned short)0x7fff, u16x8(biggest));        // 0 where finite
    return __builtin_bit_cast(elem8, bits & (__builtin_elementwise_min(over, one) - one));
}

// the smallest entry of a tile's adapters above cur (INT_MAX: none), the same in every wave
template <int TR>
__device__ __forceinline__ int next_adapter(const int* aid, int cur) {
    const int lane = threadIdx.x & 63;
    int next = 0x7fffffff;
#pragma unroll
    for (int t = 0; t < (TR + 63) / 64; ++t) {
        const int v = aid[(64 * t + lane) % TR];
        next = v > cur && v < next ? v : next;
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) next = min(next, __shfl_xor(next, o, 64));
    return __builtin_amdgcn_readfirstlane(next);
}

// Tile of 16 RT rows; the four waves take 64-wide slices of K in turn, so a tile reads its x rows once (128-byte lines) and the rank
// rows of A once from L2; a slice is requested before the last one is multiplied; the partial products meet in LDS.  One pass per adapter
// that occurs in the tile.  Bound by the x read, with few rows by latency (the search of the row's request, then K): 1851 ragged rows of 1024
// halves, rank 32: 12 us.
template <int RT, int NR>
__global__ __launch_bounds__(256) void k_shrink(const elem_t* __restrict__ x, const elem_t* __restrict__ A, Rows rows, int K, int R, float scale,
                                                elem_t* __restrict__ u, float* __restrict__ us, int* __restrict__ who) {
    constexpr int TR = 16 * RT, Rp = 16 * NR;
    __shared__ float part[4][TR][Rp + 1];
    __shared__ int aid[TR];
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, l15 = lane & 15, kq = lane >> 4;
    const long long m0 = (long long)blockIdx.x * TR;
    if (tid < TR) {
        aid[tid] = adapter_of(rows, m0 + tid);
        if (m0 + tid < rows.M) who[m0 + tid] = aid[tid];
    }
    __syncthreads();
    const elem_t* xr[RT];
#pragma unroll
    for (int t = 0; t < RT; ++t) xr[t] = x + min(m0 + 16 * t + l15, rows.M - 1) * K + 8 * kq;
    int cur = kNone;
    for (;;) {
        cur = next_adapter<TR>(aid, cur);
        if (cur == 0x7fffffff) break;
        const elem_t* ar[NR];
#pragma unroll
        for (int q = 0; q < NR; ++q) ar[q] = A + ((long long)cur * R + min(16 * q + l15, R - 1)) * K + 8 * kq;
        f32x4 acc[RT][NR];
#pragma unroll
        for (int t = 0; t < RT; ++t)
#pragma unroll
            for (int q = 0; q < NR; ++q) acc[t][q] = f32x4{0.f, 0.f, 0.f, 0.f};
        struct Slice { elem8 x[2][RT], a[2][NR]; };
        auto load = [&](int k0, Slice& f) __attribute__((always_inline)) {
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                const int k = k0 + 32 * s;
                const bool ok = k + 8 * kq < K;
                const elem8 zero = {};
#pragma unroll
                for (int t = 0; t < RT; ++t) f.x[s][t] = ok ? *reinterpret_cast<const elem8*>(xr[t] + k) : zero;
#pragma unroll
                for (int q = 0; q < NR; ++q) f.a[s][q] = ok ? *reinterpret_cast<const elem8*>(ar[q] + k) : zero;
            }
        };
        auto mul = [&](const Slice& f) __attribute__((always_inline)) {
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int t = 0; t < RT; ++t)
#pragma unroll
                    for (int q = 0; q < NR; ++q) acc[t][q] = DM_MFMA_16x16x32(f.x[s][t], f.a[s][q], acc[t][q]);
        };
        Slice f0, f1;
        int k0 = 64 * wave;
        if (k0 < K) load(k0, f0);
        while (k0 < K) {
            if (k0 + 256 < K) load(k0 + 256, f1);
            mul(f0);
            k0 += 256;
            if (k0 >= K) break;
            if (k0 + 256 < K) load(k0 + 256, f0);
            mul(f1);
            k0 += 256;
        }
        // lane: rank 16 q + l15, rows 4 kq + i
#pragma unroll
        for (int t = 0; t < RT; ++t)
#pragma unroll
            for (int q = 0; q < NR; ++q)
#pragma unroll
                for (int i = 0; i < 4; ++i) part[wave][16 * t + 4 * kq + i][16 * q + l15] = acc[t][q][i];
        __syncthreads();
        // 16 lanes per row
        for (int t = tid >> 4; t < TR; t += 16) {
            const long long m = m0 + t;
            float v[NR], big = 0.f;
#pragma unroll
            for (int q = 0; q < NR; ++q) {
                const int r = 16 * q + l15;
                v[q] = r < R ? scale * (part[0][t][r] + part[1][t][r] + part[2][t][r] + part[3][t][r]) : 0.f;
                big = fmaxf(big, finite_abs(v[q]));
            }
#if defined(DM_F16)
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) big = fmaxf(big, __shfl_xor(big, o, 16));
#endif
            if (aid[t] == cur) {
                const float p = pow2_scale(big);
#pragma unroll
                for (int q = 0; q < NR; ++q) store_pair(u + m * 2 * Rp, Rp, 16 * q + l15, v[q] / p);
                if (l15 == 0) us[m] = p;
            }
        }
        __syncthreads();
    }
}

// The same for many rows: tiles of 64 rows, x and the rank rows through a ring of LDS stages (buffer_load ... lds, whole 128-byte lines,
// three stages in flight), a wave 16 rows.  Against the kernel above, whose fragments are gathered from 16 rows by every load: rank 64 of
// [24576, 5120] 187 -> 70 us (3.6 TB/s), rank 64 of [24576, 1280] 21 us.
template <int NR>
__global__ __launch_bounds__(256) void k_shrink_ring(const elem_t* __restrict__ x, const elem_t* __restrict__ A, Rows rows, int K, int R, float scale,
                                                     elem_t* __restrict__ u, float* __restrict__ us, int* __restrict__ who) {
    [[maybe_unused]] constexpr int Rp = 16 * NR, ROWB = 128, STAGE = (64 + Rp) * ROWB, NST = 4, PA = Rp >= 32 ? Rp / 32 : 1;
    extern __shared__ __attribute__((aligned(16))) char smem[];      // NST STAGE | int aid[64]
#if defined(__HIP_DEVICE_COMPILE__)
    constexpr unsigned OOB = 0x80000000u;
    int* aid = reinterpret_cast<int*>(smem + NST * STAGE);
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, l15 = lane & 15, kq = lane >> 4;
    const long long m0 = (long long)blockIdx.x * 64;
    const int mrows = (int)min(64LL, rows.M - m0), steps = (K + 63) / 64;
    const __amdgpu_buffer_rsrc_t xrs = __builtin_amdgcn_make_buffer_rsrc((void*)(x + m0 * K), 0, mrows * K * 2, 0x00020000);
    // x pieces: rows 16 wave + 8 i; rank pieces: rows 8 p of A (with 16 ranks two waves fetch each piece)
    auto chunk_of = [&](int row) __attribute__((always_inline)) { return (unsigned)(((lane & 7) ^ ((row >> 1) & 7)) * 8); };
    if (tid < 64) {
        aid[tid] = adapter_of(rows, m0 + tid);
        if (tid < mrows) who[m0 + tid] = aid[tid];
    }
    __syncthreads();
    int cur = kNone;
    for (;;) {
        cur = next_adapter<64>(aid, cur);
        if (cur == 0x7fffffff) break;
        const __amdgpu_buffer_rsrc_t ars = __builtin_amdgcn_make_buffer_rsrc((void*)(A + (long long)cur * R * K), 0, R * K * 2, 0x00020000);
        auto issue = [&](int s, int stage) __attribute__((always_inline)) {
            char* base = smem + stage * STAGE;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int row = 16 * wave + 8 * i + (lane >> 3);
                const unsigned k = (unsigned)(s * 64) + chunk_of(row);
                const unsigned off = row < mrows && k < (unsigned)K ? ((unsigned)row * (unsigned)K + k) * 2u : OOB;
                __builtin_amdgcn_raw_ptr_buffer_load_lds(xrs, (__attribute__((address_space(3))) void*)(base + (16 * wave + 8 * i) * ROWB), 16, (int)off, 0, 0, 0);
            }
#pragma unroll
            for (int i = 0; i < PA; ++i) {
                const int p = (PA * wave + i) % (Rp / 8), row = 8 * p + (lane >> 3);
                const unsigned k = (unsigned)(s * 64) + chunk_of(row);
                const unsigned off = row < R && k < (unsigned)K ? ((unsigned)row * (unsigned)K + k) * 2u : OOB;
                __builtin_amdgcn_raw_ptr_buffer_load_lds(ars, (__attribute__((address_space(3))) void*)(base + (64 + 8 * p) * ROWB), 16, (int)off, 0, 0, 0);
            }
        };
        f32x4 acc[NR];
#pragma unroll
        for (int q = 0; q < NR; ++q) acc[q] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int q = 0; q < NST - 1; ++q)
            if (q < steps) issue(q, q);
        int stage = 0;
        for (int s = 0; s < steps; ++s) {
            if (s + NST - 2 < steps) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((NST - 2) * (2 + PA)) : "memory");
            else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
            if (s + NST - 1 < steps) issue(s + NST - 1, stage == 0 ? NST - 1 : stage - 1);
            const char* xb = smem + stage * STAGE;
            const char* ab = xb + 64 * ROWB;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                auto frag = [&](const char* base, int row) __attribute__((always_inline)) {
                    return *reinterpret_cast<const elem8*>(base + row * ROWB + (((4 * h + kq) ^ ((row >> 1) & 7)) << 4));
                };
                const elem8 xf = frag(xb, 16 * wave + l15);
#pragma unroll
                for (int q = 0; q < NR; ++q) acc[q] = DM_MFMA_16x16x32(xf, frag(ab, 16 * q + l15), acc[q]);
            }
            stage = stage + 1 == NST ? 0 : stage + 1;
        }
        // lane: rank 16 q + l15, rows 4 kq + i of the wave's 16
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int t = 16 * wave + 4 * kq + i;
            float v[NR], big = 0.f;
#pragma unroll
            for (int q = 0; q < NR; ++q) {
                v[q] = 16 * q + l15 < R ? scale * acc[q][i] : 0.f;
                big = fmaxf(big, finite_abs(v[q]));
            }
#if defined(DM_F16)
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) big = fmaxf(big, __shfl_xor(big, o, 16));
#endif
            if (aid[t] == cur) {
                const float p = pow2_scale(big);
#pragma unroll
                for (int q = 0; q < NR; ++q) store_pair(u + (m0 + t) * 2 * Rp, Rp, 16 * q + l15, v[q] / p);
                if (l15 == 0) us[m0 + t] = p;
            }
        }
        __syncthreads();                                             // the stages are free for the next adapter
    }
#endif
}

// One row per workgroup, one rank row per wave: requests of a few rows each, where a tile would hold many adapters.  Every row reads
// its own adapter (R K 2 bytes).  f32out: plain fp32 [M][Rp] for the skinny product, else the pair format.  16 rows of 1280, rank 16: 3.7 us.
__global__ __launch_bounds__(1024) void k_shrink_rows(const elem_t* __restrict__ x, const elem_t* __restrict__ A, Rows rows, int K, int R, float scale,
                                                      elem_t* __restrict__ u, float* __restrict__ us, int* __restrict__ who, float* __restrict__ f32out) {
    __shared__ float row[kMaxRank];
    const int tid = threadIdx.x, lane = tid & 63, Rp = rank_pad(R);
    for (long long m = blockIdx.x; m < rows.M; m += gridDim.x) {
        const int e = adapter_of(rows, m);
        if (!f32out && tid == 0) who[m] = e;
        if (e == kNone) continue;
        const elem_t* xr = x + m * K;
        for (int r = tid >> 6; r < R; r += blockDim.x >> 6) {
            const elem_t* ar = A + ((long long)e * R + r) * K;
            float s = 0.f;
            for (int k = lane * 8; k < K; k += 512) {
                const elem8 xv = *reinterpret_cast<const elem8*>(xr + k), av = *reinterpret_cast<const elem8*>(ar + k);
#pragma unroll
                for (int i = 0; i < 8; ++i) s += (float)xv[i] * (float)av[i];
            }
#pragma unroll
            for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
            if (lane == 0) row[r] = scale * s;
        }
        __syncthreads();
        if (f32out) {
            for (int r = tid; r < Rp; r += blockDim.x) f32out[m * Rp + r] = r < R ? row[r] : 0.f;
        } else {
            float big = 0.f;
            for (int r = 0; r < R; ++r) big = fmaxf(big, finite_abs(row[r]));
            const float p = pow2_scale(big);
            for (int r = tid; r < Rp; r += blockDim.x) store_pair(u + m * 2 * Rp, Rp, r, r < R ? row[r] / p : 0.f);
            if (tid == 0) us[m] = p;
        }
        __syncthreads();
    }
}

// ------------------------------------------------------------------------------------------------ expand
struct ExpandArgs {
    const elem_t *x, *w, *bias, *res, *u, *B;
    const float* us;
    const int* who;
    elem_t* y;
    Rows rows;
    int K, N, R, ldb;      // ldb: elements between the rows of B (a multiple of 8)
    int n_mt, n_nt, tiles;
};

// BM x BN x 64 tile, WM x WN waves, NST LDS stages filled by buffer_load ... lds (16 bytes per lane, range-checked: rows and
// columns past the end read as zeros).  LDS rows are 128 bytes, the 16-byte chunks XOR-swizzled by (row >> 1) & 7 at the source address
// and at the fragment read: conflict-free without padding.  The weights are the matrix instruction's A operand, so a lane holds one row of y
// and four consecutive columns per register group: 16-byte stores after one exchange between the wave's halves.  Bound by feeding the matrix
// pipe (two workgroups per CU cover each other's waits; it is busy 46 to 49 % of the cycles, LDS without conflicts): bf16, rank 64, [24576,
// 1280 -> 5120] 435 us = 740 TF/s of the plain product, [24576, 5120 -> 1280] 375 us = 860; [24576, 640 -> 640] rank 16 with residual 37 us,
// 2.5 TB/s.  With a short K by the latencies of a tile (its adapters, two loads, the store): [24576, 64 -> 4096] rank 16 in 67 us.
template <int BM, int BN, int WM, int WN, int NST>
__global__ __launch_bounds__(WM * WN * 64) void k_expand(ExpandArgs a) {
    [[maybe_unused]] constexpr int NW = WM * WN, ROWB = 128;
    [[maybe_unused]] constexpr int TM = BM / WM, TN = BN / WN, MT = TM / 32, NT = TN / 32;
    [[maybe_unused]] constexpr int A_BYTES = BM * ROWB, STAGE = (BM + BN) * ROWB;
    [[maybe_unused]] constexpr int AP = BM / 8 / NW, BP = BN / 8 / NW;                // 1 KB pieces (8 rows) per wave
    extern __shared__ __attribute__((aligned(16))) char smem[];      // NST STAGE | int aid[BM] | float scale_of[BM] | float bias_of[BN]
#if defined(__HIP_DEVICE_COMPILE__)
    constexpr unsigned OOB = 0x80000000u;             // past every descriptor, also with a step's scalar offset on top
    int* aid = reinterpret_cast<int*>(smem + NST * STAGE);
    float* scale_of = reinterpret_cast<float*>(aid + BM);
    float* bias_of = scale_of + BM;
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, hi = lane >> 5, l31 = lane & 31;
    const int wm = wave / WN, wn = wave % WN;
    // block b runs on XCD b % 8 (its own L2): each XCD gets a contiguous run of tiles, walked in bands of eight row panels (the
    // tiles that run together then share their panels: [24576, 5120, 1280] 418 -> 354 us on 128 tiles against whole rows of tiles)
    const int per = (a.tiles + 7) / 8, id = (int)(blockIdx.x & 7) * per + (int)(blockIdx.x >> 3);
    if ((int)(blockIdx.x >> 3) >= per || id >= a.tiles) return;
    constexpr int BAND = 8;
    const int band = (int)((unsigned)id / (unsigned)(BAND * a.n_nt)), in_band = id - band * BAND * a.n_nt, height = min(BAND, a.n_mt - band * BAND);
    const int column = height == BAND ? in_band / BAND : (int)((unsigned)in_band / (unsigned)height);      // (a division by a number in a register: 0.1 us)
    const long long m0 = (long long)(band * BAND + in_band - column * height) * BM;
    const int n0 = column * BN;
    const int mrows = (int)min((long long)BM, a.rows.M - m0), nrows = min(BN, a.N - n0);
    const int K = a.K, Rp = rank_pad(a.R);

    // this lane's 16 bytes of piece i: row wave * (rows / NW) + 8 i + lane / 8, chunk (lane % 8) ^ ((row >> 1) & 7)
    auto row_of = [&](int i, int rows) __attribute__((always_inline)) { return wave * (rows / NW) + 8 * i + (lane >> 3); };
    auto chunk_of = [&](int row) __attribute__((always_inline)) { return (unsigned)(((lane & 7) ^ ((row >> 1) & 7)) * 8); };
    unsigned a_off[AP], b_off[BP];
#pragma unroll
    for (int i = 0; i < AP; ++i) {
        const int row = row_of(i, BM);
        a_off[i] = row < mrows ? ((unsigned)row * (unsigned)K + chunk_of(row)) * 2u : OOB;
    }
#pragma unroll
    for (int i = 0; i < BP; ++i) {
        const int row = row_of(i, BN);
        b_off[i] = row < nrows ? ((unsigned)row * (unsigned)K + chunk_of(row)) * 2u : OOB;
    }
    const __amdgpu_buffer_rsrc_t xrs = __builtin_amdgcn_make_buffer_rsrc((void*)(a.x + m0 * K), 0, mrows * K * 2, 0x00020000);
    const __amdgpu_buffer_rsrc_t wrs = __builtin_amdgcn_make_buffer_rsrc((void*)(a.w + (long long)n0 * K), 0, nrows * K * 2, 0x00020000);
    const __amdgpu_buffer_rsrc_t urs = __builtin_amdgcn_make_buffer_rsrc((void*)(a.u + m0 * 2 * Rp), 0, mrows * 2 * Rp * 2, 0x00020000);

    auto to_lds = [&](const __amdgpu_buffer_rsrc_t rs, char* to, unsigned off, int soff) __attribute__((always_inline)) {
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (__attribute__((address_space(3))) void*)to, 16, (int)off, soff, 0, 0);
    };
    auto issue_main = [&](int s, int stage) __attribute__((always_inline)) {
        char* base = smem + stage * STAGE;
        const bool ragged = s * 64 + 64 > K;                         // (uniform) the last step of a K that is not whole
#pragma unroll
        for (int i = 0; i < AP; ++i) {
            unsigned off = a_off[i];
            if (ragged && (unsigned)(s * 64) + chunk_of(row_of(i, BM)) >= (unsigned)K) off = OOB;
            to_lds(xrs, base + (wave * (BM / NW) + 8 * i) * ROWB, off, s * 128);
        }
#pragma unroll
        for (int i = 0; i < BP; ++i) {
            unsigned off = b_off[i];
            if (ragged && (unsigned)(s * 64) + chunk_of(row_of(i, BN)) >= (unsigned)K) off = OOB;
            to_lds(wrs, base + A_BYTES + (wave * (BN / NW) + 8 * i) * ROWB, off, s * 128);
        }
    };
    // columns [c0, c0 + 64) of [u_value | u_rest] against the same columns of [B_e | B_e]
    auto issue_low = [&](int e, int c0, int stage) __attribute__((always_inline)) {
        char* base = smem + stage * STAGE;
        const __amdgpu_buffer_rsrc_t brs = __builtin_amdgcn_make_buffer_rsrc((void*)(a.B + ((long long)e * a.N + n0) * a.ldb), 0, nrows * a.ldb * 2, 0x00020000);
#pragma unroll
        for (int i = 0; i < AP; ++i) {
            const int row = row_of(i, BM);
            const unsigned c = (unsigned)c0 + chunk_of(row);
            to_lds(urs, base + (wave * (BM / NW) + 8 * i) * ROWB, row < mrows && c < (unsigned)(2 * Rp) ? ((unsigned)row * (unsigned)(2 * Rp) + c) * 2u : OOB, 0);
        }
#pragma unroll
        for (int i = 0; i < BP; ++i) {
            const int row = row_of(i, BN);
            const unsigned c = (unsigned)c0 + chunk_of(row), r = c >= (unsigned)Rp ? c - (unsigned)Rp : c;
            to_lds(brs, base + A_BYTES + (wave * (BN / NW) + 8 * i) * ROWB,
                   row < nrows && c < (unsigned)(2 * Rp) && r < (unsigned)a.R ? ((unsigned)row * (unsigned)a.ldb + r) * 2u : OOB, 0);
        }
    };

    // Steps run 0 .. steps - 1 over K, then the low-rank columns of the tile's adapters in ascending order.  `issue` requests the next
    // one (NST - 1 ahead of the one being multiplied) and returns whether there was one.
    const int steps = (K + 63) / 64;
    int i_step = 0, i_stage = 0, i_e = kNone, i_c0 = 2 * Rp;
    int only = 0x7fffffff;                                           // the tile's first adapter
    bool mixed = false;                                              // whether its rows differ
    auto issue = [&]() __attribute__((always_inline)) {
        if (i_step < steps) issue_main(i_step, i_stage);
        else {
            if (i_c0 >= 2 * Rp) {
                if (i_e == 0x7fffffff) return false;
                i_e = mixed ? next_adapter<BM>(aid, i_e) : i_e == kNone ? only : 0x7fffffff;
                i_c0 = 0;
                if (i_e == 0x7fffffff) { i_c0 = 2 * Rp; return false; }
            }
            issue_low(i_e, i_c0, i_stage);
            i_c0 += 64;
        }
        ++i_step;
        i_stage = i_stage + 1 == NST ? 0 : i_stage + 1;
        return true;
    };
    issue();                                                         // (the first step of K)
    int ahead = 1;
    static_assert(BM <= NW * 64 && BN <= NW * 64, "a row and a column per thread");
    if (tid < BM) {
        const int e = tid < mrows ? a.who[m0 + tid] : kNone;
        aid[tid] = e;
#if defined(DM_F16)
        const float scale = tid < mrows ? a.us[m0 + tid] : 1.f;
        scale_of[tid] = e != kNone ? scale : 1.f;                    // (us is written where there is an adapter)
#endif
    }
    if (tid < BN) bias_of[tid] = a.bias && tid < nrows ? (float)a.bias[n0 + tid] : 0.f;
    __syncthreads();
    int others = 0;
#pragma unroll
    for (int t = lane; t < BM; t += 64) others |= t < mrows && aid[t] != aid[0];
    mixed = __any(others);
    only = mixed ? next_adapter<BM>(aid, kNone) : aid[0] == kNone ? 0x7fffffff : __builtin_amdgcn_readfirstlane(aid[0]);
#pragma unroll
    for (int q = 1; q < NST; ++q) ahead += issue();                  // (at first the whole ring is free)
    // A tile of one adapter (nearly all: a request is longer than a tile): its low-rank columns are K steps like others
    const bool uniform = only != 0x7fffffff && !mixed;
    f32x16 acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;

    auto frag = [&](const char* base, int row, int kk) __attribute__((always_inline)) {
        return *reinterpret_cast<const elem8*>(base + row * ROWB + (((2 * kk + hi) ^ ((row >> 1) & 7)) << 4));
    };
    int stage = 0;
    // waits until the step to multiply has landed (the younger steps' pieces stay in flight), then requests another one into the stage that
    // all waves have read
    auto advance = [&](bool first) __attribute__((always_inline)) {
        if (ahead == NST) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((NST - 1) * (AP + BP)) : "memory");
        else if (NST > 2 && ahead == NST - 1) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((NST - 2) * (AP + BP)) : "memory");
        else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        --ahead;
        if (!first) ahead += issue();
    };
    // low: the step's columns from Rp on are rests
    auto multiply = [&](bool first, auto low, int c0) __attribute__((always_inline)) {
        advance(first);
        const char* ab = smem + stage * STAGE;
        const char* bb = ab + A_BYTES;
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
            elem8 af[MT], bf[NT];
#pragma unroll
            for (int i = 0; i < MT; ++i) af[i] = frag(ab, TM * wm + 32 * i + l31, kk);
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                bf[j] = frag(bb, TN * wn + 32 * j + l31, kk);
                if constexpr (decltype(low)::value) if (c0 + 16 * kk >= Rp) bf[j] = finite_only(bf[j]);
            }
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int j = 0; j < NT; ++j) acc[i][j] = DM_MFMA_32x32x16(bf[j], af[i], acc[i][j]);
        }
        stage = stage + 1 == NST ? 0 : stage + 1;
    };
    for (int s = 0; s < steps; ++s) multiply(s == 0, std::false_type{}, 0);
    if (uniform) {
        // in units of the row's power of two (exact; a lane's accumulators are one row per i)
        [[maybe_unused]] auto rescale = [&](auto factor) __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                const float f = factor(scale_of[TM * wm + 32 * i + l31]);
#pragma unroll
                for (int j = 0; j < NT; ++j)
#pragma unroll
                    for (int r = 0; r < 16; ++r) acc[i][j][r] *= f;
            }
        };
#if defined(DM_F16)
        rescale([](float p) { return 1.f / p; });
#endif
        for (int c0 = 0; c0 < 2 * Rp; c0 += 64) multiply(false, std::true_type{}, c0);
#if defined(DM_F16)
        rescale([](float p) { return p; });
#endif
    }
    int e = uniform ? 0x7fffffff : only, c0 = 0;
    while (e != 0x7fffffff) {
        advance(false);
        const char* ab = smem + stage * STAGE;
        const char* bb = ab + A_BYTES;
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            const int row = TM * wm + 32 * i + l31;
            const bool mine = aid[row] == e;
#if defined(DM_F16)
            const float scale = scale_of[row];
#else
            constexpr float scale = 1.f;                             // (pow2_scale)
#endif
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                f32x16 t;
#pragma unroll
                for (int r = 0; r < 16; ++r) t[r] = 0.f;
#pragma unroll
                for (int kk = 0; kk < 4; ++kk) {                     // (columns past 2 Rp are zeros)
                    const elem8 bf = frag(bb, TN * wn + 32 * j + l31, kk);
                    t = DM_MFMA_32x32x16(c0 + 16 * kk >= Rp ? finite_only(bf) : bf, frag(ab, row, kk), t);
                }
#pragma unroll
                for (int r = 0; r < 16; ++r) acc[i][j][r] += mine ? t[r] * scale : 0.f;
                __builtin_amdgcn_sched_barrier(0);                   // one fragment at a time: the accumulators leave no registers for more
            }
        }
        stage = stage + 1 == NST ? 0 : stage + 1;
        c0 += 64;
        if (c0 >= 2 * Rp) { c0 = 0; e = next_adapter<BM>(aid, e); }
    }

    // one rounding: y = acc + bias + residual.  Registers 4 g + r hold columns 8 g + 4 hi + r; exchanging group 2 gp + 1 of the lower lanes with
    // group 2 gp of the upper ones leaves lanes 0-31 with columns 16 gp .. + 7 of their row, lanes 32-63 with 16 gp + 8 .. + 15.
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        const long long m = m0 + TM * wm + 32 * i + l31;
        const bool m_ok = m < a.rows.M;
        elem8 res[NT][2];
        if (a.res) {
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int gp = 0; gp < 2; ++gp) {
                    const int n = n0 + TN * wn + 32 * j + 16 * gp + 8 * hi;
                    res[j][gp] = elem8{};
                    if (m_ok && n < a.N) res[j][gp] = *reinterpret_cast<const elem8*>(a.res + m * a.N + n);
                }
        }
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int gp = 0; gp < 2; ++gp) {
                const int col = TN * wn + 32 * j + 16 * gp + 8 * hi, n = n0 + col;
                float v[8];
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float p = acc[i][j][8 * gp + r], q = acc[i][j][8 * gp + 4 + r];
                    const auto sw = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, p), __builtin_bit_cast(unsigned, q), false, false);
                    const unsigned w0 = sw[0], w1 = sw[1];           // (a bit cast of a vector's element would take its first)
                    v[r] = __builtin_bit_cast(float, w0);
                    v[4 + r] = __builtin_bit_cast(float, w1);
                }
                const float4 b0 = *reinterpret_cast<const float4*>(bias_of + col), b1 = *reinterpret_cast<const float4*>(bias_of + col + 4);
                v[0] += b0.x; v[1] += b0.y; v[2] += b0.z; v[3] += b0.w;
                v[4] += b1.x; v[5] += b1.y; v[6] += b1.z; v[7] += b1.w;
                if (a.res)
#pragma unroll
                    for (int r = 0; r < 8; ++r) v[r] += (float)res[j][gp][r];
                elem8 o;
#pragma unroll
                for (int r = 0; r < 8; ++r) o[r] = (elem_t)v[r];
                if (m_ok && n < a.N) *reinterpret_cast<elem8*>(a.y + m * a.N + n) = o;
            }
    }
#endif
}

// M <= 32 rows (single tokens of a few requests): 16 columns per workgroup, eight waves split K and read W straight from memory (each
// element is used once per 16 rows); the low-rank part is one fp32 dot product per output with the row's own adapter.  Bound by the
// W read -- below a few MB by the launch (1280 x 1280 for 16 rows: 5.5-6 us).  Five slices of 256 columns are requested at once: as many as
// 32 rows' fragments leave registers for, and one round trip up to K = 1280.
template <int MT>
__global__ __launch_bounds__(512) void k_expand_skinny(ExpandArgs a, const float* __restrict__ u) {
    __shared__ float part[8][MT * 16][17];
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, l15 = lane & 15, kq = lane >> 4;
    const int n0 = blockIdx.x * 16, K = a.K, M = (int)a.rows.M;
    f32x4 acc[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
    const elem_t* wr = a.w + (long long)min(n0 + l15, a.N - 1) * K + 8 * kq;
    const elem_t* xr[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) xr[t] = a.x + (long long)min(16 * t + l15, M - 1) * K + 8 * kq;
    for (int k0 = 32 * wave; k0 < K; k0 += 256 * 5) {            // five slices requested at once
        elem8 wf[5], xf[MT][5];
        const elem8 zero = {};
#pragma unroll
        for (int q = 0; q < 5; ++q) {
            const int k = k0 + 256 * q;
            const bool ok = k + 8 * kq < K;
            wf[q] = ok ? *reinterpret_cast<const elem8*>(wr + k) : zero;
#pragma unroll
            for (int t = 0; t < MT; ++t) xf[t][q] = ok ? *reinterpret_cast<const elem8*>(xr[t] + k) : zero;
        }
#pragma unroll
        for (int q = 0; q < 5; ++q)
#pragma unroll
            for (int t = 0; t < MT; ++t) acc[t] = DM_MFMA_16x16x32(xf[t][q], wf[q], acc[t]);
    }
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) part[wave][16 * t + 4 * kq + i][l15] = acc[t][i];
    __syncthreads();
    if (tid < MT * 256) {
        const int m = tid >> 4, n = n0 + l15;
        if (m < M && n < a.N) {
            float v = 0.f;
#pragma unroll
            for (int w = 0; w < 8; ++w) v += part[w][m][l15];
            const int e = adapter_of(a.rows, m);
            if (e != kNone) {
                const elem_t* br = a.B + ((long long)e * a.N + n) * a.ldb;
                const float* ur = u + (long long)m * rank_pad(a.R);
                float s = 0.f;
                for (int r = 0; r < a.R; r += 8) {               // (columns of B past R within ldb are zero or absent: u is zero there)
                    const elem8 bv = *reinterpret_cast<const elem8*>(br + r);
#pragma unroll
                    for (int i = 0; i < 8; ++i) s += r + i < a.R ? ur[r + i] * (float)bv[i] : 0.f;
                }
                v += s;
            }
            if (a.bias) v += (float)a.bias[n];
            if (a.res) v += (float)a.res[(long long)m * a.N + n];
            a.y[(long long)m * a.N + n] = (elem_t)v;
        }
    }
}

// ------------------------------------------------------------------------------------------------ layouts of the adapters
// 32 x 32 tiles through LDS.  pad: dst[e][c][0 .. Rp) = src[e][c][0 .. R), zeros behind (B whose rank rows are not whole 16-byte chunks)
__global__ __launch_bounds__(256) void k_adapter_pad(const elem_t* __restrict__ src, elem_t* __restrict__ dst, long long rows, int R, int Rp) {
    for (long long at = (long long)blockIdx.x * 256 + threadIdx.x; at < rows * Rp; at += 256LL * gridDim.x) {
        const long long c = at / Rp;
        const int r = (int)(at - c * Rp);
        dst[at] = r < R ? src[c * R + r] : (elem_t)0.f;
    }
}

// The operands of the data gradient: at [E, K, Rp] = A^T with zeros past R (from A [E, R, K]) and bt [E, R, N] = B^T (from B [E, N, R]).
// blockIdx.x: the column tiles of at (none if at is NULL), then those of bt; y: rank tile; z: adapter.
__global__ __launch_bounds__(256) void k_adapter_transpose(const elem_t* __restrict__ A, const elem_t* __restrict__ B, elem_t* __restrict__ at,
                                                           elem_t* __restrict__ bt, int K, int N, int R, int Rp, int at_tiles) {
    __shared__ elem_t tile[32][34];
    const int r0 = blockIdx.y * 32, tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
    if ((int)blockIdx.x < at_tiles) {
        const int c0 = blockIdx.x * 32;
        const elem_t* s = A + (long long)blockIdx.z * R * K;
        for (int r = ty; r < 32; r += 8) tile[r][tx] = r0 + r < R && c0 + tx < K ? s[(long long)(r0 + r) * K + c0 + tx] : (elem_t)0.f;
        __syncthreads();
        elem_t* d = at + (long long)blockIdx.z * K * Rp;
        for (int c = ty; c < 32; c += 8)
            if (c0 + c < K && r0 + tx < Rp) d[(long long)(c0 + c) * Rp + r0 + tx] = tile[tx][c];
    } else {
        const int n0 = ((int)blockIdx.x - at_tiles) * 32;
        const elem_t* s = B + (long long)blockIdx.z * R * N;
        for (int n = ty; n < 32; n += 8) tile[n][tx] = n0 + n < N && r0 + tx < R ? s[(long long)(n0 + n) * R + r0 + tx] : (elem_t)0.f;
        __syncthreads();
        elem_t* d = bt + (long long)blockIdx.z * R * N;
        for (int r = ty; r < 32; r += 8)
            if (r0 + r < R && n0 + tx < N) d[(long long)(r0 + r) * N + n0 + tx] = tile[tx][r];
    }
}

// ------------------------------------------------------------------------------------------------ weight gradient
// Plan (one workgroup): first[e] = rows of adapters < e, item[e] = row ranges ("items" of `chunk` rows) of adapters < e, and perm =
// the rows in adapter order, ascending inside an adapter (-1: no row; only where offsets do not ascend).  Requests in batches of 1024 through
// LDS; thread e adds up adapter e's.  Every request is walked twice per 1024 adapters: 4 us for a few, 0.15 us each where there are thousands (a
// training step with an id for each of 24576 rows takes 3.9 ms, 0.17 with 24 requests).
__device__ __forceinline__ void request_rows(const Rows& r, int i, long long& lo, long long& hi) {
    lo = r.offsets ? r.offsets[i] : i * r.each;
    hi = r.offsets ? r.offsets[i + 1] : (i + 1) * r.each;
    lo = min(max(lo, 0LL), r.M);
    hi = min(max(hi, lo), r.M);
}

__global__ __launch_bounds__(1024) void k_wgrad_plan(Rows rows, int chunk, int* __restrict__ first, int* __restrict__ item, int* __restrict__ start,
                                                     int* __restrict__ perm) {
    __shared__ int id[1024], len[1024];
    const int tid = threadIdx.x, E = rows.E;
    for (long long m = tid; m < rows.M; m += 1024) perm[m] = kNone;
    // a thousand adapters at a time: their rows, then (one thread, in LDS) the running sums
    int f = 0, it = 0;
    for (int e0 = 0; e0 < E; e0 += 1024) {
        int count = 0;
        for (int b = 0; b < rows.n; b += 1024) {
            __syncthreads();
            if (b + tid < rows.n) {
                long long lo, hi;
                request_rows(rows, b + tid, lo, hi);
                id[tid] = checked(rows.ids[b + tid], E);
                len[tid] = (int)(hi - lo);
            }
            __syncthreads();
            const int n = min(1024, rows.n - b);
            const unsigned most = (unsigned)rows.M;                  // (sums of two stay below 2^32)
#pragma unroll 8
            for (int i = 0; i < n; ++i) count = (int)min(most, (unsigned)count + (id[i] == e0 + tid ? (unsigned)len[i] : 0u));
        }
        __syncthreads();
        id[tid] = count;
        __syncthreads();
        if (tid == 0) {
            for (int e = 0; e < min(1024, E - e0); ++e) {
                const int c = min(id[e], (int)rows.M - f);           // (offsets that do not ascend: never more than M rows)
                it += (c + chunk - 1) / chunk;
                id[e] = f += c;
                len[e] = it;
            }
        }
        __syncthreads();
        if (e0 + tid < E) {
            first[e0 + tid + 1] = id[tid];
            item[e0 + tid + 1] = len[tid];
        }
    }
    if (tid == 0) first[0] = item[0] = 0;
    __syncthreads();
    // start[i] = place of request i's first row
    for (int e0 = 0; e0 < E; e0 += 1024) {
        int at = e0 + tid < E ? first[e0 + tid] : 0;
        for (int b = 0; b < rows.n; b += 1024) {
            __syncthreads();
            if (b + tid < rows.n) {
                long long lo, hi;
                request_rows(rows, b + tid, lo, hi);
                id[tid] = checked(rows.ids[b + tid], E);
                len[tid] = (int)(hi - lo);
            }
            __syncthreads();
            const int n = min(1024, rows.n - b);
#pragma unroll 8
            for (int i = 0; i < n; ++i)
                if (id[i] == e0 + tid) { start[b + i] = at; at = (int)min((unsigned)rows.M, (unsigned)at + (unsigned)len[i]); }
        }
    }
}

// the request of row m (one that adapter_of has found to have an adapter) and its first row
__device__ __forceinline__ int request_of(const Rows& rows, long long m, long long& begin) {
    if (!rows.offsets) {
        const int i = (int)(m / rows.each);
        begin = i * rows.each;
        return i;
    }
    int lo = 0, hi = rows.n;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (rows.offsets[mid + 1] <= m) lo = mid + 1;
        else hi = mid;
    }
    begin = max(rows.offsets[lo], 0);
    return lo;
}

__global__ __launch_bounds__(256) void k_wgrad_perm(Rows rows, const int* __restrict__ start, int* __restrict__ perm) {
    const long long m = (long long)blockIdx.x * 256 + threadIdx.x;
    if (m >= rows.M || adapter_of(rows, m) == kNone) return;
    long long begin;
    const int i = request_of(rows, m, begin);
    const long long at = start[i] + (m - begin);
    if (at < rows.M) perm[at] = (int)m;
}

// Both weight gradients in one launch: dA from (du, x) over K columns, dB from (u, dy) over N.
struct WgradArgs {
    const elem_t *X[2], *u[2];
    const float* us[2];
    float* part[2];
    elem_t* out[2];
    const int *first, *item, *perm;
    int C[2], tiles[2];      // columns, 128-column tiles (0: not wanted)
    int E, R, chunk;
};

// part[item][r < Rp][C] = sum over the item's rows of (value + rest)[m, r] us[m] X[m, c].  Workgroup = one item x 128 columns (a wave 32),
// rows in stages of 64 through LDS (requested a stage ahead), both operands read with the transposing LDS read (the contraction index
// is the row).  The rows of a stage sit at a pitch of 16 or 48 dwords past a multiple of 64: the four rows and two column groups of a
// transposing read hit disjoint banks.  In half precision the pair is rescaled to the item's largest row scale while it is staged.
// Bound by the read of X: [24576, 1280 + 5120] rank 64 in 78 us, 4 TB/s.
template <int Rp>
__global__ __launch_bounds__(256) void k_wgrad(WgradArgs a) {
    constexpr int UC = 2 * Rp, UF = UC / 32;                       // columns of the pair, 32-row fragments
    constexpr int UP = UC == 32 ? 64 : UC * 2 + 64, XP = 320;      // byte pitches
    constexpr int UN = (64 * (Rp / 8) + 255) / 256;                // pair chunks per thread and stage
    __shared__ __attribute__((aligned(16))) char xs[64 * XP];
    __shared__ __attribute__((aligned(16))) char ub[64 * UP];
    [[maybe_unused]] __shared__ float red[4];
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, hi = lane >> 5, l31 = lane & 31;
    const int it = blockIdx.y, side = (int)blockIdx.x >= a.tiles[0];
    if (it >= a.item[a.E]) return;
    const elem_t* X = a.X[side];
    const elem_t* u = a.u[side];
    [[maybe_unused]] const float* us = a.us[side];
    const int C = a.C[side], c0 = ((int)blockIdx.x - (side ? a.tiles[0] : 0)) * 128;
    int lo = 0, up = a.E - 1;                                      // the adapter whose items include `it`
    while (lo < up) {
        const int mid = (lo + up) >> 1;
        if (a.item[mid + 1] <= it) lo = mid + 1;
        else up = mid;
    }
    const int v0 = a.first[lo] + (it - a.item[lo]) * a.chunk, v1 = min(v0 + a.chunk, a.first[lo + 1]);
    float top = 1.f;
#if defined(DM_F16)
    float big = 0.f;
    for (int v = v0 + tid; v < v1; v += 256) big = fmaxf(big, a.perm[v] >= 0 ? us[a.perm[v]] : 0.f);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) big = fmaxf(big, __shfl_xor(big, o, 64));
    if (lane == 0) red[wave] = big;
    __syncthreads();
    top = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    top = top > 0.f ? top : 1.f;
    const float inv = 1.f / top;
#endif
    f32x16 acc[UF];
#pragma unroll
    for (int f = 0; f < UF; ++f)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[f][r] = 0.f;
    const int i16 = lane & 15, g1 = (lane >> 4) & 1;
    // this thread's rows of a stage: x rows tid / 16 + 16 q, pair rows (tid + 256 q) / (Rp / 8)
    int xm[4], um[UN];
    u32x4 xd[4];
    elem8 ph[UN], pl[UN];
    [[maybe_unused]] float pf[UN];
    auto rows_of = [&](int v) __attribute__((always_inline)) {
#pragma unroll
        for (int q = 0; q < 4; ++q) xm[q] = v + (tid >> 4) + 16 * q < v1 ? a.perm[v + (tid >> 4) + 16 * q] : kNone;
#pragma unroll
        for (int q = 0; q < UN; ++q) {
            const int row = (tid + 256 * q) / (Rp / 8);
            um[q] = row < 64 && v + row < v1 ? a.perm[v + row] : kNone;
        }
    };
    const int xc = c0 + (tid & 15) * 8;
    auto load = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            xd[q] = u32x4{0u, 0u, 0u, 0u};
            if (xm[q] >= 0 && xc < C) xd[q] = *reinterpret_cast<const u32x4*>(X + (long long)xm[q] * C + xc);
        }
#pragma unroll
        for (int q = 0; q < UN; ++q) {
            const int c = (tid + 256 * q) % (Rp / 8) * 8;
            ph[q] = elem8{};
            pl[q] = elem8{};
#if defined(DM_F16)
            pf[q] = 0.f;
#endif
            if (um[q] >= 0) {
                ph[q] = *reinterpret_cast<const elem8*>(u + (long long)um[q] * UC + c);
                pl[q] = *reinterpret_cast<const elem8*>(u + (long long)um[q] * UC + Rp + c);
#if defined(DM_F16)
                pf[q] = us[um[q]] * inv;
#endif
            }
        }
    };
    rows_of(v0);
    load();
    rows_of(v0 + 64);
    for (int v = v0; v < v1; v += 64) {
        __syncthreads();
#pragma unroll
        for (int q = 0; q < 4; ++q) *reinterpret_cast<u32x4*>(xs + ((tid >> 4) + 16 * q) * XP + (tid & 15) * 16) = xd[q];
#pragma unroll
        for (int q = 0; q < UN; ++q) {
            const int row = (tid + 256 * q) / (Rp / 8), c = (tid + 256 * q) % (Rp / 8) * 8;
            if (row >= 64) continue;
#if defined(DM_F16)
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const float w = ((float)ph[q][k] + (float)pl[q][k]) * pf[q];
                ph[q][k] = (elem_t)w;
                pl[q][k] = rest_of(w, ph[q][k]);
            }
#endif
            *reinterpret_cast<elem8*>(ub + row * UP + c * 2) = ph[q];
            *reinterpret_cast<elem8*>(ub + row * UP + (Rp + c) * 2) = pl[q];
        }
        __syncthreads();
        if (v + 64 < v1) {
            load();
            rows_of(v + 128);
        }
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) {
            const int row = 16 * ks + 8 * hi + (i16 >> 2), col = 16 * g1 + 4 * (i16 & 3);
            const char* xp = xs + row * XP + (32 * wave + col) * 2;
            const elem4 x0 = dm_ds_read_tr16_b64(xp), x1 = dm_ds_read_tr16_b64(xp + 4 * XP);
            const elem8 xf = {x0[0], x0[1], x0[2], x0[3], x1[0], x1[1], x1[2], x1[3]};
#pragma unroll
            for (int f = 0; f < UF; ++f) {
                const char* pp = ub + row * UP + (32 * f + col) * 2;
                const elem4 u0 = dm_ds_read_tr16_b64(pp), u1 = dm_ds_read_tr16_b64(pp + 4 * UP);
                const elem8 uf = {u0[0], u0[1], u0[2], u0[3], u1[0], u1[1], u1[2], u1[3]};
                acc[f] = DM_MFMA_32x32x16(uf, xf, acc[f]);
            }
        }
    }
    // acc[f]: lane = column, register r = pair column 32 f + (r & 3) + 8 (r >> 2) + 4 hi; value and rest are Rp columns apart
    const int c = c0 + 32 * wave + l31;
    if (c >= C) return;
    float* out = a.part[side] + (long long)it * Rp * C + c;
    auto both = [&](float value, float rest) { return (fabsf(value) <= 3.4028235e38f ? value + rest : value) * top; };      // (an infinite x: the value decides)
    if constexpr (Rp == 16) {
#pragma unroll
        for (int r = 0; r < 8; ++r) out[(long long)((r & 3) + 8 * (r >> 2) + 4 * hi) * C] = both(acc[0][r], acc[0][r + 8]);
    } else {
#pragma unroll
        for (int f = 0; f < UF / 2; ++f)
#pragma unroll
            for (int r = 0; r < 16; ++r) out[(long long)(32 * f + (r & 3) + 8 * (r >> 2) + 4 * hi) * C] = both(acc[f][r], acc[f + UF / 2][r]);
    }
}

// dA[e][r][c] and dB[e][c][r] = the sums of the adapter's items in a fixed order (eight loads in flight), rounded once; an adapter without rows
// gets zeros.  Workgroup = 64 columns x RANKS ranks; blockIdx.x: the column blocks of dA, then those of dB.  RANKS 1: the waves share the
// items.  16: four ranks per wave, stored in runs of 32 bytes on the dB side, whose ranks are adjacent (64 ranks of [1280 + 5120] for 8
// adapters of 3 or 4 items each: 14 us, 27 with one rank per workgroup).
template <int RANKS>
__global__ __launch_bounds__(256) void k_wgrad_join(WgradArgs a, int blocks_a, int Rp) {
    __shared__ float red[RANKS == 1 ? 4 : RANKS][65];
    const int side = (int)blockIdx.x >= blocks_a, C = a.C[side];
    const int e = blockIdx.z, tx = threadIdx.x & 63, q = threadIdx.x >> 6, c0 = ((int)blockIdx.x - (side ? blocks_a : 0)) * 64, c = c0 + tx;
    const int lo = a.item[e], n = a.item[e + 1] - lo;
    if constexpr (RANKS == 1) {
        const int r = blockIdx.y;
        const float* p = a.part[side] + ((long long)lo * Rp + r) * C + c;
        float s = 0.f;
        if (c < C) {
#pragma unroll 8
            for (int i = q; i < n; i += 4) s += p[(long long)i * Rp * C];
        }
        red[q][tx] = s;
        __syncthreads();
        if (q || c >= C) return;
        s = red[0][tx] + red[1][tx] + red[2][tx] + red[3][tx];
        if (side) a.out[1][((long long)e * C + c) * a.R + r] = (elem_t)s;
        else a.out[0][((long long)e * a.R + r) * C + c] = (elem_t)s;
    } else {
        const int r0 = blockIdx.y * RANKS + q * (RANKS / 4);
        const float* p = a.part[side] + ((long long)lo * Rp + r0) * C + c;
        float s[RANKS / 4];
#pragma unroll
        for (int k = 0; k < RANKS / 4; ++k) s[k] = 0.f;
        if (c < C) {
#pragma unroll 2
            for (int i = 0; i < n; ++i)
#pragma unroll
                for (int k = 0; k < RANKS / 4; ++k) s[k] += p[((long long)i * Rp + k) * C];      // (r0 + k < Rp: whole sixteens)
        }
        if (!side) {
#pragma unroll
            for (int k = 0; k < RANKS / 4; ++k)
                if (c < C && r0 + k < a.R) a.out[0][((long long)e * a.R + r0 + k) * C + c] = (elem_t)s[k];
            return;
        }
#pragma unroll
        for (int k = 0; k < RANKS / 4; ++k) red[q * (RANKS / 4) + k][tx] = s[k];
        __syncthreads();
        const int cc = threadIdx.x >> 2, rk = (threadIdx.x & 3) * 4, r1 = blockIdx.y * RANKS + rk;
        if (c0 + cc >= C) return;
        elem_t* to = a.out[1] + ((long long)e * C + c0 + cc) * a.R + r1;
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (r1 + k < a.R) to[k] = (elem_t)red[rk + k][cc];
    }
}

// ------------------------------------------------------------------------------------------------ host side
constexpr long long kMostRows = 1 << 30;        // a grid holds fewer than 2^32 threads: 256 per 64 rows of x A^T, and of a result of up to 64 columns

int check_rows(const int* ids, long long n, long long M, int E, bool offsets) {
    if (!ids || n <= 0 || n > 0x7fffffff || M < 0 || M > 0x7fffffff || E <= 0) return DM_ERR_ARG;
    if (!offsets && (M % n)) return DM_ERR_ARG;
    return M < kMostRows ? DM_OK : DM_ERR_UNSUPPORTED;
}

Rows make_rows(const int* ids, const int* offsets, long long n, long long M, int E) {
    Rows r;
    r.ids = ids; r.offsets = offsets; r.M = M; r.n = (int)n; r.E = E;
    r.each = offsets ? 1 : std::max<long long>(1, M / n);
    return r;
}

constexpr long long kMostBlocks = 1 << 20;      // of a grid whose workgroups loop (a grid holds fewer than 2^32 threads)

// requests shorter than this share a tile with many others: one row at a time then
bool few_rows_each(long long M, long long n) { return M < 8 * n; }

template <int RT, int NR>
void launch_shrink(const elem_t* x, const elem_t* A, const Rows& rows, int K, int R, float scale, elem_t* u, float* us, int* who, hipStream_t stream) {
    hipLaunchKernelGGL((k_shrink<RT, NR>), dim3((unsigned)((rows.M + 16 * RT - 1) / (16 * RT))), dim3(256), 0, stream, x, A, rows, K, R, scale, u, us, who);
}

template <int NR>
int launch_ring(const elem_t* x, const elem_t* A, const Rows& rows, int K, int R, float scale, elem_t* u, float* us, int* who, hipStream_t stream) {
    constexpr int LDS = 4 * (64 + 16 * NR) * 128 + 64 * 4;
    static unsigned long long devices = 0;
    DM_HIP(dm_dynamic_lds(reinterpret_cast<const void*>(&k_shrink_ring<NR>), LDS, devices));
    hipLaunchKernelGGL((k_shrink_ring<NR>), dim3((unsigned)((rows.M + 63) / 64)), dim3(256), LDS, stream, x, A, rows, K, R, scale, u, us, who);
    DM_LAUNCH_CHECK();
    return DM_OK;
}

// Many rows: 64-row tiles through LDS; few: 32 or 16 rows per workgroup, whose waves share K; requests of a few rows: one row each.
int shrink(const elem_t* x, const elem_t* A, const Rows& rows, int K, int R, float scale, elem_t* u, float* us, int* who, hipStream_t stream) {
    if (few_rows_each(rows.M, rows.n)) {
        hipLaunchKernelGGL(k_shrink_rows, dim3((unsigned)std::min(rows.M, kMostBlocks)), dim3(std::min(1024, 64 * R)), 0, stream, x, A, rows, K, R, scale, u, us, who, (float*)nullptr);
        DM_LAUNCH_CHECK();
        return DM_OK;
    }
    const int Rp = rank_pad(R);
    if (rows.M >= 64 * 192) {                                        // (tiles for three quarters of the CUs)
        switch (Rp) {
            case 16: return launch_ring<1>(x, A, rows, K, R, scale, u, us, who, stream);
            case 32: return launch_ring<2>(x, A, rows, K, R, scale, u, us, who, stream);
            case 64: return launch_ring<4>(x, A, rows, K, R, scale, u, us, who, stream);
            default: return launch_ring<8>(x, A, rows, K, R, scale, u, us, who, stream);
        }
    }
    auto go = [&](auto rt_tag) {
        constexpr int RT = decltype(rt_tag)::value;
        switch (Rp) {
            case 16: launch_shrink<RT, 1>(x, A, rows, K, R, scale, u, us, who, stream); break;
            case 32: launch_shrink<RT, 2>(x, A, rows, K, R, scale, u, us, who, stream); break;
            case 64: launch_shrink<RT, 4>(x, A, rows, K, R, scale, u, us, who, stream); break;
            default: launch_shrink<RT, 8>(x, A, rows, K, R, scale, u, us, who, stream); break;
        }
    };
    if (rows.M >= 32 * 256) go(std::integral_constant<int, 2>{});
    else go(std::integral_constant<int, 1>{});
    DM_LAUNCH_CHECK();
    return DM_OK;
}

template <int BM, int BN, int WM, int WN, int NST>
int launch_expand(ExpandArgs a, hipStream_t stream) {
    constexpr int LDS = NST * (BM + BN) * 128 + BM * 8 + BN * 4;
    const long long n_mt = (a.rows.M + BM - 1) / BM;
    a.n_nt = (a.N + BN - 1) / BN;
    if (n_mt * a.n_nt > (1LL << 24) - 8) return DM_ERR_UNSUPPORTED;        // 2^32 threads; past the memory of any result that takes 128 tiles
    a.n_mt = (int)n_mt;
    a.tiles = (int)(n_mt * a.n_nt);
    static unsigned long long devices = 0;
    DM_HIP(dm_dynamic_lds(reinterpret_cast<const void*>(&k_expand<BM, BN, WM, WN, NST>), LDS, devices));
    hipLaunchKernelGGL((k_expand<BM, BN, WM, WN, NST>), dim3((unsigned)((a.tiles + 7) / 8 * 8)), dim3(WM * WN * 64), LDS, stream, a);
    DM_LAUNCH_CHECK();
    return DM_OK;
}

// Tile by the rounds a launch takes: a round of 768 tiles of 64 x 64 (three per CU) takes 0.34 / 0.6 of one of 512 tiles of 128 x 128 (two per
// CU) for 0.37 of the work.  Where every CU gets at most one 64 tile its ring is as deep as LDS allows (both directions of [382, 976, 728]
// 21.6 -> 19.7 us).  (256 x 256 tiles are 6-14 % faster on the bare product, but their accumulators leave no registers for rows
// of several adapters: with spills 850 against 500 us on [24576, 1280, 5120].)
int expand(const ExpandArgs& a, hipStream_t stream) {
    auto rounds = [&](long long t, long long per) { return (double)(((a.rows.M + t - 1) / t * ((a.N + t - 1) / t) + per - 1) / per); };
    if (0.6 * rounds(128, 512) <= 0.34 * rounds(64, 768)) return launch_expand<128, 128, 2, 2, 2>(a, stream);
    if ((a.rows.M + 63) / 64 * ((a.N + 63) / 64) <= 256) return launch_expand<64, 64, 2, 2, 8>(a, stream);
    return launch_expand<64, 64, 2, 2, 3>(a, stream);
}

constexpr long long kSkinny = 32;

long long align256(long long v) { return (v + 255) / 256 * 256; }
long long u_bytes(long long M, int R) { return align256(M * (4LL * rank_pad(R) + 8)); }

int check_product(const Rows& r, const void* x, const void* w, const void* lora_a, const void* lora_b, int K, int N, int R) {
    if (!x || !lora_a || !lora_b || K <= 0 || N <= 0 || R <= 0) return DM_ERR_ARG;
    if (R > kMaxRank || K % 8 || N % 8 || K > (1 << 20) || N > (1 << 20) || r.E > 65535) return DM_ERR_UNSUPPORTED;
    if (((uintptr_t)x | (uintptr_t)w | (uintptr_t)lora_a | (uintptr_t)lora_b) & 15) return DM_ERR_ARG;
    return DM_OK;
}

// row ranges of the weight gradients: enough workgroups to fill the chip (four per CU over the 128-column tiles of both), but whole 64-row
// stages and few partial sums
int wgrad_chunk(long long M, int K, int N) { return (int)std::max<long long>(128, (M * ((K + N + 127) / 128) / 1024 + 63) / 64 * 64); }
// the most row ranges: full ones, and one that ends early for every adapter that a request can name
long long wgrad_items(long long M, int E, long long n, int chunk) { return std::min<long long>(M, M / chunk + std::min<long long>(E, n)); }

}  // namespace

extern "C" {

#if !defined(DM_F16)
// bytes of the forward's workspace: u as pairs of 16-bit columns, one fp32 scale and one adapter per row, then B with padded rank rows where R % 8 != 0
size_t dm_linear_adapted_workspace_bytes(long long M, int N, int R, int E) {
    if (M <= 0 || N <= 0 || R <= 0 || R > kMaxRank || E <= 0) return 0;
    return (size_t)(u_bytes(M, R) + (R % 8 ? 2LL * E * N * rank_pad(R) : 0));
}

// bytes of the backward's: du, A^T, B^T, the plan (first | item | start | perm) and the weight gradients' partial sums
size_t dm_linear_adapted_bwd_workspace_bytes(long long M, int K, int N, int R, int E, long long n) {
    if (M <= 0 || K <= 0 || N <= 0 || R <= 0 || R > kMaxRank || E <= 0 || n <= 0) return 0;
    const int Rp = rank_pad(R);
    return (size_t)(u_bytes(M, R) + align256(2LL * E * K * Rp) + align256(2LL * E * N * R) + align256(4 * (2LL * (E + 1) + n + M)) +
                    4LL * wgrad_items(M, E, n, wgrad_chunk(M, K, N)) * Rp * (K + N));
}
#endif

// y = x W^T + bias + s (x A_e^T) B_e^T + residual, see the head of this file.  x [M, K], w [N, K], bias [N] or NULL, residual [M, N] or
// NULL, lora_a [E, R, K], lora_b [E, N, R], ids [n] int32, offsets [n + 1] int32 or NULL (then M % n == 0), ws of
// dm_linear_adapted_workspace_bytes; keep_u != 0: u is left at its head for dm_linear_adapted_bwd_*.  K % 8 == N % 8 == 0, R <= 128.
int DM_T(dm_linear_adapted_, )(const void* x, const void* w, const void* bias, const void* residual, const void* lora_a, const void* lora_b, const int* ids,
                               const int* offsets, long long n, float scale, void* ws, size_t ws_bytes, void* y, long long M, int K, int N, int R, int E,
                               int keep_u, hipStream_t stream) {
    if (int rc = check_rows(ids, n, M, E, offsets != nullptr)) return rc;
    const Rows rows = make_rows(ids, offsets, n, M, E);
    if (int rc = check_product(rows, x, w, lora_a, lora_b, K, N, R)) return rc;
    if (!w || !ws || !y || (((uintptr_t)bias | (uintptr_t)residual | (uintptr_t)ws | (uintptr_t)y) & 15)) return DM_ERR_ARG;
    if (M == 0) return DM_OK;
    const int Rp = rank_pad(R);
    if ((long long)ws_bytes < u_bytes(M, R) + (R % 8 ? 2LL * E * N * Rp : 0)) return DM_ERR_WORKSPACE;
    ExpandArgs a{};
    a.x = (const elem_t*)x; a.w = (const elem_t*)w; a.bias = (const elem_t*)bias; a.res = (const elem_t*)residual;
    a.u = (const elem_t*)ws; a.us = (const float*)((const elem_t*)ws + M * 2 * Rp); a.who = (const int*)(a.us + M); a.B = (const elem_t*)lora_b; a.y = (elem_t*)y;
    a.rows = rows;
    a.K = K; a.N = N; a.R = R; a.ldb = R;
    DM_ENTER();
    if (R % 8) {
        elem_t* padded = (elem_t*)((char*)ws + u_bytes(M, R));
        hipLaunchKernelGGL(k_adapter_pad, dim3((unsigned)std::min(((long long)E * N * Rp + 255) / 256, kMostBlocks)), dim3(256), 0, stream, a.B, padded, (long long)E * N, R, Rp);
        a.B = padded;
        a.ldb = Rp;
    }
    if (M <= kSkinny && !keep_u) {
        float* uf = (float*)ws;
        hipLaunchKernelGGL(k_shrink_rows, dim3((unsigned)M), dim3(std::min(1024, 64 * R)), 0, stream, a.x, (const elem_t*)lora_a, a.rows, K, R, scale,
                           (elem_t*)nullptr, (float*)nullptr, (int*)nullptr, uf);
        const dim3 grid((unsigned)((N + 15) / 16));
        if (M <= 16) hipLaunchKernelGGL(k_expand_skinny<1>, grid, dim3(512), 0, stream, a, uf);
        else hipLaunchKernelGGL(k_expand_skinny<2>, grid, dim3(512), 0, stream, a, uf);
        DM_LAUNCH_CHECK();
        return DM_OK;
    }
    if (int rc = shrink(a.x, (const elem_t*)lora_a, a.rows, K, R, scale, (elem_t*)ws, const_cast<float*>(a.us), const_cast<int*>(a.who), stream)) return rc;
    return expand(a, stream);
}

// The gradients: dx [M, K] = dy W + s (dy B_e) A_e (w_t = W^T [K, N]), da [E, R, K], db [E, N, R]; each may be NULL (not wanted).  u = the
// forward's workspace with keep_u (needed for db).
int DM_T(dm_linear_adapted_bwd_, )(const void* x, const void* dy, const void* w_t, const void* lora_a, const void* lora_b, const int* ids, const int* offsets,
                                   long long n, float scale, const void* u, void* ws, size_t ws_bytes, void* dx, void* da, void* db, long long M, int K, int N,
                                   int R, int E, hipStream_t stream) {
    if (int rc = check_rows(ids, n, M, E, offsets != nullptr)) return rc;
    const Rows rows = make_rows(ids, offsets, n, M, E);
    if (int rc = check_product(rows, x, w_t, lora_a, lora_b, K, N, R)) return rc;
    if (!dy || !ws || M == 0 || (dx && !w_t) || (db && !u) || (((uintptr_t)dy | (uintptr_t)u | (uintptr_t)ws | (uintptr_t)dx) & 15)) return DM_ERR_ARG;
    const int Rp = rank_pad(R), chunk = wgrad_chunk(M, K, N);
    const long long items = wgrad_items(M, E, n, chunk);
    if (items > 65535) return DM_ERR_UNSUPPORTED;
    if ((long long)ws_bytes < u_bytes(M, R) + align256(2LL * E * K * Rp) + align256(2LL * E * N * R) + align256(4 * (2LL * (E + 1) + n + M)) + 4LL * items * Rp * (K + N))
        return DM_ERR_WORKSPACE;
    char* p = (char*)ws;
    auto take = [&](long long bytes) { char* q = p; p += align256(bytes); return q; };
    elem_t* du = (elem_t*)take(u_bytes(M, R));
    float* dus = (float*)(du + M * 2 * Rp);
    elem_t* at = (elem_t*)take(2LL * E * K * Rp);
    elem_t* bt = (elem_t*)take(2LL * E * N * R);
    int* plan = (int*)take(4 * (2LL * (E + 1) + n + M));
    float* part = (float*)p;
    DM_ENTER();
    if (dx || da) {
        const int at_tiles = dx ? (K + 31) / 32 : 0;
        hipLaunchKernelGGL(k_adapter_transpose, dim3((unsigned)(at_tiles + (N + 31) / 32), (unsigned)((Rp + 31) / 32), (unsigned)E), dim3(256), 0, stream,
                           (const elem_t*)lora_a, (const elem_t*)lora_b, at, bt, K, N, R, Rp, at_tiles);
        if (int rc = shrink((const elem_t*)dy, bt, rows, N, R, scale, du, dus, (int*)(dus + M), stream)) return rc;
    }
    if (dx) {
        ExpandArgs a{};
        a.x = (const elem_t*)dy; a.w = (const elem_t*)w_t; a.u = du; a.us = dus; a.who = (const int*)(dus + M); a.B = at; a.y = (elem_t*)dx; a.rows = rows;
        a.K = N; a.N = K; a.R = R; a.ldb = Rp;
        if (int rc = expand(a, stream)) return rc;
    }
    if (da || db) {
        int *first = plan, *item = first + E + 1, *start = item + E + 1, *perm = start + n;
        hipLaunchKernelGGL(k_wgrad_plan, dim3(1), dim3(1024), 0, stream, rows, chunk, first, item, start, perm);
        hipLaunchKernelGGL(k_wgrad_perm, dim3((unsigned)((M + 255) / 256)), dim3(256), 0, stream, rows, start, perm);
        WgradArgs g{};
        g.X[0] = (const elem_t*)x; g.u[0] = du; g.us[0] = dus; g.C[0] = K; g.out[0] = (elem_t*)da; g.part[0] = part;
        g.X[1] = (const elem_t*)dy; g.u[1] = (const elem_t*)u; g.us[1] = (const float*)((const elem_t*)u + M * 2 * Rp); g.C[1] = N; g.out[1] = (elem_t*)db;
        g.part[1] = part + items * Rp * K;
        g.tiles[0] = da ? (K + 127) / 128 : 0;
        g.tiles[1] = db ? (N + 127) / 128 : 0;
        g.first = first; g.item = item; g.perm = perm; g.E = E; g.R = R; g.chunk = chunk;
        const dim3 grid((unsigned)(g.tiles[0] + g.tiles[1]), (unsigned)items);
        switch (Rp) {
            case 16: hipLaunchKernelGGL(k_wgrad<16>, grid, dim3(256), 0, stream, g); break;
            case 32: hipLaunchKernelGGL(k_wgrad<32>, grid, dim3(256), 0, stream, g); break;
            case 64: hipLaunchKernelGGL(k_wgrad<64>, grid, dim3(256), 0, stream, g); break;
            default: hipLaunchKernelGGL(k_wgrad<128>, grid, dim3(256), 0, stream, g); break;
        }
        const int ba = da ? (K + 63) / 64 : 0, bb = db ? (N + 63) / 64 : 0;
        // 16 ranks per workgroup where adapters have few items and that leaves two workgroups per CU
        if (items <= 8LL * E && (long long)(ba + bb) * ((R + 15) / 16) * E >= 512)
            hipLaunchKernelGGL(k_wgrad_join<16>, dim3((unsigned)(ba + bb), (unsigned)((R + 15) / 16), (unsigned)E), dim3(256), 0, stream, g, ba, Rp);
        else hipLaunchKernelGGL(k_wgrad_join<1>, dim3((unsigned)(ba + bb), (unsigned)R, (unsigned)E), dim3(256), 0, stream, g, ba, Rp);
        DM_LAUNCH_CHECK();
    }
    return DM_OK;
}

}  // extern "C"
