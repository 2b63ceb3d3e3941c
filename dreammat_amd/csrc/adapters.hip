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
//           scaled by a power of two first (its largest entry near 2^8): half's exponent range must not bound u.
//   expand  the big product, its K loop extended by [u_value | u_rest] [B | B]^T: the low-rank product costs 2 ceil(R/16) 16
//           columns of K and no pass over y.  Rows of a tile that belong to another adapter are left out by selection (never by
//           a multiplication with zero: 0 * inf of another request's adapter would reach them).
//   wgrad   dA_e = du^T x and dB_e = dy^T u over the rows of e, rows gathered in adapter order, split over row ranges and joined in
//           a fixed order (no atomics).
// The data gradient is the same pair of kernels on (dy, W^T, B^T, A^T): dx = dy W + (s dy B_e) A_e.
#include <algorithm>

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
    // 2^k with |u| / 2^k in [2^8, 2^9): half's value and remainder both stay normal; 1 for a row of zeros, infinities or NaN
    if (!(biggest > 0.f) || biggest > 3.0e38f) return 1.f;
    int e;
    frexpf(biggest, &e);
    return ldexpf(1.f, min(max(e - 9, -100), 100));
#else
    return 1.f;
#endif
}

// ------------------------------------------------------------------------------------------------ shrink
// u rows are stored [value: Rp | rest: Rp] elem_t (Rp = rank_pad(R), columns past R zero) with us[m] = the row's power of two.
__device__ __forceinline__ void store_pair(elem_t* u, int Rp, int r, float v) {
    const elem_t hi = (elem_t)v;
    u[r] = hi;
    u[Rp + r] = (elem_t)(v - (float)hi);
}

// Tile of 16 RT rows; the four waves take 64-wide slices of K in turn, so a tile reads its x rows once (128-byte lines) and the rank
// rows of A once from L2; the partial products meet in LDS.  One pass per adapter that occurs in the tile.  Bound by the x read.
template <int RT, int NR>
__global__ __launch_bounds__(256) void k_shrink(const elem_t* __restrict__ x, const elem_t* __restrict__ A, Rows rows, int K, int R, float scale,
                                                elem_t* __restrict__ u, float* __restrict__ us) {
    constexpr int TR = 16 * RT, Rp = 16 * NR;
    __shared__ float part[4][TR][Rp + 1];
    __shared__ int aid[TR];
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, l15 = lane & 15, kq = lane >> 4;
    const long long m0 = (long long)blockIdx.x * TR;
    if (tid < TR) aid[tid] = adapter_of(rows, m0 + tid);
    __syncthreads();
    const elem_t* xr[RT];
#pragma unroll
    for (int t = 0; t < RT; ++t) xr[t] = x + min(m0 + 16 * t + l15, rows.M - 1) * K + 8 * kq;
    int cur = kNone;
    for (;;) {
        int next = 0x7fffffff;                              // the next adapter of the tile, found by every thread alike
        for (int t = 0; t < TR; ++t) {
            const int v = aid[t];
            next = v > cur && v < next ? v : next;
        }
        if (next == 0x7fffffff) break;
        cur = next;
        const elem_t* ar = A + (long long)cur * R * K + 8 * kq;
        f32x4 acc[RT][NR];
#pragma unroll
        for (int t = 0; t < RT; ++t)
#pragma unroll
            for (int q = 0; q < NR; ++q) acc[t][q] = f32x4{0.f, 0.f, 0.f, 0.f};
        for (int k0 = 64 * wave; k0 < K; k0 += 256) {
            elem8 xf[2][RT], af[2][NR];
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                const int k = k0 + 32 * s;
                const bool ok = k + 8 * kq < K;
                const elem8 zero = {};
#pragma unroll
                for (int t = 0; t < RT; ++t) xf[s][t] = ok ? *reinterpret_cast<const elem8*>(xr[t] + k) : zero;
#pragma unroll
                for (int q = 0; q < NR; ++q) af[s][q] = ok ? *reinterpret_cast<const elem8*>(ar + (long long)min(16 * q + l15, R - 1) * K + k) : zero;
            }
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int t = 0; t < RT; ++t)
#pragma unroll
                    for (int q = 0; q < NR; ++q) acc[t][q] = DM_MFMA_16x16x32(xf[s][t], af[s][q], acc[t][q]);
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
                big = fmaxf(big, fabsf(v[q]));
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

// One row per blockIdx.x, one rank row per wave: requests of a few rows each, where a tile would hold many adapters.  Every row reads
// its own adapter (R K 2 bytes).  f32out: plain fp32 [M][Rp] for the skinny product, else the pair format.
__global__ __launch_bounds__(1024) void k_shrink_rows(const elem_t* __restrict__ x, const elem_t* __restrict__ A, Rows rows, int K, int R, float scale,
                                                      elem_t* __restrict__ u, float* __restrict__ us, float* __restrict__ f32out) {
    __shared__ float row[kMaxRank];
    const long long m = blockIdx.x;
    const int tid = threadIdx.x, lane = tid & 63, Rp = rank_pad(R);
    const int e = adapter_of(rows, m);
    if (e == kNone) return;
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
        return;
    }
    float big = 0.f;
    for (int r = 0; r < R; ++r) big = fmaxf(big, fabsf(row[r]));
    const float p = pow2_scale(big);
    for (int r = tid; r < Rp; r += blockDim.x) store_pair(u + m * 2 * Rp, Rp, r, r < R ? row[r] / p : 0.f);
    if (tid == 0) us[m] = p;
}

// ------------------------------------------------------------------------------------------------ expand
struct ExpandArgs {
    const elem_t *x, *w, *bias, *res, *u, *B;
    const float* us;
    elem_t* y;
    Rows rows;
    int K, N, R, ldb;      // ldb: elements between the rows of B (a multiple of 8)
    int n_nt, tiles;
};

// BM x BN x 64 tile, WM x WN waves of 64 x 64, two LDS stages filled by buffer_load ... lds (16 bytes per lane, range-checked: rows and
// columns past the end read as zeros).  LDS rows are 128 bytes, the 16-byte chunks XOR-swizzled by (row >> 1) & 7 at the source address
// and at the fragment read: conflict-free without padding.  The weights are the matrix instruction's A operand, so a lane holds one row
// of y and four consecutive columns per register group: 16-byte stores after one exchange between the wave's halves.
template <int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(WM * WN * 64) void k_expand(ExpandArgs a) {
    [[maybe_unused]] constexpr int NW = WM * WN, ROWB = 128;
    [[maybe_unused]] constexpr int TM = BM / WM, TN = BN / WN, MT = TM / 32, NT = TN / 32;
    [[maybe_unused]] constexpr int A_BYTES = BM * ROWB, STAGE = (BM + BN) * ROWB;
    [[maybe_unused]] constexpr int AP = BM / 8 / NW, BP = BN / 8 / NW;                // 1 KB pieces (8 rows) per wave
    extern __shared__ __attribute__((aligned(16))) char smem[];      // 2 STAGE | int aid[BM]
#if defined(__HIP_DEVICE_COMPILE__)
    constexpr unsigned OOB = 0xfffffff0u;
    int* aid = reinterpret_cast<int*>(smem + 2 * STAGE);
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, hi = lane >> 5, l31 = lane & 31;
    const int wm = wave / WN, wn = wave % WN;
    // block b runs on XCD b % 8 (its own L2): each XCD gets a contiguous run of tiles, the N tiles of one row panel side by side
    const int per = (a.tiles + 7) / 8, id = (int)(blockIdx.x & 7) * per + (int)(blockIdx.x >> 3);
    if ((int)(blockIdx.x >> 3) >= per || id >= a.tiles) return;
    const long long m0 = (long long)(id / a.n_nt) * BM;
    const int n0 = id % a.n_nt * BN;
    const int mrows = (int)min((long long)BM, a.rows.M - m0), nrows = min(BN, a.N - n0);
    const int K = a.K, Rp = rank_pad(a.R);

    const int lrow = lane >> 3, slot = lane & 7;
    unsigned a_off[AP], b_off[BP], a_chunk[AP], b_chunk[BP];
#pragma unroll
    for (int i = 0; i < AP; ++i) {
        const int row = wave * (BM / NW) + 8 * i + lrow;
        a_chunk[i] = (unsigned)((slot ^ ((row >> 1) & 7)) * 8);
        a_off[i] = row < mrows ? (unsigned)row : OOB;
    }
#pragma unroll
    for (int i = 0; i < BP; ++i) {
        const int row = wave * (BN / NW) + 8 * i + lrow;
        b_chunk[i] = (unsigned)((slot ^ ((row >> 1) & 7)) * 8);
        b_off[i] = row < nrows ? (unsigned)row : OOB;
    }
    const __amdgpu_buffer_rsrc_t xrs = __builtin_amdgcn_make_buffer_rsrc((void*)(a.x + m0 * K), 0, mrows * K * 2, 0x00020000);
    const __amdgpu_buffer_rsrc_t wrs = __builtin_amdgcn_make_buffer_rsrc((void*)(a.w + (long long)n0 * K), 0, nrows * K * 2, 0x00020000);
    const __amdgpu_buffer_rsrc_t urs = __builtin_amdgcn_make_buffer_rsrc((void*)(a.u + m0 * 2 * Rp), 0, mrows * 2 * Rp * 2, 0x00020000);

    auto issue_main = [&](int s, int stage) __attribute__((always_inline)) {
        char* base = smem + stage * STAGE;
#pragma unroll
        for (int i = 0; i < AP; ++i) {
            const unsigned k = (unsigned)(s * 64) + a_chunk[i];
            const unsigned off = a_off[i] != OOB && k < (unsigned)K ? (a_off[i] * (unsigned)K + k) * 2u : OOB;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(xrs, (__attribute__((address_space(3))) void*)(base + (wave * (BM / NW) + 8 * i) * ROWB), 16, (int)off, 0, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < BP; ++i) {
            const unsigned k = (unsigned)(s * 64) + b_chunk[i];
            const unsigned off = b_off[i] != OOB && k < (unsigned)K ? (b_off[i] * (unsigned)K + k) * 2u : OOB;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(wrs, (__attribute__((address_space(3))) void*)(base + A_BYTES + (wave * (BN / NW) + 8 * i) * ROWB), 16, (int)off, 0, 0, 0);
        }
    };
    // columns [c0, c0 + 64) of [u_value | u_rest] against the same columns of [B_e | B_e]
    auto issue_low = [&](int e, int c0, int stage) __attribute__((always_inline)) {
        char* base = smem + stage * STAGE;
        const __amdgpu_buffer_rsrc_t brs = __builtin_amdgcn_make_buffer_rsrc((void*)(a.B + ((long long)e * a.N + n0) * a.ldb), 0, nrows * a.ldb * 2, 0x00020000);
#pragma unroll
        for (int i = 0; i < AP; ++i) {
            const unsigned c = (unsigned)c0 + a_chunk[i];
            const unsigned off = a_off[i] != OOB && c < (unsigned)(2 * Rp) ? (a_off[i] * (unsigned)(2 * Rp) + c) * 2u : OOB;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(urs, (__attribute__((address_space(3))) void*)(base + (wave * (BM / NW) + 8 * i) * ROWB), 16, (int)off, 0, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < BP; ++i) {
            const unsigned c = (unsigned)c0 + b_chunk[i], r = c >= (unsigned)Rp ? c - (unsigned)Rp : c;
            const unsigned off = b_off[i] != OOB && c < (unsigned)(2 * Rp) && r < (unsigned)a.R ? (b_off[i] * (unsigned)a.ldb + r) * 2u : OOB;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(brs, (__attribute__((address_space(3))) void*)(base + A_BYTES + (wave * (BN / NW) + 8 * i) * ROWB), 16, (int)off, 0, 0, 0);
        }
    };

    issue_main(0, 0);
    for (int t = tid; t < BM; t += NW * 64) aid[t] = adapter_of(a.rows, m0 + t);
    __syncthreads();
    int my_aid[MT];
    float my_us[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        const int row = TM * wm + 32 * i + l31;
        my_aid[i] = aid[row];
        my_us[i] = my_aid[i] != kNone ? a.us[m0 + row] : 0.f;
    }
    // the tile's adapters in ascending order: every wave finds the next one for itself
    auto next_adapter = [&](int cur) __attribute__((always_inline)) {
        int next = 0x7fffffff;
#pragma unroll
        for (int t = 0; t < BM / 64; ++t) {
            const int v = aid[64 * t + lane];
            next = v > cur && v < next ? v : next;
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) next = min(next, __shfl_xor(next, o, 64));
        return __builtin_amdgcn_readfirstlane(next);
    };

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
    const int steps = (K + 63) / 64;
    int e = next_adapter(kNone);                    // adapter of the low-rank step to issue next (INT_MAX: none left)
    for (int s = 0; s < steps; ++s) {
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        if (s + 1 < steps) issue_main(s + 1, (s + 1) & 1);
        else if (e != 0x7fffffff) issue_low(e, 0, (s + 1) & 1);
        const char* ab = smem + (s & 1) * STAGE;
        const char* bb = ab + A_BYTES;
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
            elem8 af[MT], bf[NT];
#pragma unroll
            for (int i = 0; i < MT; ++i) af[i] = frag(ab, TM * wm + 32 * i + l31, kk);
#pragma unroll
            for (int j = 0; j < NT; ++j) bf[j] = frag(bb, TN * wn + 32 * j + l31, kk);
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int j = 0; j < NT; ++j) acc[i][j] = DM_MFMA_32x32x16(bf[j], af[i], acc[i][j]);
        }
    }
    int s = steps, c0 = 0;
    while (e != 0x7fffffff) {
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        const int cur = e, cols = min(64, 2 * Rp - c0);
        c0 += 64;
        if (c0 >= 2 * Rp) { c0 = 0; e = next_adapter(e); }
        if (e != 0x7fffffff) issue_low(e, c0, (s + 1) & 1);
        const char* ab = smem + (s & 1) * STAGE;
        const char* bb = ab + A_BYTES;
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            const bool mine = my_aid[i] == cur;
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                f32x16 t;
#pragma unroll
                for (int r = 0; r < 16; ++r) t[r] = 0.f;
                for (int kk = 0; 16 * kk < cols; ++kk)
                    t = DM_MFMA_32x32x16(frag(bb, TN * wn + 32 * j + l31, kk), frag(ab, TM * wm + 32 * i + l31, kk), t);
#pragma unroll
                for (int r = 0; r < 16; ++r) acc[i][j][r] += mine ? t[r] * my_us[i] : 0.f;
            }
        }
        ++s;
    }

    // one rounding: y = acc + bias + residual
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        const long long m = m0 + TM * wm + 32 * i + l31;
        const bool m_ok = m < a.rows.M;
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int gp = 0; gp < 2; ++gp) {
                unsigned pk[2][2];
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                    const int g = 2 * gp + q, n = n0 + TN * wn + 32 * j + 8 * g + 4 * hi;      // this lane's four columns
                    float v[4];
#pragma unroll
                    for (int r = 0; r < 4; ++r) v[r] = acc[i][j][4 * g + r];
                    if (a.bias && n < a.N) {
                        const elem4 bv = *reinterpret_cast<const elem4*>(a.bias + n);
#pragma unroll
                        for (int r = 0; r < 4; ++r) v[r] += (float)bv[r];
                    }
                    if (a.res && n < a.N && m_ok) {
                        const elem4 rv = *reinterpret_cast<const elem4*>(a.res + m * a.N + n);
#pragma unroll
                        for (int r = 0; r < 4; ++r) v[r] += (float)rv[r];
                    }
                    const elem4 o = {(elem_t)v[0], (elem_t)v[1], (elem_t)v[2], (elem_t)v[3]};
                    const u32x2 w2 = __builtin_bit_cast(u32x2, o);
                    pk[q][0] = w2[0];
                    pk[q][1] = w2[1];
                }
                // lanes 0-31 get columns 16 gp .. + 7 of their row, lanes 32-63 columns 16 gp + 8 .. + 15
                const auto s0 = __builtin_amdgcn_permlane32_swap(pk[0][0], pk[1][0], false, false);
                const auto s1 = __builtin_amdgcn_permlane32_swap(pk[0][1], pk[1][1], false, false);
                const u32x4 out = {s0[0], s1[0], s0[1], s1[1]};
                const int n = n0 + TN * wn + 32 * j + 16 * gp + 8 * hi;
                if (m_ok && n < a.N) *reinterpret_cast<u32x4*>(a.y + m * a.N + n) = out;
            }
    }
#endif
}

// M <= 32 rows (single tokens of a few requests): 16 columns per workgroup, eight waves split K and read W straight from memory (each
// element is used once per 16 rows); the low-rank part is one fp32 dot product per output with the row's own adapter.  Bound by the
// W read -- below a few MB by the launch.
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
    for (int k = 32 * wave; k < K; k += 256) {
        const bool ok = k + 8 * kq < K;
        const elem8 zero = {};
        const elem8 wf = ok ? *reinterpret_cast<const elem8*>(wr + k) : zero;
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            const elem8 xf = ok ? *reinterpret_cast<const elem8*>(xr[t] + k) : zero;
            acc[t] = DM_MFMA_16x16x32(xf, wf, acc[t]);
        }
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
// dst[e][c][0 .. Rp) = src[e][0 .. R)[c] (transpose: A^T from A; src [E, R, C]) or src[e][c][0 .. R) (copy: B into padded rows, src
// [E, C, R]); columns past R are zero.  32 x 32 tiles through LDS; blockIdx = (column tile, rank tile, adapter).
__global__ __launch_bounds__(256) void k_adapter_rows(const elem_t* __restrict__ src, elem_t* __restrict__ dst, int C, int R, int Rp, int transpose) {
    __shared__ elem_t tile[32][34];
    const int c0 = blockIdx.x * 32, r0 = blockIdx.y * 32, tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
    const elem_t* s = src + (long long)blockIdx.z * R * C;
    elem_t* d = dst + (long long)blockIdx.z * C * Rp;
    if (transpose) {
        for (int r = ty; r < 32; r += 8) tile[r][tx] = r0 + r < R && c0 + tx < C ? s[(long long)(r0 + r) * C + c0 + tx] : (elem_t)0.f;
        __syncthreads();
    }
    for (int c = ty; c < 32; c += 8)
        if (c0 + c < C && r0 + tx < Rp)
            d[(long long)(c0 + c) * Rp + r0 + tx] = transpose ? tile[tx][c] : r0 + tx < R ? s[(long long)(c0 + c) * R + r0 + tx] : (elem_t)0.f;
}

// dst[e][r][n] = src[e][n][r] for r < R: B^T rows of the data gradient's shrink
__global__ __launch_bounds__(256) void k_adapter_cols(const elem_t* __restrict__ src, elem_t* __restrict__ dst, int N, int R) {
    __shared__ elem_t tile[32][34];
    const int n0 = blockIdx.x * 32, r0 = blockIdx.y * 32, tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
    const elem_t* s = src + (long long)blockIdx.z * R * N;
    elem_t* d = dst + (long long)blockIdx.z * R * N;
    for (int n = ty; n < 32; n += 8) tile[n][tx] = n0 + n < N && r0 + tx < R ? s[(long long)(n0 + n) * R + r0 + tx] : (elem_t)0.f;
    __syncthreads();
    for (int r = ty; r < 32; r += 8)
        if (r0 + r < R && n0 + tx < N) d[(long long)(r0 + r) * N + n0 + tx] = tile[tx][r];
}

// ------------------------------------------------------------------------------------------------ weight gradient
// Plan (one workgroup): first[e] = rows of adapters < e, item[e] = row ranges ("items" of `chunk` rows) of adapters < e, and perm =
// the rows in adapter order, ascending inside an adapter (-1: no row; only where offsets do not ascend).  Requests in batches of 1024 through LDS; thread e adds up adapter e's.
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
    // counts into first[e + 1]
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
            for (int i = 0; i < n; ++i) count = (int)min(rows.M, (long long)count + (id[i] == e0 + tid ? len[i] : 0));
        }
        if (e0 + tid < E) first[e0 + tid + 1] = count;
    }
    __syncthreads();
    if (tid == 0) {
        int f = 0, it = 0;
        first[0] = item[0] = 0;
        for (int e = 0; e < E; ++e) {
            const int c = min(first[e + 1], (int)rows.M - f);       // (offsets that do not ascend: never more than M rows)
            it += (c + chunk - 1) / chunk;
            first[e + 1] = f += c;
            item[e + 1] = it;
        }
    }
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
            for (int i = 0; i < n; ++i)
                if (id[i] == e0 + tid) { start[b + i] = at; at = (int)min(rows.M, (long long)at + len[i]); }
        }
    }
}

__global__ __launch_bounds__(256) void k_wgrad_perm(Rows rows, const int* __restrict__ start, int* __restrict__ perm) {
    const long long m = (long long)blockIdx.x * 256 + threadIdx.x;
    if (m >= rows.M) return;
    if (adapter_of(rows, m) == kNone) return;
    int lo = 0, hi = rows.n;
    long long begin;
    if (rows.offsets) {
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (rows.offsets[mid + 1] <= m) lo = mid + 1;
            else hi = mid;
        }
        begin = max(rows.offsets[lo], 0);
    } else {
        lo = (int)(m / rows.each);
        begin = lo * rows.each;
    }
    const long long at = start[lo] + (m - begin);
    if (at < rows.M) perm[at] = (int)m;
}

// part[item][r < Rp][C] = sum over the item's rows of (value + rest)[m, r] us[m] X[m, c].  Workgroup = one item x 128 columns (a wave 32),
// rows in stages of 64 through LDS, both operands read with the transposing LDS read (the contraction index is the row).  The rows of a
// stage sit at a pitch of 16 or 48 dwords past a multiple of 64: the four rows and two column groups of a transposing read hit
// disjoint banks.  In half precision the pair is rescaled to the item's largest row scale while it is staged.
template <int Rp>
__global__ __launch_bounds__(256) void k_wgrad(const elem_t* __restrict__ X, const elem_t* __restrict__ u, const float* __restrict__ us,
                                               const int* __restrict__ first, const int* __restrict__ item, const int* __restrict__ perm, int E,
                                               int chunk, int C, float* __restrict__ part) {
    constexpr int UC = 2 * Rp, UF = UC / 32;                       // columns of the pair, 32-row fragments
    constexpr int UP = UC == 32 ? 64 : UC * 2 + 64, XP = 320;      // byte pitches
    __shared__ __attribute__((aligned(16))) char xs[64 * XP];
    __shared__ __attribute__((aligned(16))) char ub[64 * UP];
    [[maybe_unused]] __shared__ float red[4];
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, hi = lane >> 5, l31 = lane & 31;
    const int it = blockIdx.y;
    if (it >= item[E]) return;
    int lo = 0, up = E - 1;                                        // the adapter whose items include `it`
    while (lo < up) {
        const int mid = (lo + up) >> 1;
        if (item[mid + 1] <= it) lo = mid + 1;
        else up = mid;
    }
    const int v0 = first[lo] + (it - item[lo]) * chunk, v1 = min(v0 + chunk, first[lo + 1]);
    const int c0 = blockIdx.x * 128;
    float top = 1.f;
#if defined(DM_F16)
    float big = 0.f;
    for (int v = v0 + tid; v < v1; v += 256) big = fmaxf(big, perm[v] >= 0 ? us[perm[v]] : 0.f);
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
    for (int v = v0; v < v1; v += 64) {
        __syncthreads();
#pragma unroll
        for (int q = 0; q < 4; ++q) {                              // 64 rows x 16 chunks of x
            const int idx = tid + 256 * q, row = idx >> 4, c = c0 + (idx & 15) * 8;
            u32x4 d = {0u, 0u, 0u, 0u};
            const int m = v + row < v1 ? perm[v + row] : kNone;
            if (m >= 0 && c < C) d = *reinterpret_cast<const u32x4*>(X + (long long)m * C + c);
            *reinterpret_cast<u32x4*>(xs + row * XP + (idx & 15) * 16) = d;
        }
        for (int idx = tid; idx < 64 * (Rp / 8); idx += 256) {     // 64 rows of pairs
            const int row = idx / (Rp / 8), c = idx % (Rp / 8) * 8;
            elem8 p = {}, q = {};
            const int m = v + row < v1 ? perm[v + row] : kNone;
            if (m >= 0) {
                p = *reinterpret_cast<const elem8*>(u + (long long)m * UC + c);
                q = *reinterpret_cast<const elem8*>(u + (long long)m * UC + Rp + c);
#if defined(DM_F16)
                const float f = us[m] * inv;
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const float w = ((float)p[k] + (float)q[k]) * f;
                    p[k] = (elem_t)w;
                    q[k] = (elem_t)(w - (float)p[k]);
                }
#endif
            }
            *reinterpret_cast<elem8*>(ub + row * UP + c * 2) = p;
            *reinterpret_cast<elem8*>(ub + row * UP + (Rp + c) * 2) = q;
        }
        __syncthreads();
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
    float* out = part + (long long)it * Rp * C + c;
    if constexpr (Rp == 16) {
#pragma unroll
        for (int r = 0; r < 8; ++r) out[(long long)((r & 3) + 8 * (r >> 2) + 4 * hi) * C] = (acc[0][r] + acc[0][r + 8]) * top;
    } else {
#pragma unroll
        for (int f = 0; f < UF / 2; ++f)
#pragma unroll
            for (int r = 0; r < 16; ++r) out[(long long)(32 * f + (r & 3) + 8 * (r >> 2) + 4 * hi) * C] = (acc[f][r] + acc[f + UF / 2][r]) * top;
    }
}

// out[e][r][c] (transpose: out[e][c][r]) = sum of the adapter's items in order, rounded once; an adapter without rows gets zeros.
// 64 columns x 4 ranks per workgroup; the transposed store goes through LDS.
__global__ __launch_bounds__(256) void k_wgrad_join(const float* __restrict__ part, const int* __restrict__ item, int C, int R, int Rp, int transpose,
                                                    elem_t* __restrict__ out) {
    const int e = blockIdx.z, c = blockIdx.x * 64 + (threadIdx.x & 63), r = blockIdx.y * 4 + (threadIdx.x >> 6);
    if (c >= C || r >= R) return;
    float s = 0.f;
    for (int it = item[e]; it < item[e + 1]; ++it) s += part[((long long)it * Rp + r) * C + c];
    if (transpose) out[((long long)e * C + c) * R + r] = (elem_t)s;
    else out[((long long)e * R + r) * C + c] = (elem_t)s;
}

// ------------------------------------------------------------------------------------------------ host side
int check_rows(const int* ids, long long n, long long M, int E, bool offsets) {
    if (!ids || n <= 0 || n > 0x7fffffff || M < 0 || M > 0x7fffffff || E <= 0) return DM_ERR_ARG;
    if (!offsets && (M % n)) return DM_ERR_ARG;
    return DM_OK;
}

Rows make_rows(const int* ids, const int* offsets, long long n, long long M, int E) {
    Rows r;
    r.ids = ids; r.offsets = offsets; r.M = M; r.n = (int)n; r.E = E;
    r.each = offsets ? 1 : std::max<long long>(1, M / n);
    return r;
}

// requests shorter than this share a tile with many others: one row at a time then
bool few_rows_each(long long M, long long n) { return M < 8 * n; }

template <int RT>
int launch_shrink(const elem_t* x, const elem_t* A, const Rows& rows, int K, int R, float scale, elem_t* u, float* us, hipStream_t stream) {
    const dim3 grid((unsigned)((rows.M + 16 * RT - 1) / (16 * RT)));
    switch (rank_pad(R)) {
        case 16: hipLaunchKernelGGL((k_shrink<RT, 1>), grid, dim3(256), 0, stream, x, A, rows, K, R, scale, u, us); break;
        case 32: hipLaunchKernelGGL((k_shrink<RT, 2>), grid, dim3(256), 0, stream, x, A, rows, K, R, scale, u, us); break;
        case 64: hipLaunchKernelGGL((k_shrink<(RT > 2 ? 2 : RT), 4>), dim3((unsigned)((rows.M + 16 * std::min(RT, 2) - 1) / (16 * std::min(RT, 2)))), dim3(256), 0, stream, x, A, rows, K, R, scale, u, us); break;
        default: hipLaunchKernelGGL((k_shrink<1, 8>), dim3((unsigned)((rows.M + 15) / 16)), dim3(256), 0, stream, x, A, rows, K, R, scale, u, us); break;
    }
    DM_LAUNCH_CHECK();
    return DM_OK;
}

int shrink(const elem_t* x, const elem_t* A, const Rows& rows, int K, int R, float scale, elem_t* u, float* us, hipStream_t stream) {
    if (few_rows_each(rows.M, rows.n)) {
        const int threads = std::min(1024, 64 * R);
        hipLaunchKernelGGL(k_shrink_rows, dim3((unsigned)rows.M), dim3(threads), 0, stream, x, A, rows, K, R, scale, u, us, (float*)nullptr);
        DM_LAUNCH_CHECK();
        return DM_OK;
    }
    if (rows.M >= 64 * 512) return launch_shrink<4>(x, A, rows, K, R, scale, u, us, stream);
    if (rows.M >= 32 * 512) return launch_shrink<2>(x, A, rows, K, R, scale, u, us, stream);
    return launch_shrink<1>(x, A, rows, K, R, scale, u, us, stream);
}

template <int BM, int BN, int WM, int WN>
int launch_expand(ExpandArgs a, hipStream_t stream) {
    constexpr int LDS = 2 * (BM + BN) * 128 + BM * 4;
    const long long n_mt = (a.rows.M + BM - 1) / BM;
    a.n_nt = (a.N + BN - 1) / BN;
    if (n_mt * a.n_nt > (1LL << 30)) return DM_ERR_UNSUPPORTED;
    a.tiles = (int)(n_mt * a.n_nt);
    static hipError_t attr = hipFuncSetAttribute(reinterpret_cast<const void*>(&k_expand<BM, BN, WM, WN>), hipFuncAttributeMaxDynamicSharedMemorySize, LDS);
    if (attr != hipSuccess) return (int)attr;
    const unsigned blocks = (unsigned)((a.tiles + 7) / 8 * 8);
    hipLaunchKernelGGL((k_expand<BM, BN, WM, WN>), dim3(blocks), dim3(WM * WN * 64), LDS, stream, a);
    DM_LAUNCH_CHECK();
    return DM_OK;
}

constexpr long long kSkinny = 32;

}  // namespace

extern "C" {

#if !defined(DM_F16)
// bytes of the u buffer for M rows: pairs of 16-bit columns, then one fp32 scale per row
size_t dm_adapter_u_bytes(long long M, int R) {
    if (M <= 0 || R <= 0 || R > kMaxRank) return 0;
    return (size_t)M * (4 * rank_pad(R) + 4);
}

// int32 words of the weight-gradient plan (first | item | start | perm) and its largest number of items
size_t dm_adapter_plan_words(long long M, long long n, int E) { return M <= 0 || n <= 0 || E <= 0 ? 0 : (size_t)(2 * (E + 1) + n + M); }
long long dm_adapter_plan_items(long long M, int E, int chunk) { return M <= 0 || E <= 0 || chunk <= 0 ? 0 : std::min<long long>(M, M / chunk + E); }

// the adapter order of the rows for dm_adapter_wgrad_*: plan [dm_adapter_plan_words] int32; chunk = rows per item (a multiple of 64)
int dm_adapter_plan(const int* ids, const int* offsets, long long n, long long M, int E, int chunk, int* plan, hipStream_t stream) {
    if (int rc = check_rows(ids, n, M, E, offsets != nullptr)) return rc;
    if (!plan || chunk <= 0 || chunk % 64 || M == 0) return DM_ERR_ARG;
    const Rows rows = make_rows(ids, offsets, n, M, E);
    int *first = plan, *item = first + E + 1, *start = item + E + 1, *perm = start + n;
    DM_ENTER();
    hipLaunchKernelGGL(k_wgrad_plan, dim3(1), dim3(1024), 0, stream, rows, chunk, first, item, start, perm);
    hipLaunchKernelGGL(k_wgrad_perm, dim3((unsigned)((M + 255) / 256)), dim3(256), 0, stream, rows, start, perm);
    DM_LAUNCH_CHECK();
    return DM_OK;
}
#endif

// y = x W^T + bias + s (x A_e^T) B_e^T + residual, see the head of this file.  x [M, K], w [N, K], bias [N] or NULL, residual [M, N] or
// NULL, lora_a [E, R, K], lora_b [E, N] rows of R elements `ldb` apart, ids [n] int32, offsets [n + 1] int32 or NULL (then M % n == 0), u
// scratch of dm_adapter_u_bytes; keep_u != 0: u is left in pair format for dm_adapter_wgrad_* (y NULL: nothing else is computed).  K % 8 == N % 8 == ldb % 8 == 0, R <= 128.
int DM_T(dm_linear_adapted_, )(const void* x, const void* w, const void* bias, const void* residual, const void* lora_a, const void* lora_b, int ldb,
                               const int* ids, const int* offsets, long long n, float scale, void* u, size_t u_bytes, void* y, long long M, int K,
                               int N, int R, int E, int keep_u, hipStream_t stream) {
    if (int rc = check_rows(ids, n, M, E, offsets != nullptr)) return rc;
    if (!x || !lora_a || !u || (y ? !w || !lora_b || ldb < R : !keep_u) || K <= 0 || N <= 0 || R <= 0) return DM_ERR_ARG;
    if (R > kMaxRank || K % 8 || N % 8 || (y && ldb % 8) || K > (1 << 20) || N > (1 << 24)) return DM_ERR_UNSUPPORTED;
    if (((uintptr_t)x | (uintptr_t)w | (uintptr_t)bias | (uintptr_t)residual | (uintptr_t)lora_a | (uintptr_t)lora_b | (uintptr_t)u | (uintptr_t)y) & 15) return DM_ERR_ARG;
    if (M == 0) return DM_OK;
    const int Rp = rank_pad(R);
    if (u_bytes < (size_t)M * (4 * Rp + 4)) return DM_ERR_WORKSPACE;
    ExpandArgs a{};
    a.x = (const elem_t*)x; a.w = (const elem_t*)w; a.bias = (const elem_t*)bias; a.res = (const elem_t*)residual;
    a.u = (const elem_t*)u; a.us = (const float*)((const elem_t*)u + M * 2 * Rp); a.B = (const elem_t*)lora_b; a.y = (elem_t*)y;
    a.rows = make_rows(ids, offsets, n, M, E);
    a.K = K; a.N = N; a.R = R; a.ldb = ldb;
    DM_ENTER();
    if (M <= kSkinny && !keep_u) {
        float* uf = (float*)u;
        hipLaunchKernelGGL(k_shrink_rows, dim3((unsigned)M), dim3(std::min(1024, 64 * R)), 0, stream, a.x, (const elem_t*)lora_a, a.rows, K, R, scale,
                           (elem_t*)nullptr, (float*)nullptr, uf);
        const dim3 grid((unsigned)((N + 15) / 16));
        if (M <= 16) hipLaunchKernelGGL(k_expand_skinny<1>, grid, dim3(512), 0, stream, a, uf);
        else hipLaunchKernelGGL(k_expand_skinny<2>, grid, dim3(512), 0, stream, a, uf);
        DM_LAUNCH_CHECK();
        return DM_OK;
    }
    if (int rc = shrink(a.x, (const elem_t*)lora_a, a.rows, K, R, scale, (elem_t*)u, const_cast<float*>(a.us), stream)) return rc;
    if (!y) return DM_OK;
    return launch_expand<128, 128, 2, 2>(a, stream);
}

// the adapters laid out for a product with padded rank rows: dst [E, C, rank padded to 16 | 32 | 64 | 128], zeros past R.  mode 0: src
// [E, C, R] copied; mode 1: src [E, R, C] transposed; mode 2: src [E, C, R] -> dst [E, R, C] (no padding)
int DM_T(dm_adapter_layout_, )(const void* src, void* dst, int E, int C, int R, int mode, hipStream_t stream) {
    if (!src || !dst || E <= 0 || C <= 0 || R <= 0 || mode < 0 || mode > 2) return DM_ERR_ARG;
    if (R > kMaxRank || E > 65535) return DM_ERR_UNSUPPORTED;
    const int Rp = rank_pad(R);
    const dim3 grid((unsigned)((C + 31) / 32), (unsigned)((Rp + 31) / 32), (unsigned)E);
    DM_ENTER();
    if (mode == 2) hipLaunchKernelGGL(k_adapter_cols, grid, dim3(256), 0, stream, (const elem_t*)src, (elem_t*)dst, C, R);
    else hipLaunchKernelGGL(k_adapter_rows, grid, dim3(256), 0, stream, (const elem_t*)src, (elem_t*)dst, C, R, Rp, mode);
    DM_LAUNCH_CHECK();
    return DM_OK;
}

// out[e] = sum over the rows m of adapter e of u[m, :]^T X[m, :]: [E, R, C], or (transpose) [E, C, R].  u as dm_linear_adapted_* left it (keep_u),
// plan from dm_adapter_plan with the same chunk, part fp32 [dm_adapter_plan_items][rank padded][C].
int DM_T(dm_adapter_wgrad_, )(const void* X, const void* u, const int* plan, long long n, long long M, int C, int R, int E, int chunk, int transpose,
                              float* part, size_t part_floats, void* out, hipStream_t stream) {
    if (!X || !u || !plan || !part || !out || n <= 0 || M <= 0 || M > 0x7fffffff || C <= 0 || R <= 0 || E <= 0 || chunk <= 0 || chunk % 64) return DM_ERR_ARG;
    if (R > kMaxRank || C % 8 || E > 65535) return DM_ERR_UNSUPPORTED;
    if (((uintptr_t)X | (uintptr_t)u) & 15) return DM_ERR_ARG;
    const int Rp = rank_pad(R);
    const long long items = std::min<long long>(M, M / chunk + E);
    if (items > 65535) return DM_ERR_UNSUPPORTED;
    if ((long long)part_floats < items * Rp * C) return DM_ERR_WORKSPACE;
    const int *first = plan, *item = first + E + 1, *perm = item + E + 1 + n;
    const elem_t* up = (const elem_t*)u;
    const float* us = (const float*)(up + M * 2 * Rp);
    const dim3 grid((unsigned)((C + 127) / 128), (unsigned)items);
    DM_ENTER();
    switch (Rp) {
        case 16: hipLaunchKernelGGL(k_wgrad<16>, grid, dim3(256), 0, stream, (const elem_t*)X, up, us, first, item, perm, E, chunk, C, part); break;
        case 32: hipLaunchKernelGGL(k_wgrad<32>, grid, dim3(256), 0, stream, (const elem_t*)X, up, us, first, item, perm, E, chunk, C, part); break;
        case 64: hipLaunchKernelGGL(k_wgrad<64>, grid, dim3(256), 0, stream, (const elem_t*)X, up, us, first, item, perm, E, chunk, C, part); break;
        default: hipLaunchKernelGGL(k_wgrad<128>, grid, dim3(256), 0, stream, (const elem_t*)X, up, us, first, item, perm, E, chunk, C, part); break;
    }
    hipLaunchKernelGGL(k_wgrad_join, dim3((unsigned)((C + 63) / 64), (unsigned)((R + 3) / 4), (unsigned)E), dim3(256), 0, stream, part, item, C, R, Rp,
                       transpose, (elem_t*)out);
    DM_LAUNCH_CHECK();
    return DM_OK;
}

}  // extern "C"
