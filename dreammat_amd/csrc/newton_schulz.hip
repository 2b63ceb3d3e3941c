// Orthogonalised matrix updates (gfx950): the Newton-Schulz iteration and the momentum step that uses it (Muon).
//
//   X0 = U / (|U|_F + eps), transposed so that it has m <= n;      five times:  S = X X^T,  P = b S + c S S,  X <- a X + P X
//   momentum step:  M <- mu M + g;  U = g + mu M (nesterov) or M;  p <- p (1 - lr wd) - lr s X
//
// (a, b, c) = (3.4445, -4.7750, 2.0315): every singular value s in (0, 1] runs through s <- a s + b s^3 + c s^5 and lands near 1.
//
// Bound by the matrix pipe: m^2 n + m^3 + 2 m^2 n flops per iteration (S and S S are symmetric: only the tiles on and below the diagonal
// are computed and stored twice).  All products are row-by-row (both operands contiguous along the contraction): X is kept in both
// orientations, S and P are symmetric, and an epilogue writes its tile both ways.
//
// Precision.  The iteration multiplies a small singular value -- and every rounding error next to it -- by a^5 = 485, so 8 bits (bf16
// storage) leave 1e-2 of error in the result and 11 bits (half) 1e-3, 1e-2 where a few directions dominate the matrix.  Numbers are
// therefore kept as a PAIR of halves, value + rest (22 bits; scaled by 2^13, so that neither leaves half's range: |X| <= 1.2, |S| <=
// 1.5, |P| <= 2.9), and a product is value value + value rest + rest value with fp32 sums: the result agrees with fp32 arithmetic to its
// own rounding (1.7e-6 against 1.7e-6 of the fp32 form on a 1024^2 Gaussian).  For bf16 input the last two iterations, whose
// errors are hardly amplified any more, take the values only: 0.6e-3 of error under the 1.7e-3 of the rounding to bf16.
// Pairs are stored as 128-byte blocks, 32 values then their 32 rests: a K step of the paired product loads the same lines as a K
// step of 64 plain halves.
#include <algorithm>
#include <type_traits>

#include "dm_common.h"

namespace {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

[[maybe_unused]] constexpr float kA = 3.4445f, kB = -4.7750f, kC = 2.0315f;
[[maybe_unused]] constexpr float kScale = 8192.f, kInv = 1.f / 8192.f;        // 2^13, see above
constexpr int kGroup = 16;                                   // matrices of one launch
constexpr int kNormParts = 64;                               // partial sums of a squared norm

// One group of same-shaped matrices [rows, cols] (row-major, contiguous)
struct Mats {
    const void* g[kGroup];
    float* mom[kGroup];      // momentum, or NULL
    float* p[kGroup];        // parameter, or NULL
    void* out[kGroup];       // orthogonalised matrix, or NULL
};

struct NsArgs {
    Mats t;
    int rows, cols;          // as given
    int m, n;                // m <= n: the iteration's orientation
    int mp, np;              // padded to multiples of 64
    int flip;                // rows > cols
    double* norm;            // [count][kNormParts]
    _Float16* x;             // pairs [count][mp][np]
    _Float16* xt[2];         // pairs [count][np][mp], ping-pong
    _Float16* s;             // pairs [count][mp][mp]
    _Float16* pm;            // pairs [count][mp][mp]
    float mu, eps, decay, step;
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
__device__ __forceinline__ float direction(const NsArgs& a, int b, long long i) {
    const float g = (float)reinterpret_cast<const T*>(a.t.g[b])[i];
    if (!a.t.mom[b]) return g;
    const float m = a.t.mom[b][i];
    return a.nesterov ? g + a.mu * m : m;
}

// momentum update and the squared norm of the direction: kNormParts workgroups per matrix, sums in 64 bits
template <typename T>
__global__ __launch_bounds__(256) void k_ns_norm(NsArgs a) {
    __shared__ double red[4];
    const int b = blockIdx.y;
    const long long total = (long long)a.rows * a.cols;
    double s = 0.0;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total; i += 256 * kNormParts) {
        if (a.t.mom[b]) a.t.mom[b][i] = a.mu * a.t.mom[b][i] + (float)reinterpret_cast<const T*>(a.t.g[b])[i];
        const double u = (double)direction<T>(a, b, i);
        s += u * u;
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) a.norm[(long long)b * kNormParts + blockIdx.x] = red[0] + red[1] + red[2] + red[3];
}

// X0 and X0^T as pairs, zero past m and n; a 64 x 64 tile through LDS per workgroup
template <typename T>
__global__ __launch_bounds__(256) void k_ns_pack(NsArgs a) {
    __shared__ float tile[64][65];
    const int b = blockIdx.z, i0 = blockIdx.y * 64, j0 = blockIdx.x * 64;       // rows / columns of X
    double sum = 0.0;
    for (int k = 0; k < kNormParts; ++k) sum += a.norm[(long long)b * kNormParts + k];
    const float inv = (float)((double)kScale / (sqrt(sum) + (double)a.eps));
    const int tx = threadIdx.x & 63, ty = threadIdx.x >> 6;
    for (int r = ty; r < 64; r += 4) {
        // read along the rows as given
        const int i = a.flip ? i0 + tx : i0 + r, j = a.flip ? j0 + r : j0 + tx;
        const bool ok = i < a.m && j < a.n;
        const float v = ok ? direction<T>(a, b, a.flip ? (long long)j * a.cols + i : (long long)i * a.cols + j) * inv : 0.f;
        if (a.flip) tile[tx][r] = v;
        else tile[r][tx] = v;
    }
    __syncthreads();
    _Float16* x = a.x + (long long)b * a.mp * 2 * a.np;
    _Float16* xt = a.xt[0] + (long long)b * a.np * 2 * a.mp;
    for (int r = ty; r < 64; r += 4) {
        _Float16 hi, lo;
        split(tile[r][tx], hi, lo);
        const long long p = pair_at(i0 + r, j0 + tx, a.np);
        x[p] = hi;
        x[p + 32] = lo;
        split(tile[tx][r], hi, lo);
        const long long q = pair_at(j0 + r, i0 + tx, a.mp);
        xt[q] = hi;
        xt[q + 32] = lo;
    }
}

enum { NS_GRAM = 0, NS_POLY = 1, NS_STEP = 2, NS_LAST = 3 };

// C[i, j] = sum_k A[i, k] B[j, k] over pair matrices, tile T x T, four waves of T/2 x T/2.  K goes in blocks of 32 pairs = 128 bytes per
// row, two LDS stages filled by buffer_load ... lds, chunks XOR-swizzled by (row >> 1) & 7.  PAIR: three products per block, else the
// values only (half of the loaded bytes; the block layout stays).
//   GRAM  A = B = X,          S = C                       (tiles i >= j, stored twice)
//   POLY  A = B = S,          P = b S + c C               (tiles i >= j, stored twice)
//   STEP  A = P, B = X^T,     X <- a X + C  in both orientations (X in place: a tile is read and written by its own workgroup only)
//   LAST  the same, into the parameter or the output
template <int KIND, int T, bool PAIR, typename OT>
__global__ __launch_bounds__(256) void k_ns_gemm(NsArgs a, int in, int tiles_i, int tiles_j) {
    [[maybe_unused]] constexpr int ROWB = 128, STAGE = 2 * T * ROWB, TW = T / 2, FT = TW / 32, PIECES = T / 32;
    [[maybe_unused]] __shared__ __attribute__((aligned(16))) char smem[2 * STAGE];
#if defined(__HIP_DEVICE_COMPILE__)
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, hi = lane >> 5, l31 = lane & 31;
    const int wi = wave >> 1, wj = wave & 1;
    // XCD-contiguous tile order (block b runs on XCD b % 8), matrix by matrix
    const int per_mat = KIND <= NS_POLY ? tiles_i * (tiles_i + 1) / 2 : tiles_i * tiles_j;
    const int total = per_mat * (int)gridDim.y;
    const int lin = blockIdx.y * gridDim.x + blockIdx.x;
    const int per = (total + 7) / 8;
    const int id = (lin & 7) * per + (lin >> 3);
    if ((lin >> 3) >= per || id >= total) return;
    const int b = id / per_mat, rem = id - b * per_mat;
    int ti, tj;
    if constexpr (KIND <= NS_POLY) {
        ti = (int)((sqrtf(8.f * (float)rem + 1.f) - 1.f) * 0.5f);
        while ((ti + 1) * (ti + 2) / 2 <= rem) ++ti;
        while (ti * (ti + 1) / 2 > rem) --ti;
        tj = rem - ti * (ti + 1) / 2;
    } else {
        ti = rem % tiles_i;                     // the row tiles of one X^T panel side by side
        tj = rem / tiles_i;
    }
    const int i0 = ti * T, j0 = tj * T;
    const int kw = KIND == NS_GRAM ? a.np : a.mp;                 // contraction width (padded)
    const _Float16* A = KIND == NS_GRAM ? a.x + (long long)b * a.mp * 2 * a.np : (KIND == NS_POLY ? a.s : a.pm) + (long long)b * a.mp * 2 * a.mp;
    const _Float16* B = KIND <= NS_POLY ? A : a.xt[in] + (long long)b * a.np * 2 * a.mp;
    const int arows = min(T, a.mp - i0), brows = min(T, (KIND <= NS_POLY ? a.mp : a.np) - j0);
    const __amdgpu_buffer_rsrc_t ars = __builtin_amdgcn_make_buffer_rsrc((void*)(A + (long long)i0 * 2 * kw), 0, arows * kw * 4, 0x00020000);
    const __amdgpu_buffer_rsrc_t brs = __builtin_amdgcn_make_buffer_rsrc((void*)(B + (long long)j0 * 2 * kw), 0, brows * kw * 4, 0x00020000);
    unsigned off[PIECES];                                          // rows past the matrix lie past the descriptor: zeros
#pragma unroll
    for (int p = 0; p < PIECES; ++p) {
        const int row = wave * (T / 4) + 8 * p + (lane >> 3);
        off[p] = (unsigned)row * (unsigned)kw * 4u + (unsigned)(((lane & 7) ^ ((row >> 1) & 7)) * 16);
    }
    auto issue = [&](int s, int stage) __attribute__((always_inline)) {
        char* base = smem + stage * STAGE;
#pragma unroll
        for (int p = 0; p < PIECES; ++p)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(ars, (__attribute__((address_space(3))) void*)(base + (wave * (T / 4) + 8 * p) * ROWB), 16, (int)off[p], s * 128, 0, 0);
#pragma unroll
        for (int p = 0; p < PIECES; ++p)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(brs, (__attribute__((address_space(3))) void*)(base + T * ROWB + (wave * (T / 4) + 8 * p) * ROWB), 16, (int)off[p], s * 128, 0, 0);
    };
    f32x16 acc[FT][FT];
#pragma unroll
    for (int i = 0; i < FT; ++i)
#pragma unroll
        for (int j = 0; j < FT; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;
    auto frag = [&](const char* base, int row, int chunk) __attribute__((always_inline)) {
        return *reinterpret_cast<const half8*>(base + row * ROWB + ((chunk ^ ((row >> 1) & 7)) << 4));
    };
    const int steps = kw / 32;
    issue(0, 0);
    for (int s = 0; s < steps; ++s) {
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        if (s + 1 < steps) issue(s + 1, (s + 1) & 1);
        const char* ab = smem + (s & 1) * STAGE;
        const char* bb = ab + T * ROWB;
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
            half8 ah[FT], al[FT], bh[FT], bl[FT];
#pragma unroll
            for (int i = 0; i < FT; ++i) {
                const int ra = TW * wi + 32 * i + l31, rb = TW * wj + 32 * i + l31;
                ah[i] = frag(ab, ra, 2 * kk + hi);
                bh[i] = frag(bb, rb, 2 * kk + hi);
                if constexpr (PAIR) {
                    al[i] = frag(ab, ra, 4 + 2 * kk + hi);
                    bl[i] = frag(bb, rb, 4 + 2 * kk + hi);
                }
            }
            // B as the matrix instruction's first operand: a lane holds one row i and four consecutive columns j per group
#pragma unroll
            for (int i = 0; i < FT; ++i)
#pragma unroll
                for (int j = 0; j < FT; ++j) {
                    if constexpr (PAIR) {
                        acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(bl[j], ah[i], acc[i][j], 0, 0, 0);
                        acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(bh[j], al[i], acc[i][j], 0, 0, 0);
                    }
                    acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(bh[j], ah[i], acc[i][j], 0, 0, 0);
                }
        }
    }

    // ---- epilogue.  lane: row i = l31 of the fragment, registers 4 g + r: columns 8 g + 4 hi + r.
    const int ow = KIND <= NS_POLY ? a.mp : a.np, oh = a.mp;
#pragma unroll
    for (int fi = 0; fi < FT; ++fi) {
        const int i = i0 + TW * wi + 32 * fi + l31;
#pragma unroll
        for (int fj = 0; fj < FT; ++fj) {
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int j = j0 + TW * wj + 32 * fj + 8 * g + 4 * hi;
                if (i >= oh || j >= ow) continue;
                float v[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) v[r] = acc[fi][fj][4 * g + r] * kInv;
                const long long at = pair_at(i, j, ow);
                if constexpr (KIND == NS_POLY) {
                    const _Float16* S = a.s + (long long)b * a.mp * 2 * a.mp + at;
                    const half4 h = *reinterpret_cast<const half4*>(S), l = *reinterpret_cast<const half4*>(S + 32);
#pragma unroll
                    for (int r = 0; r < 4; ++r) v[r] = kB * ((float)h[r] + (float)l[r]) + kC * v[r];
                }
                if constexpr (KIND >= NS_STEP) {
                    const _Float16* X = a.x + (long long)b * a.mp * 2 * a.np + at;
                    const half4 h = *reinterpret_cast<const half4*>(X), l = *reinterpret_cast<const half4*>(X + 32);
#pragma unroll
                    for (int r = 0; r < 4; ++r) v[r] = kA * ((float)h[r] + (float)l[r]) + v[r];
                }
                if constexpr (KIND == NS_LAST) {
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        if (i >= a.m || j + r >= a.n) continue;
                        const long long to = a.flip ? (long long)(j + r) * a.cols + i : (long long)i * a.cols + j + r;
                        const float o = v[r] * kInv;
                        if (a.t.p[b]) a.t.p[b][to] = a.t.p[b][to] * a.decay - a.step * o;
                        else reinterpret_cast<OT*>(a.t.out[b])[to] = (OT)o;
                    }
                } else {
                    half4 h, l;
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        _Float16 p, q;
                        split(v[r], p, q);
                        h[r] = p;
                        l[r] = q;
                    }
                    _Float16* D = KIND == NS_GRAM ? a.s : KIND == NS_POLY ? a.pm : a.x;
                    D += (long long)b * oh * 2 * ow;
                    *reinterpret_cast<half4*>(D + at) = h;
                    *reinterpret_cast<half4*>(D + at + 32) = l;
                    if (KIND == NS_STEP || ti != tj) {             // the other orientation
                        _Float16* E = KIND == NS_STEP ? a.xt[in ^ 1] + (long long)b * a.np * 2 * a.mp : D;
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            const long long q = pair_at(j + r, i, a.mp);
                            E[q] = h[r];
                            E[q + 32] = l[r];
                        }
                    }
                }
            }
        }
    }
#endif
}

long long pad64(long long v) { return (v + 63) / 64 * 64; }

// bytes of one matrix's workspace and of a group's
long long mat_bytes(long long rows, long long cols) {
    const long long m = pad64(std::min(rows, cols)), n = pad64(std::max(rows, cols));
    return 4 * (3 * m * n + 2 * m * m) + 8 * kNormParts;
}

// 128-wide tiles where they fill the chip (and the padded size loses little), else 64
bool wide_tiles(long long i, long long j, long long count) { return i >= 128 && j >= 128 && (i / 128) * (j / 128) * count >= 256; }

template <int KIND, typename OT>
void launch_gemm(const NsArgs& a, int in, bool pair, int count, hipStream_t stream) {
    const int cols = KIND <= NS_POLY ? a.mp : a.np;
    auto go = [&](auto t_tag, auto pair_tag) {
        constexpr int T = decltype(t_tag)::value;
        const int ti = (a.mp + T - 1) / T, tj = (cols + T - 1) / T;
        const int per_mat = KIND <= NS_POLY ? ti * (ti + 1) / 2 : ti * tj;
        const int per = (per_mat * count + 7) / 8;                 // the kernel's XCD order wants 8 * per blocks in all
        const unsigned gx = (unsigned)((8LL * per + count - 1) / count);
        hipLaunchKernelGGL((k_ns_gemm<KIND, T, decltype(pair_tag)::value, OT>), dim3(gx, (unsigned)count), dim3(256), 0, stream, a, in, ti, tj);
    };
    const bool wide = wide_tiles(a.mp, cols, count);
    if (wide) pair ? go(std::integral_constant<int, 128>{}, std::true_type{}) : go(std::integral_constant<int, 128>{}, std::false_type{});
    else pair ? go(std::integral_constant<int, 64>{}, std::true_type{}) : go(std::integral_constant<int, 64>{}, std::false_type{});
}

template <typename T>
int run_group(NsArgs& a, int count, int steps, int plain_steps, hipStream_t stream) {
    hipLaunchKernelGGL((k_ns_norm<T>), dim3(kNormParts, count), dim3(256), 0, stream, a);
    hipLaunchKernelGGL((k_ns_pack<T>), dim3(a.np / 64, a.mp / 64, count), dim3(256), 0, stream, a);
    DM_LAUNCH_CHECK();
    for (int k = 0; k < steps; ++k) {
        const bool pair = k < steps - plain_steps;
        launch_gemm<NS_GRAM, T>(a, k & 1, pair, count, stream);
        launch_gemm<NS_POLY, T>(a, k & 1, pair, count, stream);
        if (k + 1 < steps) launch_gemm<NS_STEP, T>(a, k & 1, pair, count, stream);
        else launch_gemm<NS_LAST, T>(a, k & 1, pair, count, stream);
        DM_LAUNCH_CHECK();
    }
    return DM_OK;
}

// dtype of the gradients / outputs: 0 bf16, 1 half, 2 fp32
int run(const void* const* g, float* const* mom, float* const* p, void* const* out, int count, int rows, int cols, int dtype, int steps, float mu,
        int nesterov, float eps, float decay, float step, void* ws, size_t ws_bytes, hipStream_t stream) {
    if (count < 0 || rows <= 0 || cols <= 0 || steps < 1 || steps > 64 || dtype < 0 || dtype > 2 || !ws) return DM_ERR_ARG;
    if ((long long)rows * cols > (1LL << 31) || std::min(rows, cols) > 32768 || std::max(rows, cols) > (1 << 20)) return DM_ERR_UNSUPPORTED;
    if ((uintptr_t)ws & 255) return DM_ERR_ARG;
    const long long one = mat_bytes(rows, cols);
    const int fit = (int)std::min<long long>(kGroup, (long long)ws_bytes / one);
    if (count && fit < 1) return DM_ERR_WORKSPACE;
    NsArgs a{};
    a.rows = rows; a.cols = cols; a.flip = rows > cols;
    a.m = std::min(rows, cols); a.n = std::max(rows, cols);
    a.mp = (int)pad64(a.m); a.np = (int)pad64(a.n);
    a.mu = mu; a.nesterov = nesterov; a.eps = eps; a.decay = decay; a.step = step;
    DM_ENTER();
    for (int at = 0; at < count; at += fit) {
        const int c = std::min(fit, count - at);
        for (int i = 0; i < c; ++i) {
            a.t.g[i] = g[at + i];
            a.t.mom[i] = mom ? mom[at + i] : nullptr;
            a.t.p[i] = p ? p[at + i] : nullptr;
            a.t.out[i] = out ? out[at + i] : nullptr;
            if (!a.t.g[i] || (mom && !a.t.mom[i]) || (p ? !a.t.p[i] : !a.t.out[i])) return DM_ERR_ARG;
        }
        char* w = (char*)ws;
        auto take = [&](long long bytes) { char* q = w; w += bytes * c; return q; };
        a.norm = (double*)take(8 * kNormParts);
        a.x = (_Float16*)take(4LL * a.mp * a.np);
        a.xt[0] = (_Float16*)take(4LL * a.mp * a.np);
        a.xt[1] = (_Float16*)take(4LL * a.mp * a.np);
        a.s = (_Float16*)take(4LL * a.mp * a.mp);
        a.pm = (_Float16*)take(4LL * a.mp * a.mp);
        // (bf16: the last two iterations without the rests, see the head of the file)
        const int rc = dtype == 0 ? run_group<__bf16>(a, c, steps, std::min(2, steps - 1), stream)
                     : dtype == 1 ? run_group<_Float16>(a, c, steps, 0, stream) : run_group<float>(a, c, steps, 0, stream);
        if (rc) return rc;
    }
    return DM_OK;
}

}  // namespace

extern "C" {

// workspace bytes that take `count` [rows, cols] matrices in one launch (at most 16 at once; less memory means more launches)
size_t dm_orthogonalize_workspace_bytes(int count, int rows, int cols) {
    if (count <= 0 || rows <= 0 || cols <= 0) return 0;
    return (size_t)(std::min(count, kGroup) * mat_bytes(rows, cols));
}

// out[i] = five-step Newton-Schulz of g[i]: `count` same-shaped matrices [rows, cols] behind HOST arrays of device pointers; dtype 0 bf16 |
// 1 half | 2 fp32 of both; ws 256-byte aligned
int dm_orthogonalize(const void* const* g_host, void* const* out_host, int count, int rows, int cols, int dtype, int steps, float eps, void* ws,
                     size_t ws_bytes, hipStream_t stream) {
    if (count && (!g_host || !out_host)) return DM_ERR_ARG;
    return run(g_host, nullptr, nullptr, out_host, count, rows, cols, dtype, steps, 0.f, 0, eps, 1.f, 0.f, ws, ws_bytes, stream);
}

// momentum step on fp32 masters: mom <- mu mom + g;  u = g + mu mom or mom;  p <- p decay - step orth(u).  g of `dtype`, mom / p fp32
int dm_muon_step(const void* const* g_host, float* const* mom_host, float* const* p_host, int count, int rows, int cols, int dtype, int steps, float mu,
                 int nesterov, float eps, float decay, float step, void* ws, size_t ws_bytes, hipStream_t stream) {
    if (count && (!g_host || !mom_host || !p_host)) return DM_ERR_ARG;
    return run(g_host, mom_host, p_host, nullptr, count, rows, cols, dtype, steps, mu, nesterov, eps, decay, step, ws, ws_bytes, stream);
}

}  // extern "C"
