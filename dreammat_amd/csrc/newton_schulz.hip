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
// errors are hardly amplified any more, take (and are given) the values only: 1e-3 of error under the 1.7e-3 of the rounding to bf16.
// (Taking the polynomials of S = X X^T alone and multiplying X0 once saves half the products of a wide matrix, but S holds squared singular
// values: on the gradients of a small ControlNet, which a few directions dominate, the result was 1e-3 to 1e-2 off where this form is 3e-5.)
// Pairs are stored as 128-byte blocks, 32 values then their 32 rests: a K step of the paired product loads the same lines as a K
// step of 64 plain halves.
#include <algorithm>
#include <type_traits>

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
    int whole;               // rows and pointers of the norm pass are whole 16-byte chunks
    int parts;               // workgroups per matrix of the norm pass
    double* norm;            // [count][kNormParts]
    float* part;             // partial sums of a split contraction
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

// momentum update and the squared norm of the direction: a.parts workgroups per matrix, four elements per thread, sums in 64 bits
template <typename T>
__global__ __launch_bounds__(256) void k_ns_norm(NsArgs a) {
    __shared__ double red[4];
    const int b = blockIdx.y;
    const long long total = (long long)a.rows * a.cols;
    const T* g = reinterpret_cast<const T*>(a.t.g[b]);
    float* mom = a.t.mom[b];
    double s = 0.0;
    auto add = [&](float u) { s += (double)u * (double)u; };
    if (a.whole) {
        typedef T vec __attribute__((ext_vector_type(4)));
        for (long long i = ((long long)blockIdx.x * 256 + threadIdx.x) * 4; i < total; i += 1024LL * a.parts) {
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
        for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total; i += 256LL * a.parts) {
            if (mom) mom[i] = a.mu * mom[i] + (float)g[i];
            add(direction<T>(a, b, i));
        }
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
    __shared__ double red[4];
    const int b = blockIdx.z, i0 = blockIdx.y * 64, j0 = blockIdx.x * 64;       // rows / columns of X
    const int tx = threadIdx.x & 63, ty = threadIdx.x >> 6;
    float v[16];
#pragma unroll
    for (int q = 0; q < 16; ++q) {                                              // read along the rows as given
        const int r = ty + 4 * q, i = a.flip ? i0 + tx : i0 + r, j = a.flip ? j0 + r : j0 + tx;
        v[q] = i < a.m && j < a.n ? direction<T>(a, b, a.flip ? (long long)j * a.cols + i : (long long)i * a.cols + j) : 0.f;
    }
    double s = 0.0;
    for (int k = threadIdx.x; k < a.parts; k += 256) s += a.norm[(long long)b * kNormParts + k];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
    if (tx == 0) red[ty] = s;
    __syncthreads();
    const float inv = (float)((double)kScale / (sqrt(red[0] + red[1] + red[2] + red[3]) + (double)a.eps));
#pragma unroll
    for (int q = 0; q < 16; ++q) {
        const int r = ty + 4 * q;
        if (a.flip) tile[tx][r] = v[q] * inv;
        else tile[r][tx] = v[q] * inv;
    }
    __syncthreads();
    _Float16* x = a.x + (long long)b * a.mp * 2 * a.np;
    _Float16* xt = a.xt[0] + (long long)b * a.np * 2 * a.mp;
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
        const long long at = pair_at(i0 + r, j0 + c, a.np);
        *reinterpret_cast<half8*>(x + at) = h;
        *reinterpret_cast<half8*>(x + at + 32) = l;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            _Float16 p, w;
            split(tile[c + k][r], p, w);
            h[k] = p;
            l[k] = w;
        }
        const long long to = pair_at(j0 + r, i0 + c, a.mp);
        *reinterpret_cast<half8*>(xt + to) = h;
        *reinterpret_cast<half8*>(xt + to + 32) = l;
    }
}

constexpr int threads_of(int T) { return T == 256 ? 512 : 256; }

template <int T>
__device__ __forceinline__ int tile_at(int row, int blk, int chunk) {
    return (row * (T / 32) + (blk ^ ((row >> 3) & 1))) * 128 + ((chunk ^ (row & 7)) << 4);
}

// One launch: D = src_c * src + acc_c * (A B^T) for `count` matrices
struct Product {
    const _Float16 *A, *B;           // [a_rows][kw], [b_rows][kw] pairs
    const _Float16* src;             // [a_rows][b_rows] pairs (SRC)
    _Float16* D;                     // the result as pairs [a_rows][b_rows]; symmetric: both halves of it
    _Float16* E;                     // not symmetric: the result transposed [b_rows][a_rows]
    int a_rows, b_rows, kw;          // padded
    float src_c, acc_c;
    int src_rests, rests;            // whether the source has rests, whether the result needs them (its readers take pairs)
    int tiles_i, tiles_j, count;
    int mode, splits;
};

// Tile T x T, two rows of WJ waves of T/2 x T/WJ.  K goes in blocks of 128 bytes per row through a ring of NST LDS stages filled by
// buffer_load ... lds (chunks XOR-swizzled by (row >> 1) & 7), NST - 1 of them in flight: 32 pairs (PAIR: three products per block) or the
// values of 64.
//   SYM   A B^T is symmetric: tiles i >= j, stored twice
//   SRC   the result adds src_c src (SYM: another matrix; else the matrix that D replaces, read and written by its own workgroup only)
//   LAST  the result goes into the parameter or the output instead of pairs
// The epilogue goes through LDS: the source tile arrives as whole lines, every lane replaces its own entries, and whole lines leave in both
// orientations (the transposed one by ds_read_b64_tr_b16); a 256 tile does that half by half.
// mode 0: the whole product.  1: this workgroup's share (blockIdx.z) of a split contraction, fp32 sums to a.part.  2: joins those shares.
template <int T, int NST, bool PAIR, bool SYM, bool SRC, bool LAST, typename OT>
__global__ __launch_bounds__(threads_of(T)) void k_ns_gemm(NsArgs a, Product g) {
    [[maybe_unused]] constexpr int NT = threads_of(T), NW = NT / 64, WJ = NW / 2, ROWB = 128, STAGE = 2 * T * ROWB, TI = T / 2, TJ = T / WJ, FI = TI / 32, FJ = TJ / 32,
                                   PIECES = T / 8 / NW, H = T == 256 ? 2 : 1, TR = T / H;       // TR rows per epilogue pass
    extern __shared__ __attribute__((aligned(16))) char smem[];      // max(NST * STAGE, 4 TR T)
#if defined(__HIP_DEVICE_COMPILE__)
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, hi = lane >> 5, l31 = lane & 31;
    const int wi = wave / WJ, wj = wave % WJ;
    const int mode = g.mode, splits = g.splits;
    // XCD-contiguous tile order (block b runs on XCD b % 8), matrix by matrix
    const int per_mat = SYM ? g.tiles_i * (g.tiles_i + 1) / 2 : g.tiles_i * g.tiles_j;
    const int total = per_mat * g.count, per = (total + 7) / 8;
    const int id = (int)(blockIdx.x & 7) * per + (int)(blockIdx.x >> 3);
    if ((int)(blockIdx.x >> 3) >= per || id >= total) return;
    const int b = id / per_mat, rem = id - b * per_mat;
    int ti, tj;
    if constexpr (SYM) {
        ti = (int)((sqrtf(8.f * (float)rem + 1.f) - 1.f) * 0.5f);
        while ((ti + 1) * (ti + 2) / 2 <= rem) ++ti;
        while (ti * (ti + 1) / 2 > rem) --ti;
        tj = rem - ti * (ti + 1) / 2;
    } else {
        ti = rem % g.tiles_i;                   // the row tiles of one panel of B side by side
        tj = rem / g.tiles_i;
    }
    const int i0 = ti * T, j0 = tj * T;
    f32x16 acc[FI][FJ];
    if (mode == 2) {
#pragma unroll
        for (int i = 0; i < FI; ++i)
#pragma unroll
            for (int j = 0; j < FJ; ++j)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const float4* p = reinterpret_cast<const float4*>(a.part) + ((long long)id * splits * FI * FJ * 4 + (i * FJ + j) * 4 + q) * NT + tid;
                    float4 v = p[0];
                    for (int z = 1; z < splits; ++z) {
                        const float4 o = p[(long long)z * FI * FJ * 4 * NT];
                        v.x += o.x; v.y += o.y; v.z += o.z; v.w += o.w;
                    }
                    acc[i][j][4 * q] = v.x; acc[i][j][4 * q + 1] = v.y; acc[i][j][4 * q + 2] = v.z; acc[i][j][4 * q + 3] = v.w;
                }
    } else {
        const int kw = g.kw;
        const _Float16* A = g.A + (long long)b * g.a_rows * 2 * kw;
        const _Float16* B = g.B + (long long)b * g.b_rows * 2 * kw;
        const int arows = min(T, g.a_rows - i0), brows = min(T, g.b_rows - j0);
        const __amdgpu_buffer_rsrc_t ars = __builtin_amdgcn_make_buffer_rsrc((void*)(A + (long long)i0 * 2 * kw), 0, arows * kw * 4, 0x00020000);
        const __amdgpu_buffer_rsrc_t brs = __builtin_amdgcn_make_buffer_rsrc((void*)(B + (long long)j0 * 2 * kw), 0, brows * kw * 4, 0x00020000);
        unsigned off[PIECES];                                      // rows past the matrix lie past the descriptor: zeros
#pragma unroll
        for (int p = 0; p < PIECES; ++p) {
            const int row = wave * (T / NW) + 8 * p + (lane >> 3);
            const int chunk = (lane & 7) ^ ((row >> 1) & 7);       // (values only: chunks 4 .. 7 are the next block's values)
            off[p] = (unsigned)row * (unsigned)kw * 4u + (unsigned)(PAIR ? chunk * 16 : (chunk >> 2) * 128 + (chunk & 3) * 16);
        }
        auto issue = [&](int s, int stage) __attribute__((always_inline)) {
            char* base = smem + stage * STAGE;
#pragma unroll
            for (int p = 0; p < PIECES; ++p)
                __builtin_amdgcn_raw_ptr_buffer_load_lds(ars, (__attribute__((address_space(3))) void*)(base + (wave * (T / NW) + 8 * p) * ROWB), 16, (int)off[p], s * (PAIR ? 128 : 256), 0, 0);
#pragma unroll
            for (int p = 0; p < PIECES; ++p)
                __builtin_amdgcn_raw_ptr_buffer_load_lds(brs, (__attribute__((address_space(3))) void*)(base + T * ROWB + (wave * (T / NW) + 8 * p) * ROWB), 16, (int)off[p], s * (PAIR ? 128 : 256), 0, 0);
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
        const int all = kw / (PAIR ? 32 : 64);
        const int s_lo = mode == 1 ? (int)((long long)all * blockIdx.z / splits) : 0, s_hi = mode == 1 ? (int)((long long)all * (blockIdx.z + 1) / splits) : all;
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
            const int fill = st == 0 ? NST - 1 : st - 1;           // the stage read one step ago
            if (s + NST - 1 < s_hi) issue(s + NST - 1, fill);
            const char* ab = smem + st * STAGE;
            const char* bb = ab + T * ROWB;
#pragma unroll
            for (int kk = 0; kk < (PAIR ? 2 : 4); ++kk) {
                half8 ah[FI], al[FI], bh[FJ], bl[FJ];
#pragma unroll
                for (int i = 0; i < FI; ++i) {
                    const int row = TI * wi + 32 * i + l31;
                    ah[i] = frag(ab, row, 2 * kk + hi);
                    if constexpr (PAIR) al[i] = frag(ab, row, 4 + 2 * kk + hi);
                }
#pragma unroll
                for (int j = 0; j < FJ; ++j) {
                    const int row = TJ * wj + 32 * j + l31;
                    bh[j] = frag(bb, row, 2 * kk + hi);
                    if constexpr (PAIR) bl[j] = frag(bb, row, 4 + 2 * kk + hi);
                }
                // B as the matrix instruction's first operand: a lane holds one row i and four consecutive columns j per group
#pragma unroll
                for (int i = 0; i < FI; ++i)
#pragma unroll
                    for (int j = 0; j < FJ; ++j) {
                        if constexpr (PAIR) {
                            acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(bl[j], ah[i], acc[i][j], 0, 0, 0);
                            acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(bh[j], al[i], acc[i][j], 0, 0, 0);
                        }
                        acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(bh[j], ah[i], acc[i][j], 0, 0, 0);
                    }
            }
            st = st + 1 == NST ? 0 : st + 1;
        }
        if (mode == 1) {
#pragma unroll
            for (int i = 0; i < FI; ++i)
#pragma unroll
                for (int j = 0; j < FJ; ++j)
#pragma unroll
                    for (int q = 0; q < 4; ++q)
                        reinterpret_cast<float4*>(a.part)[(((long long)id * splits + blockIdx.z) * FI * FJ * 4 + (i * FJ + j) * 4 + q) * NT + tid] =
                            make_float4(acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]);
            return;
        }
    }

    // ---- epilogue.  lane: row i = l31 of the fragment, registers 4 g + r: columns 8 g + 4 hi + r
    typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
    const int ow = g.b_rows, oh = g.a_rows;
    for (int h = 0; h < H; ++h) {
        const int r0 = i0 + h * TR;                                    // first row of this pass
        if (h && r0 >= oh) break;
        __syncthreads();                                               // every wave has read its last fragments (its share of the last pass)
        if constexpr (SRC) {
            constexpr int P = TR * T / 256 / NW;                       // 1 KB = 8 blocks per wave and request
            const _Float16* src = g.src + (long long)b * oh * 2 * ow;
            const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc((void*)(src + (long long)r0 * 2 * ow), 0, min(TR, oh - r0) * ow * 4, 0x00020000);
#pragma unroll
            for (int p = 0; p < P; ++p) {
                const int q = (wave * P + p) * 8 + (lane >> 3), row = q / (T / 32), blk = (q % (T / 32)) ^ ((row >> 3) & 1);
                const int chunk = (lane & 7) ^ (row & 7);
                const unsigned o = chunk < 4 || g.src_rests ? (unsigned)row * (unsigned)ow * 4u + (unsigned)((j0 / 32 + blk) * 128 + (chunk << 4)) : 0x80000000u;
                __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (__attribute__((address_space(3))) void*)(smem + (wave * P + p) * 1024), 16, (int)o, 0, 0, 0);
            }
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
                        half4* vp = reinterpret_cast<half4*>(smem + tile_at<T>(row, blk, q) + 8 * hi);
                        half4* rp = reinterpret_cast<half4*>(smem + tile_at<T>(row, blk, 4 + q) + 8 * hi);
                        float v[4];
#pragma unroll
                        for (int r = 0; r < 4; ++r) v[r] = acc[fi][fj][4 * q + r] * g.acc_c;
                        if constexpr (SRC) {
                            const half4 hv = *vp, lv = *rp;
#pragma unroll
                            for (int r = 0; r < 4; ++r) v[r] += g.src_c * ((float)hv[r] + (float)lv[r]);
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
            float* p = a.t.p[b];
            OT* out = reinterpret_cast<OT*>(a.t.out[b]);
            // four entries per thread along the fast axis of the matrix as given, a batch of loads in flight
            constexpr int Q = TR * T / 4 / NT, U = T == 256 ? 4 : Q < 8 ? Q : 8;
            static_assert(Q % U == 0, "whole batches");
            const bool four = (a.flip ? a.m : a.n) % 4 == 0 && !((uintptr_t)(p ? (void*)p : (void*)out) & 15);
            for (int k0 = 0; k0 < Q; k0 += U) {
                float4 old[U];
                long long to[U];
                int ok[U];
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int k = tid + (k0 + u) * NT;
                    const int row = a.flip ? k % (TR / 4) * 4 : k / (T / 4), col = a.flip ? k / (TR / 4) : k % (T / 4) * 4, i = r0 + row, j = j0 + col;
                    const int fast = a.flip ? a.m - i : a.n - j, slow = a.flip ? a.n - j : a.m - i;
                    ok[u] = slow > 0 ? max(0, min(4, fast)) : 0;
                    to[u] = a.flip ? (long long)j * a.cols + i : (long long)i * a.cols + j;
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
                    const int row = a.flip ? k % (TR / 4) * 4 : k / (T / 4), col = a.flip ? k / (TR / 4) : k % (T / 4) * 4;
                    float o[4];
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const int rr = a.flip ? row + r : row, cc = a.flip ? col : col + r;
                        o[r] = *reinterpret_cast<const float*>(smem + tile_at<T>(rr, cc >> 5, ((cc & 31) >> 3) + ((cc & 2) << 1)) + ((cc & 4) << 1) + ((cc & 1) << 2));
                    }
                    if (p) {
                        const float w[4] = {old[u].x * a.decay - a.step * o[0], old[u].y * a.decay - a.step * o[1], old[u].z * a.decay - a.step * o[2],
                                            old[u].w * a.decay - a.step * o[3]};
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
            _Float16* D = g.D + (long long)b * oh * 2 * ow;
#pragma unroll 4
            for (int q = tid; q < TR * T / 4; q += NT) {               // 16-byte chunks, whole rows of blocks
                const int chunk = q & 7, blk = (q >> 3) % (T / 32), row = (q >> 3) / (T / 32);
                if (r0 + row < oh && j0 + 32 * blk < ow && (chunk < 4 || g.rests))
                    *reinterpret_cast<u32x4*>(D + (long long)(r0 + row) * 2 * ow + (j0 / 32 + blk) * 64 + chunk * 8) =
                        *reinterpret_cast<const u32x4*>(smem + tile_at<T>(row, blk, chunk));
            }
            if (!SYM || ti != tj) {                                    // the other orientation: rows j, blocks of 32 i
                _Float16* E = SYM ? D : g.E + (long long)b * ow * 2 * oh;
                const int l15 = lane & 15, grp = lane >> 4;
                for (int u = wave; u < (T / 16) * (TR / 32) * (1 + g.rests); u += NW) {
                    const int part = g.rests ? u & 1 : 0, v = u >> g.rests, ib = v % (TR / 32), c0 = v / (TR / 32) * 16;
                    const int row = 32 * ib + 8 * grp + (l15 >> 2), cc = (c0 & 31) + 4 * (l15 & 3);
                    const char* p0 = smem + tile_at<T>(row, c0 >> 5, (cc >> 3) + 4 * part) + ((cc & 4) << 1);
                    const char* p1 = smem + tile_at<T>(row + 4, c0 >> 5, (cc >> 3) + 4 * part) + ((cc & 4) << 1);
                    const elem4 q0 = dm_ds_read_tr16_b64(p0), q1 = dm_ds_read_tr16_b64(p1);
                    const elem8 o = {q0[0], q0[1], q0[2], q0[3], q1[0], q1[1], q1[2], q1[3]};
                    const int j = j0 + c0 + l15, i = r0 + 32 * ib;
                    if (j < ow && i < oh) *reinterpret_cast<elem8*>(E + pair_at(j, i, oh) + 8 * grp + 32 * part) = o;
                }
            }
        }
    }
#endif
}

long long pad64(long long v) { return (v + 63) / 64 * 64; }

// Split of the Gram contraction: a wide X (n much larger than m) has few tiles with a long K each.  Shares of at least 16 steps, at most
// two workgroups per CU in all.  1: no split.
constexpr int kSplitTiles = 512;
int gram_splits(int mp, int np, int count) {
    const int t = (mp + 127) / 128, tiles = t * (t + 1) / 2 * count;
    return std::max(1, std::min(kSplitTiles / tiles, np / 32 / 16));
}

// bytes of one matrix's workspace (x, two x^T, s, p); of the split's partial sums
long long mat_bytes(long long rows, long long cols) {
    const long long m = pad64(std::min(rows, cols)), n = pad64(std::max(rows, cols));
    return 4 * (3 * m * n + 2 * m * m) + 8 * kNormParts;
}
long long part_bytes(long long rows, long long cols) {
    const int m = (int)pad64(std::min(rows, cols)), n = (int)pad64(std::max(rows, cols));
    return m >= 128 && gram_splits(m, n, 1) > 1 ? kSplitTiles * 4LL * 128 * 128 : 0;
}

template <int T, int NST, bool PAIR, bool SYM, bool SRC, bool LAST, typename OT>
int launch_tile(const NsArgs& a, Product g, int mode, int splits, hipStream_t stream) {
    constexpr int LDS = std::max(NST * 2 * T * 128, T == 256 ? 2 * T * T : 4 * T * T);
    static hipError_t attr = hipFuncSetAttribute(reinterpret_cast<const void*>(&k_ns_gemm<T, NST, PAIR, SYM, SRC, LAST, OT>), hipFuncAttributeMaxDynamicSharedMemorySize, LDS);
    if (attr != hipSuccess) return (int)attr;
    g.tiles_i = (g.a_rows + T - 1) / T;
    g.tiles_j = (g.b_rows + T - 1) / T;
    g.mode = mode;
    g.splits = splits;
    const long long total = (SYM ? (long long)g.tiles_i * (g.tiles_i + 1) / 2 : (long long)g.tiles_i * g.tiles_j) * g.count;
    hipLaunchKernelGGL((k_ns_gemm<T, NST, PAIR, SYM, SRC, LAST, OT>), dim3((unsigned)((total + 7) / 8 * 8), 1, mode == 1 ? splits : 1), dim3(threads_of(T)), LDS, stream, a, g);
    DM_LAUNCH_CHECK();
    return DM_OK;
}

// Tile by the time a launch takes, in rounds of the chip at one 256 tile per CU (measured on 1280^2, paired): a 256 tile needs a third of a
// 128 tile's LDS and request traffic per product; 128 tiles run two per CU and a round of 512 costs 1.15, half a round 0.6; 64 tiles 0.3
// per 512, 0.25 where a CU gets one (then with a ring as deep as LDS allows: its loads have nothing else to hide behind).
template <bool PAIR, bool SYM, bool SRC, bool LAST, typename OT>
int launch_gemm(const NsArgs& a, const Product& g, hipStream_t stream) {
    auto tiles = [&](int T) {
        const long long t = (g.a_rows + T - 1) / T, u = (g.b_rows + T - 1) / T;
        return (SYM ? t * (t + 1) / 2 : t * u) * g.count;
    };
    if (SYM && !SRC && a.part && g.a_rows >= 128) {
        const int splits = gram_splits(g.a_rows, g.kw, g.count);
        if (splits > 1) {
            if (int rc = launch_tile<128, 2, PAIR, SYM, SRC, LAST, OT>(a, g, 1, splits, stream)) return rc;
            return launch_tile<128, 2, PAIR, SYM, SRC, LAST, OT>(a, g, 2, splits, stream);
        }
    }
    const double c256 = g.a_rows >= 256 ? (double)((tiles(256) + 255) / 256) : 1e30;
    const double c128 = g.a_rows >= 128 ? std::max(0.6, 1.15 * (double)tiles(128) / 512) : 1e30;
    const double c64 = tiles(64) <= 256 ? 0.25 : 0.3 * (double)((tiles(64) + 511) / 512);
    if (c256 <= c128 && c256 <= c64) return launch_tile<256, 2, PAIR, SYM, SRC, LAST, OT>(a, g, 0, 1, stream);
    if (c128 <= c64) return launch_tile<128, 2, PAIR, SYM, SRC, LAST, OT>(a, g, 0, 1, stream);
    if (tiles(64) <= 256) return launch_tile<64, 8, PAIR, SYM, SRC, LAST, OT>(a, g, 0, 1, stream);
    return launch_tile<64, 4, PAIR, SYM, SRC, LAST, OT>(a, g, 0, 1, stream);
}

// the products of the iteration
struct Iteration {
    const NsArgs& a;
    int count;
    hipStream_t stream;
    Product make(const _Float16* A, int a_rows, const _Float16* B, int b_rows, int kw, const _Float16* src, float src_c, float acc_c, _Float16* D, _Float16* E) const {
        Product g{};
        g.A = A; g.B = B; g.src = src; g.D = D; g.E = E;
        g.a_rows = a_rows; g.b_rows = b_rows; g.kw = kw; g.src_c = src_c; g.acc_c = acc_c; g.count = count;
        return g;
    }
    // S = X X^T
    template <bool PAIR> int gram() const {
        Product g = make(a.x, a.mp, a.x, a.mp, a.np, nullptr, 0.f, kInv, a.s, nullptr);
        g.rests = PAIR;
        return launch_gemm<PAIR, true, false, false, float>(a, g, stream);
    }
    // P = b S + c S S
    template <bool PAIR> int poly() const {
        Product g = make(a.s, a.mp, a.s, a.mp, a.mp, a.s, kB, kC * kInv, a.pm, nullptr);
        g.src_rests = g.rests = PAIR;
        return launch_gemm<PAIR, true, true, false, float>(a, g, stream);
    }
    // X <- a X + P X, in both orientations; rests: the next iteration takes pairs
    template <bool PAIR> int step(int in, bool rests) const {
        Product g = make(a.pm, a.mp, a.xt[in], a.np, a.mp, a.x, kA, kInv, a.x, a.xt[in ^ 1]);
        g.src_rests = PAIR;
        g.rests = rests;
        return launch_gemm<PAIR, false, true, false, float>(a, g, stream);
    }
    // the result a X + P X
    template <bool PAIR, typename T> int last(int in) const {
        Product g = make(a.pm, a.mp, a.xt[in], a.np, a.mp, a.x, kA * kInv, kInv * kInv, nullptr, nullptr);
        g.src_rests = PAIR;
        return launch_gemm<PAIR, false, true, true, T>(a, g, stream);
    }
};

#define NS_TRY(call) if (int rc_ = (call)) return rc_

template <typename T>
int run_group(NsArgs& a, int count, int steps, hipStream_t stream) {
    hipLaunchKernelGGL((k_ns_norm<T>), dim3(a.parts, count), dim3(256), 0, stream, a);
    hipLaunchKernelGGL((k_ns_pack<T>), dim3(a.np / 64, a.mp / 64, count), dim3(256), 0, stream, a);
    DM_LAUNCH_CHECK();
    const Iteration it{a, count, stream};
    constexpr bool SHORT = std::is_same<T, __bf16>::value;       // bf16: the last two iterations without the rests, see the head of the file
    const int plain_from = SHORT ? std::max(1, steps - 2) : steps;
    for (int k = 0; k < steps; ++k) {
        if (k < plain_from) {
            NS_TRY(it.gram<true>());
            NS_TRY(it.poly<true>());
            NS_TRY(k + 1 < steps ? it.step<true>(k & 1, k + 1 < plain_from) : (it.last<true, T>(k & 1)));
        } else if constexpr (SHORT) {
            NS_TRY(it.gram<false>());
            NS_TRY(it.poly<false>());
            NS_TRY(k + 1 < steps ? it.step<false>(k & 1, false) : (it.last<false, T>(k & 1)));
        }
    }
    return DM_OK;
}

// dtype of the gradients / outputs: 0 bf16, 1 half, 2 fp32
int run(const void* const* g, float* const* mom, float* const* p, void* const* out, int count, int rows, int cols, int dtype, int steps, float mu,
        int nesterov, float eps, float decay, float step, void* ws, size_t ws_bytes, hipStream_t stream) {
    if (count < 0 || rows <= 0 || cols <= 0 || steps < 1 || steps > 64 || dtype < 0 || dtype > 2 || !ws) return DM_ERR_ARG;
    if ((long long)rows * cols > (1LL << 31) || std::min(rows, cols) > 32768 || std::max(rows, cols) > (1 << 20)) return DM_ERR_UNSUPPORTED;
    if ((uintptr_t)ws & 255) return DM_ERR_ARG;
    const long long one = mat_bytes(rows, cols), extra = part_bytes(rows, cols);
    const int fit = (int)std::min<long long>(kGroup, std::max<long long>(0, (long long)ws_bytes - extra) / one);
    if (count && fit < 1) return DM_ERR_WORKSPACE;
    NsArgs a{};
    a.rows = rows; a.cols = cols; a.flip = rows > cols;
    a.m = std::min(rows, cols); a.n = std::max(rows, cols);
    a.mp = (int)pad64(a.m); a.np = (int)pad64(a.n);
    a.mu = mu; a.nesterov = nesterov; a.eps = eps; a.decay = decay; a.step = step;
    a.parts = (int)std::max<long long>(1, std::min<long long>(kNormParts, (long long)rows * cols / (256 * 8)));
    DM_ENTER();
    for (int at = 0; at < count; at += fit) {
        const int c = std::min(fit, count - at);
        bool whole = cols % 4 == 0;                                // rows of 16-byte (8-byte) chunks in every operand of the norm pass
        for (int i = 0; i < c; ++i) {
            a.t.g[i] = g[at + i];
            a.t.mom[i] = mom ? mom[at + i] : nullptr;
            a.t.p[i] = p ? p[at + i] : nullptr;
            a.t.out[i] = out ? out[at + i] : nullptr;
            if (!a.t.g[i] || (mom && !a.t.mom[i]) || (p ? !a.t.p[i] : !a.t.out[i])) return DM_ERR_ARG;
            whole = whole && !(((uintptr_t)a.t.g[i] | (uintptr_t)a.t.mom[i]) & 15);
        }
        a.whole = whole;
        char* w = (char*)ws;
        a.part = extra ? (float*)w : nullptr;
        w += extra;
        auto take = [&](long long bytes) { char* q = w; w += bytes * c; return q; };
        a.norm = (double*)take(8 * kNormParts);
        a.x = (_Float16*)take(4LL * a.mp * a.np);
        a.xt[0] = (_Float16*)take(4LL * a.mp * a.np);
        a.xt[1] = (_Float16*)take(4LL * a.mp * a.np);
        a.s = (_Float16*)take(4LL * a.mp * a.mp);
        a.pm = (_Float16*)take(4LL * a.mp * a.mp);
        const int rc = dtype == 0 ? run_group<__bf16>(a, c, steps, stream) : dtype == 1 ? run_group<_Float16>(a, c, steps, stream) : run_group<float>(a, c, steps, stream);
        if (rc) return rc;
    }
    return DM_OK;
}

}  // namespace

extern "C" {

// workspace bytes that take `count` [rows, cols] matrices in one launch (at most 16 at once; less memory means more launches)
size_t dm_orthogonalize_workspace_bytes(int count, int rows, int cols) {
    if (count <= 0 || rows <= 0 || cols <= 0) return 0;
    return (size_t)(std::min(count, kGroup) * mat_bytes(rows, cols) + part_bytes(rows, cols));
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
