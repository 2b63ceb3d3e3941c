// Norms before and after a transformer block fused with its gate and residual scale, for gfx950.
//
//   y = x + scale * g * N_post(h)        z = N_pre(y)
//
// x is the residual stream, h the block's output, g a gate per channel or per (item, channel), N_post the norm behind the block and
// N_pre the one in front of the next (either may be absent); N is LayerNorm ((v - mean) rstd gamma + beta) or RMSNorm (v rstd gamma
// + beta).  The framework's k_layernorm (transformer.hip) is the bare forward; a training step's norms, gates and residual adds
// otherwise run as separate ATen passes.
//
// Bound by HBM: the forward reads x, h and writes y, z; the backward reads x, h, dy, dz and writes dx, dh -- each exactly once.  A
// row lives in the registers of L lanes (L = 16 | 32 | 64 lanes of a wave, or a workgroup of 256 ... 1024) as NC 16-byte chunks per lane;
// statistics are two passes over those registers (mean, then centred second moment) in fp32, and y enters N_pre as the fp32 value,
// not as its 16-bit rounding.  The backward recomputes y from x and h (the same bytes as reading y, and exact) with the row
// statistics the forward kept (16 bytes per row).
//
// Backward formulas (dY = gradient of y from both outputs, dn = scale g dY):
//   dY = dy + N_pre'(dz)      dx = dY      dh = N_post'(dn)      dg = sum_rows scale N_post(h) dY
//   dgamma_post = sum dn hhat      dbeta_post = sum dn      dgamma_pre = sum dz yhat      dbeta_pre = sum dz
//   N'(d) = rstd (d gamma - mean(d gamma) - vhat mean(d gamma vhat))      (RMS: without the first mean)
// The column sums accumulate in fp32 registers over the rows of a workgroup and are joined in a fixed order (no atomics): through LDS
// across the workgroup's row groups, then over the workgroups by k_gan_reduce.
#include <algorithm>
#include <initializer_list>

#include "dm_common.h"

namespace {

struct GanArgs {
    const void *x, *h, *gate, *post_g, *post_b, *pre_g, *pre_b, *dy, *dz;
    void *y, *z, *dx, *dh;
    float* stats;            // [rows][4] post mean, post rstd, pre mean, pre rstd
    float* part;             // backward partial sums, see k_gan_bwd
    long long rows, item_rows;
    long long rows_per_block;
    int C;
    float scale, eps;
    int rms, post, pre;
    int want;                // GAN_D* bits: which column sums the caller wants
};

enum { GAN_DGATE = 1, GAN_DPOST_G = 2, GAN_DPOST_B = 4, GAN_DPRE_G = 8, GAN_DPRE_B = 16 };

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

template <typename T> struct Elems;
template <> struct Elems<float> { static constexpr int N = 4; };
template <> struct Elems<__bf16> { static constexpr int N = 8; };
template <> struct Elems<_Float16> { static constexpr int N = 8; };

// one chunk = 16 bytes (VEC > 1) or one element (VEC == 1: rows that are not whole 16-byte chunks), held as stored until it is used
template <typename T, int VEC> struct Chunk {
    typedef T vec __attribute__((ext_vector_type(VEC)));
    vec v;
    __device__ __forceinline__ float operator[](int k) const { return (float)v[k]; }
};

template <typename T, int VEC>
__device__ __forceinline__ Chunk<T, VEC> load_chunk(const void* p, long long at) {
    Chunk<T, VEC> c;
    const T* q = reinterpret_cast<const T*>(p) + at;
    if constexpr (VEC == 1) c.v[0] = q[0];
    else c.v = *reinterpret_cast<const typename Chunk<T, VEC>::vec*>(q);
    return c;
}

template <typename T, int VEC>
__device__ __forceinline__ Chunk<T, VEC> fill_chunk(float x) {
    Chunk<T, VEC> c;
#pragma unroll
    for (int k = 0; k < VEC; ++k) c.v[k] = (T)x;
    return c;
}

template <typename T, int VEC>
__device__ __forceinline__ void store_chunk(void* p, long long at, const float (&v)[VEC]) {
    Chunk<T, VEC> c;
#pragma unroll
    for (int k = 0; k < VEC; ++k) c.v[k] = (T)v[k];
    T* q = reinterpret_cast<T*>(p) + at;
    if constexpr (VEC == 1) q[0] = c.v[0];
    else *reinterpret_cast<typename Chunk<T, VEC>::vec*>(q) = c.v;
}

constexpr int threads_of(int L) { return L < 256 ? 256 : L; }

// sum over the L lanes of a row (L > 64: several waves, through LDS; every thread of the workgroup must call it)
template <int L>
__device__ __forceinline__ float row_sum(float v, float* red) {
#pragma unroll
    for (int o = (L < 64 ? L : 64) / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    if constexpr (L > 64) {
        const int w0 = threadIdx.x / L * (L / 64);
        __syncthreads();
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
        __syncthreads();
        v = 0.f;
#pragma unroll
        for (int w = 0; w < L / 64; ++w) v += red[w0 + w];
    }
    return v;
}

// statistics of a row held as v (invalid chunks are zero): mean (0 for rms) and 1 / sqrt(second moment + eps)
template <int VEC, int L, int NC>
__device__ __forceinline__ void row_stats(const float (&v)[NC][VEC], int chunks, int l, int rms, float inv_c, float eps, float* red,
                                          float& mean, float& rstd) {
    mean = 0.f;
    if (!rms) {
        float s = 0.f;
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int k = 0; k < VEC; ++k) s += v[c][k];
        mean = row_sum<L>(s, red) * inv_c;
    }
    float q = 0.f;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        const bool ok = l + L * c < chunks;
#pragma unroll
        for (int k = 0; k < VEC; ++k) { const float d = v[c][k] - mean; q += ok ? d * d : 0.f; }
    }
    rstd = 1.f / sqrtf(row_sum<L>(q, red) * inv_c + eps);
}

// this lane's chunks of a parameter vector; a NULL gamma is 1, a NULL beta 0
template <typename T, int VEC, int L, int NC>
__device__ __forceinline__ void load_params(const void* p, long long at, int l, int chunks, float absent, Chunk<T, VEC> (&out)[NC]) {
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        const int ch = l + L * c;
        if (p) out[c] = load_chunk<T, VEC>(p, at + (ch < chunks ? ch : 0) * VEC);
        else out[c] = fill_chunk<T, VEC>(absent);
    }
}

// Workgroup b owns rows [b R, (b + 1) R) (R = rows_per_block), G row groups at a time, one gate item after the other; parameters stay in
// registers, and the next rows are requested before this one's statistics.  [24, 4096, 320] bf16 with z: 43 us, 5.8 TB/s; [24, 1024, 1280]
// fp32: 93-97 us, 5.3 TB/s.
template <typename T, int VEC, int L, int NC>
__global__ __launch_bounds__(threads_of(L)) void k_gan_fwd(GanArgs a) {
    __shared__ float red[16];
    constexpr int G = threads_of(L) / L;
    const int l = threadIdx.x % L, grp = threadIdx.x / L;
    const int chunks = a.C / VEC;
    const float inv_c = 1.f / (float)a.C;
    const long long row_lo = (long long)blockIdx.x * a.rows_per_block, row_hi = min(row_lo + a.rows_per_block, a.rows);
    Chunk<T, VEC> pg[NC], pb[NC], qg[NC], qb[NC], g[NC], xn[NC], hn[NC];
    auto fetch = [&](long long r) __attribute__((always_inline)) {
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const int ch = l + L * c;
            const long long at = r * a.C + (ch < chunks ? ch : 0) * VEC;
            hn[c] = load_chunk<T, VEC>(a.h, at);
            xn[c] = load_chunk<T, VEC>(a.x, at);
        }
    };
    fetch(min(row_lo + grp, row_hi - 1));
    load_params<T, VEC, L, NC>(a.post_g, 0, l, chunks, 1.f, pg);
    load_params<T, VEC, L, NC>(a.post_b, 0, l, chunks, 0.f, pb);
    load_params<T, VEC, L, NC>(a.pre_g, 0, l, chunks, 1.f, qg);
    load_params<T, VEC, L, NC>(a.pre_b, 0, l, chunks, 0.f, qb);
    long long seg_lo = row_lo;
    while (seg_lo < row_hi) {
        const long long item = a.item_rows ? seg_lo / a.item_rows : 0;
        const long long seg_hi = a.item_rows ? min((item + 1) * a.item_rows, row_hi) : row_hi;
        load_params<T, VEC, L, NC>(a.gate, item * a.C, l, chunks, 1.f, g);
        // (the loop bounds are the workgroup's, not the row's: row_sum synchronises where a row is the workgroup's)
        for (long long r0 = seg_lo; r0 < seg_hi; r0 += G) {
            const long long r = min(r0 + grp, seg_hi - 1);
            const bool live = r0 + grp < seg_hi;
            float v[NC][VEC], y[NC][VEC];
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                const bool ok = l + L * c < chunks;
#pragma unroll
                for (int k = 0; k < VEC; ++k) v[c][k] = ok ? hn[c][k] : 0.f, y[c][k] = ok ? xn[c][k] : 0.f;
            }
            const long long next = r0 + G < seg_hi ? min(r0 + G + grp, seg_hi - 1) : min(seg_hi + grp, row_hi - 1);
            if (r0 + G < seg_hi || seg_hi < row_hi) fetch(next);
            float pm = 0.f, pr = 1.f, qm = 0.f, qr = 1.f;
            if (a.post) row_stats<VEC, L, NC>(v, chunks, l, a.rms, inv_c, a.eps, red, pm, pr);
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                const int ch = l + L * c;
                if (ch >= chunks) continue;
#pragma unroll
                for (int k = 0; k < VEC; ++k) {
                    const float n = a.post ? (v[c][k] - pm) * pr * pg[c][k] + pb[c][k] : v[c][k];
                    y[c][k] += a.scale * g[c][k] * n;
                }
                if (live) store_chunk<T, VEC>(a.y, r * a.C + ch * VEC, y[c]);
            }
            if (a.pre) {
                row_stats<VEC, L, NC>(y, chunks, l, a.rms, inv_c, a.eps, red, qm, qr);
#pragma unroll
                for (int c = 0; c < NC; ++c) {
                    const int ch = l + L * c;
                    if (ch >= chunks) continue;
                    float z[VEC];
#pragma unroll
                    for (int k = 0; k < VEC; ++k) z[k] = (y[c][k] - qm) * qr * qg[c][k] + qb[c][k];
                    if (live) store_chunk<T, VEC>(a.z, r * a.C + ch * VEC, z);
                }
            }
            if (a.stats && live && l == 0) *reinterpret_cast<float4*>(a.stats + r * 4) = make_float4(pm, pr, qm, qr);
        }
        seg_lo = seg_hi;
    }
}

// Rows as in the forward.  Column sums that run over all rows go to part[slot][b][C], one slot per wanted vector.  The gate's gradient is
// per item where the gate is: rows of an item may span workgroups and a workgroup may hold several items, so its partial sums are flushed
// at every item boundary to gate_part[item + b][C] -- along a walk over the rows (item, b) only grows, so item + b names the pair -- behind
// the other slots.  fp32: bound by HBM, [24, 1024, 1280] 160 us, 4.7 TB/s.  16 bits: by the vector pipe (eight entries of six tensors and five
// sums per chunk), whose instructions take two thirds of the cycles, a third of its lanes without a chunk at these widths (80 chunks on 128
// lanes): [4, 4096, 640] bf16 50 us, 2.5 TB/s.
template <typename T, int VEC, int L, int NC>
__global__ __launch_bounds__(threads_of(L)) void k_gan_bwd(GanArgs a) {
    __shared__ float red[16];
    constexpr int G = threads_of(L) / L;
    __shared__ float join[G == 1 ? 1 : G * L * NC * VEC];
    const int l = threadIdx.x % L, grp = threadIdx.x / L;
    const int chunks = a.C / VEC;
    const float inv_c = 1.f / (float)a.C;
    const long long row_lo = (long long)blockIdx.x * a.rows_per_block, row_hi = min(row_lo + a.rows_per_block, a.rows);
    Chunk<T, VEC> pg[NC], pb[NC], qg[NC], g[NC], xn[NC], hn[NC], dyn[NC], dzn[NC];
    float4 sn;
    auto fetch = [&](long long r) __attribute__((always_inline)) {
        sn = *reinterpret_cast<const float4*>(a.stats + r * 4);
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const int ch = l + L * c;
            const long long at = r * a.C + (ch < chunks ? ch : 0) * VEC;
            hn[c] = load_chunk<T, VEC>(a.h, at);
            xn[c] = load_chunk<T, VEC>(a.x, at);
            if (a.dy) dyn[c] = load_chunk<T, VEC>(a.dy, at);
            if (a.pre) dzn[c] = load_chunk<T, VEC>(a.dz, at);
        }
    };
#pragma unroll
    for (int c = 0; c < NC; ++c) dyn[c] = fill_chunk<T, VEC>(0.f), dzn[c] = fill_chunk<T, VEC>(0.f);
    fetch(min(row_lo + grp, row_hi - 1));
    load_params<T, VEC, L, NC>(a.post_g, 0, l, chunks, 1.f, pg);
    load_params<T, VEC, L, NC>(a.post_b, 0, l, chunks, 0.f, pb);
    load_params<T, VEC, L, NC>(a.pre_g, 0, l, chunks, 1.f, qg);
    float dg[NC][VEC], dpg[NC][VEC], dpb[NC][VEC], dqg[NC][VEC], dqb[NC][VEC];
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int k = 0; k < VEC; ++k) dg[c][k] = dpg[c][k] = dpb[c][k] = dqg[c][k] = dqb[c][k] = 0.f;

    // adds the G row groups' sums in order and writes the workgroup's row of `out`
    auto flush = [&](float (&s)[NC][VEC], float* out) __attribute__((always_inline)) {
        if constexpr (G == 1) {
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                const int ch = l + L * c;
                if (ch < chunks)
#pragma unroll
                    for (int k = 0; k < VEC; ++k) out[ch * VEC + k] = s[c][k];
            }
        } else {
            __syncthreads();
#pragma unroll
            for (int c = 0; c < NC; ++c)
#pragma unroll
                for (int k = 0; k < VEC; ++k) join[(grp * NC * VEC + c * VEC + k) * L + l] = s[c][k];
            __syncthreads();
            for (int t = threadIdx.x; t < L * NC * VEC; t += threads_of(L)) {
                const int tl = t % L, ck = t / L, ch = tl + L * (ck / VEC);
                if (ch >= chunks) continue;
                float sum = 0.f;
#pragma unroll
                for (int q = 0; q < G; ++q) sum += join[(q * NC * VEC + ck) * L + tl];
                out[ch * VEC + ck % VEC] = sum;
            }
        }
    };

    const long long nblk = gridDim.x;
    float* gate_part = a.part + (long long)__popc(a.want & ~GAN_DGATE) * nblk * a.C;
    long long seg_lo = row_lo;
    while (seg_lo < row_hi) {                                       // one item's rows at a time (uniform for the workgroup)
        const long long item = a.item_rows ? seg_lo / a.item_rows : 0;
        const long long seg_hi = a.item_rows ? min((item + 1) * a.item_rows, row_hi) : row_hi;
        load_params<T, VEC, L, NC>(a.gate, item * a.C, l, chunks, 1.f, g);
        for (long long r0 = seg_lo; r0 < seg_hi; r0 += G) {
            const long long base = min(r0 + grp, seg_hi - 1) * a.C;
            const bool live = r0 + grp < seg_hi;
            const float4 st = sn;
            float hh[NC][VEC], y[NC][VEC], d[NC][VEC], dz[NC][VEC];   // hhat, then yhat, dY, dz gamma_pre
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                const bool use = l + L * c < chunks && live;
#pragma unroll
                for (int k = 0; k < VEC; ++k) {
                    hh[c][k] = use ? hn[c][k] : 0.f;
                    y[c][k] = use ? xn[c][k] : 0.f;
                    d[c][k] = use ? dyn[c][k] : 0.f;
                    dz[c][k] = use ? dzn[c][k] : 0.f;
                }
            }
            if (r0 + G < seg_hi || seg_hi < row_hi) fetch(r0 + G < seg_hi ? min(r0 + G + grp, seg_hi - 1) : min(seg_hi + grp, row_hi - 1));
            // y in fp32, exactly as the forward formed it
            float s1 = 0.f, s2 = 0.f;
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                const bool use = l + L * c < chunks && live;
#pragma unroll
                for (int k = 0; k < VEC; ++k) {
                    if (a.post) hh[c][k] = use ? (hh[c][k] - st.x) * st.y : 0.f;
                    const float n = a.post ? hh[c][k] * pg[c][k] + pb[c][k] : hh[c][k];
                    y[c][k] += a.scale * g[c][k] * n;
                    if (a.pre) {
                        y[c][k] = use ? (y[c][k] - st.z) * st.w : 0.f;        // yhat
                        dqg[c][k] += dz[c][k] * y[c][k];
                        dqb[c][k] += dz[c][k];
                        dz[c][k] *= qg[c][k];
                        s1 += dz[c][k];
                        s2 += dz[c][k] * y[c][k];
                    }
                }
            }
            if (a.pre) {
                const float m2 = row_sum<L>(s2, red) * inv_c, m1 = a.rms ? 0.f : row_sum<L>(s1, red) * inv_c;
#pragma unroll
                for (int c = 0; c < NC; ++c)
#pragma unroll
                    for (int k = 0; k < VEC; ++k) d[c][k] += st.w * (dz[c][k] - m1 - y[c][k] * m2);
            }
            float t1 = 0.f, t2 = 0.f;
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                const int ch = l + L * c;
                const bool use = ch < chunks && live;
                if (use && a.dx) store_chunk<T, VEC>(a.dx, base + ch * VEC, d[c]);
#pragma unroll
                for (int k = 0; k < VEC; ++k) {
                    const float dY = use ? a.scale * d[c][k] : 0.f;
                    const float n = a.post ? hh[c][k] * pg[c][k] + pb[c][k] : hh[c][k];
                    dg[c][k] += dY * n;
                    const float dn = dY * g[c][k];
                    dpg[c][k] += dn * hh[c][k];
                    dpb[c][k] += dn;
                    d[c][k] = dn * (a.post ? pg[c][k] : 1.f);
                    t1 += d[c][k];
                    t2 += d[c][k] * hh[c][k];
                }
            }
            if (a.post) {
                const float m2 = row_sum<L>(t2, red) * inv_c, m1 = a.rms ? 0.f : row_sum<L>(t1, red) * inv_c;
#pragma unroll
                for (int c = 0; c < NC; ++c)
#pragma unroll
                    for (int k = 0; k < VEC; ++k) d[c][k] = st.y * (d[c][k] - m1 - hh[c][k] * m2);
            }
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                const int ch = l + L * c;
                if (ch < chunks && live && a.dh) store_chunk<T, VEC>(a.dh, base + ch * VEC, d[c]);
            }
        }
        if (a.want & GAN_DGATE) {
            flush(dg, gate_part + (item + blockIdx.x) * a.C);
#pragma unroll
            for (int c = 0; c < NC; ++c)
#pragma unroll
                for (int k = 0; k < VEC; ++k) dg[c][k] = 0.f;
        }
        seg_lo = seg_hi;
    }
    float* out = a.part + (long long)blockIdx.x * a.C;
    if (a.want & GAN_DPOST_G) { flush(dpg, out); out += nblk * a.C; }
    if (a.want & GAN_DPOST_B) { flush(dpb, out); out += nblk * a.C; }
    if (a.want & GAN_DPRE_G) { flush(dqg, out); out += nblk * a.C; }
    if (a.want & GAN_DPRE_B) flush(dqb, out);
}

struct GanReduceArgs {
    const float* part;
    void* out[5];            // gate, post gamma, post beta, pre gamma, pre beta (NULL where not wanted)
    int want, C;
    long long nblk, rows_per_block, item_rows, rows, items;
};

// grid (column blocks of 32, 4 + items): y < 4 the vectors summed over all workgroups, y >= 4 the gate row of item y - 4.  1024 threads =
// 32 columns x 32 shares of the workgroups, eight loads in flight each, joined in order.  512 workgroups' sums of 640 to 1280 columns: 4-5 us.
template <typename T>
__global__ __launch_bounds__(1024) void k_gan_reduce(GanReduceArgs a) {
    __shared__ float red[32][33];
    const int tx = threadIdx.x & 31, q = threadIdx.x >> 5, col = blockIdx.x * 32 + tx;
    const long long which = blockIdx.y;
    const float* src;
    long long n;
    T* out;
    if (which < 4) {
        const int bit = 2 << which;
        if (!(a.want & bit)) return;
        src = a.part + (long long)__popc(a.want & (bit - 1) & ~GAN_DGATE) * a.nblk * a.C;
        n = a.nblk;
        out = reinterpret_cast<T*>(a.out[1 + which]);
    } else {
        if (!(a.want & GAN_DGATE)) return;
        const long long item = which - 4;
        const long long b0 = a.item_rows ? item * a.item_rows / a.rows_per_block : 0;
        const long long b1 = a.item_rows ? ((item + 1) * a.item_rows - 1) / a.rows_per_block : a.nblk - 1;
        src = a.part + (long long)__popc(a.want & ~GAN_DGATE) * a.nblk * a.C + (item + b0) * a.C;
        n = b1 - b0 + 1;
        out = reinterpret_cast<T*>(a.out[0]) + item * a.C;
    }
    float s = 0.f;
    if (col < a.C) {
#pragma unroll 8
        for (long long i = q; i < n; i += 32) s += src[i * a.C + col];
    }
    red[q][tx] = s;
    __syncthreads();
    if (q == 0 && col < a.C) {
        s = 0.f;
#pragma unroll
        for (int k = 0; k < 32; ++k) s += red[k][tx];
        out[col] = (T)s;
    }
}

// Rows of 16-byte chunks: the fewest lanes per row that keep a lane at few chunks -- three in the forward, two in the backward, which holds
// four rows, the next four and five sums of them in registers -- else the whole workgroup.  Rows that are not whole aligned chunks go
// element by element.
bool chunked(int C, int per, std::initializer_list<const void*> ptrs) {
    if (C % per) return false;
    for (const void* p : ptrs)
        if ((uintptr_t)p & 15) return false;
    return true;
}

constexpr int kMaxC = 8192;

template <typename T, bool BWD, template <typename, int, int, int> class Launch>
int dispatch(GanArgs& a, bool vec, hipStream_t stream) {
    constexpr int V = Elems<T>::N;
    if (vec) {
        const int ch = a.C / V;
        if constexpr (BWD) {
            if (ch <= 16) return Launch<T, V, 16, 1>::go(a, stream);
            if (ch <= 32) return Launch<T, V, 32, 1>::go(a, stream);
            if (ch <= 64) return Launch<T, V, 64, 1>::go(a, stream);
            if (ch <= 128) return Launch<T, V, 128, 1>::go(a, stream);
            if (ch <= 256) return Launch<T, V, 256, 1>::go(a, stream);
            if (ch <= 512) return Launch<T, V, 512, 1>::go(a, stream);
            if (ch <= 1024) return Launch<T, V, 512, 2>::go(a, stream);
        } else {
            if (ch <= 16) return Launch<T, V, 16, 1>::go(a, stream);
            if (ch <= 32) return Launch<T, V, 16, 2>::go(a, stream);
            if (ch <= 48) return Launch<T, V, 16, 3>::go(a, stream);
            if (ch <= 64) return Launch<T, V, 32, 2>::go(a, stream);
            if (ch <= 96) return Launch<T, V, 32, 3>::go(a, stream);
            if (ch <= 128) return Launch<T, V, 64, 2>::go(a, stream);
            if (ch <= 192) return Launch<T, V, 64, 3>::go(a, stream);
            if (ch <= 256) return Launch<T, V, 256, 1>::go(a, stream);
            if (ch <= 512) return Launch<T, V, 256, 2>::go(a, stream);
            if (ch <= 1024) return Launch<T, V, 512, 2>::go(a, stream);
        }
        if constexpr (V == 4) return Launch<T, V, 512, 4>::go(a, stream);
        return DM_ERR_UNSUPPORTED;
    }
    if (a.C <= 256) return Launch<T, 1, 64, 4>::go(a, stream);
    if (a.C <= 2048) return Launch<T, 1, 256, 8>::go(a, stream);
    return Launch<T, 1, 1024, 8>::go(a, stream);
}

template <typename T, int VEC, int L, int NC>
struct Fwd {
    static int go(GanArgs& a, hipStream_t stream) {
        constexpr int G = threads_of(L) / L;
        // workgroups: rows of a wave two per CU, which loop over rows that are requested ahead ([24, 4096, 320] bf16 44 us against 47 with
        // eight); rows of 256 threads, whose loads wait for their barriers, eight ([24, 1024, 1280] fp32 93 against 118 us with two); rows of
        // 512 and 1024 threads, which fill a CU with two, two ([12000, 8192] bf16 164 against 181 us with eight, [9000, 5001] 167 against 193)
        const long long most = 256 * (L == 256 ? 8 : 2);
        a.rows_per_block = ((a.rows + most - 1) / most + G - 1) / G * G;
        hipLaunchKernelGGL((k_gan_fwd<T, VEC, L, NC>), dim3((unsigned)((a.rows + a.rows_per_block - 1) / a.rows_per_block)), dim3(threads_of(L)), 0, stream, a);
        DM_LAUNCH_CHECK();
        return DM_OK;
    }
};

// workgroups of the backward: two per CU (registers allow no more), whole row groups each (the rows that a workgroup of chunked 16-bit rows has
// at once, so that few rows spread out too: [16, 1136] bf16 41.6 us with 16 rows to a workgroup)
long long bwd_rows_per_block(long long rows, int C) {
    const long long per = (rows + 511) / 512, group = C <= 128 ? 16 : C <= 256 ? 8 : C <= 512 ? 4 : C <= 1024 ? 2 : 1;
    return (per + group - 1) / group * group;
}

template <typename T, int VEC, int L, int NC>
struct Bwd {
    static int go(GanArgs& a, hipStream_t stream) {
        hipLaunchKernelGGL((k_gan_bwd<T, VEC, L, NC>), dim3((unsigned)((a.rows + a.rows_per_block - 1) / a.rows_per_block)), dim3(threads_of(L)), 0, stream, a);
        DM_LAUNCH_CHECK();
        return DM_OK;
    }
};

int check_common(const void* x, const void* h, long long rows, long long item_rows, int C, const void* gate) {
    if (!x || !h || rows < 0 || C <= 0 || item_rows < 0) return DM_ERR_ARG;
    if (C > kMaxC) return DM_ERR_UNSUPPORTED;
    if (gate && item_rows && rows % item_rows) return DM_ERR_ARG;
    return DM_OK;
}

template <typename T>
int gan_fwd(const void* x, const void* h, const void* gate, long long item_rows, int post, const void* post_g, const void* post_b, int pre,
            const void* pre_g, const void* pre_b, void* y, void* z, float* stats, long long rows, int C, float scale, float eps, int rms,
            hipStream_t stream) {
    if (int rc = check_common(x, h, rows, item_rows, C, gate)) return rc;
    if (!y || (pre && !z) || ((uintptr_t)stats & 15)) return DM_ERR_ARG;
    if (!rows) return DM_OK;
    GanArgs a{};
    a.x = x; a.h = h; a.gate = gate; a.y = y; a.z = z; a.stats = stats;
    a.post = post; a.pre = pre;
    if (post) { a.post_g = post_g; a.post_b = post_b; }
    if (pre) { a.pre_g = pre_g; a.pre_b = pre_b; }
    a.rows = rows; a.item_rows = gate ? item_rows : 0; a.C = C; a.scale = scale; a.eps = eps; a.rms = rms;
    DM_ENTER();
    return dispatch<T, false, Fwd>(a, chunked(C, Elems<T>::N, {x, h, gate, a.post_g, a.post_b, a.pre_g, a.pre_b, y, z}), stream);
}

template <typename T>
int gan_bwd(const void* x, const void* h, const void* gate, long long item_rows, int post, const void* post_g, const void* post_b, int pre,
            const void* pre_g, const void* dy, const void* dz, const float* stats, void* dx, void* dh, void* dgate, void* dpost_g,
            void* dpost_b, void* dpre_g, void* dpre_b, float* ws, size_t ws_floats, long long rows, int C, float scale, float eps, int rms,
            hipStream_t stream) {
    if (int rc = check_common(x, h, rows, item_rows, C, gate)) return rc;
    if ((pre && !dz) || !stats || ((uintptr_t)stats & 15) || rows == 0) return DM_ERR_ARG;
    GanArgs a{};
    a.x = x; a.h = h; a.gate = gate; a.dy = dy; a.dz = pre ? dz : nullptr; a.dx = dx; a.dh = dh;
    a.stats = const_cast<float*>(stats); a.part = ws;
    a.post = post; a.pre = pre;
    if (post) { a.post_g = post_g; a.post_b = post_b; }
    if (pre) a.pre_g = pre_g;
    a.rows = rows; a.item_rows = gate ? item_rows : 0; a.C = C; a.scale = scale; a.eps = eps; a.rms = rms;
    a.want = (dgate && gate ? GAN_DGATE : 0) | (dpost_g && post ? GAN_DPOST_G : 0) | (dpost_b && post ? GAN_DPOST_B : 0) |
             (dpre_g && pre ? GAN_DPRE_G : 0) | (dpre_b && pre ? GAN_DPRE_B : 0);
    a.rows_per_block = bwd_rows_per_block(rows, C);
    const long long nblk = (rows + a.rows_per_block - 1) / a.rows_per_block;
    const long long items = a.item_rows ? rows / a.item_rows : 1;
    const long long need = ((long long)__builtin_popcount(a.want & ~GAN_DGATE) * nblk + (a.want & GAN_DGATE ? items + nblk : 0)) * C;
    if (a.want && (!ws || (long long)ws_floats < need)) return DM_ERR_WORKSPACE;
    if (items > 65000) return DM_ERR_UNSUPPORTED;        // grid.y of the join
    DM_ENTER();
    const bool vec = chunked(C, Elems<T>::N, {x, h, gate, a.post_g, a.post_b, a.pre_g, dy, a.dz, dx, dh});
    if (int rc = dispatch<T, true, Bwd>(a, vec, stream)) return rc;
    if (a.want) {
        GanReduceArgs r{};
        r.part = ws; r.want = a.want; r.C = C; r.nblk = nblk; r.rows_per_block = a.rows_per_block; r.item_rows = a.item_rows; r.rows = rows;
        r.items = items;
        r.out[0] = dgate; r.out[1] = dpost_g; r.out[2] = dpost_b; r.out[3] = dpre_g; r.out[4] = dpre_b;
        hipLaunchKernelGGL((k_gan_reduce<T>), dim3((unsigned)((C + 31) / 32), (unsigned)(4 + (a.want & GAN_DGATE ? items : 0))), dim3(1024), 0, stream, r);
        DM_LAUNCH_CHECK();
    }
    return DM_OK;
}

}  // namespace

extern "C" {

// fp32 words of backward workspace: five column sums of every workgroup, the gate's also per item
size_t dm_gated_add_norm_workspace_floats(long long rows, long long item_rows, int C) {
    if (rows <= 0 || C <= 0 || item_rows < 0) return 0;
    const long long per = bwd_rows_per_block(rows, C), nblk = (rows + per - 1) / per;
    const long long items = item_rows ? (rows + item_rows - 1) / item_rows : 1;
    return (size_t)((5 * nblk + items) * C);
}

#define GAN_ENTRY(T, sfx)                                                                                                                   \
    int dm_gated_add_norm_fwd_##sfx(const void* x, const void* h, const void* gate, long long item_rows, int post, const void* post_g,      \
                                    const void* post_b, int pre, const void* pre_g, const void* pre_b, void* y, void* z, float* stats,      \
                                    long long rows, int C, float scale, float eps, int rms, hipStream_t stream) {                           \
        return gan_fwd<T>(x, h, gate, item_rows, post, post_g, post_b, pre, pre_g, pre_b, y, z, stats, rows, C, scale, eps, rms, stream);   \
    }                                                                                                                                       \
    int dm_gated_add_norm_bwd_##sfx(const void* x, const void* h, const void* gate, long long item_rows, int post, const void* post_g,      \
                                    const void* post_b, int pre, const void* pre_g, const void* dy, const void* dz, const float* stats,     \
                                    void* dx, void* dh, void* dgate, void* dpost_g, void* dpost_b, void* dpre_g, void* dpre_b, float* ws,   \
                                    size_t ws_floats, long long rows, int C, float scale, float eps, int rms, hipStream_t stream) {         \
        return gan_bwd<T>(x, h, gate, item_rows, post, post_g, post_b, pre, pre_g, dy, dz, stats, dx, dh, dgate, dpost_g, dpost_b, dpre_g,  \
                          dpre_b, ws, ws_floats, rows, C, scale, eps, rms, stream);                                                         \
    }

GAN_ENTRY(__bf16, bf16)
GAN_ENTRY(_Float16, f16)
GAN_ENTRY(float, f32)

}  // extern "C"
