// Group norm with an activation over the rows of each graph, channels last: statistics per (graph, group of columns).
//
//   xh = (x - mean) * rstd,  z = xh * w + b,  out = act(z)
//   backward:  dz = g * act'(z),  gw = sum_n dz * xh,  gb = sum_n dz,  a = dz * w,
//              gx = rstd * (a - mean(a) - xh * mean(a * xh))          (means over the graph's rows and the group's columns)
//
// All sums are taken in fp64 (four fp64 operations per element; the kernels wait for memory), of differences from one value of
// the group, so the variance loses nothing to a mean far from zero, and the order of the sums, which is fixed, does not show in
// fp32.  The mean is kept in fp64 and subtracted in two fp32 pieces, so a column
// far from zero loses nothing but the bits that its own values lack.  The backward pass recomputes xh and z from x, or from the
// 8-bit values that were kept of it.
//
// Two ways to run:  graphs whose columns of one slab (whole groups, 32 columns or more) fit into the registers of a workgroup
// are read once (k_gn_small);  larger ones take a pass for the sums over row chunks, a small pass that joins them per graph and
// a pass that applies them.  Bound by memory: 3 passes over the matrix forward (2 would be the least), 5 backward (3).  1.28 M x 138
// forward: sums 135 us (5.2 TB/s), applied 280 (5.1);  backward: sums 275 (5.2), applied 423 (5.0); a large copy on the same card
// reaches 5.2.  Taking the graphs in batches of 48 ... 192 MB, so that the second read meets the memory-side cache, was measured and
// is slower (forward and backward 1.78 ... 1.37 ms against 1.23 in one piece): the ends of the many short launches cost more than the
// cache brings.  Streaming loads in the last pass: 160 001 x 256 3 % faster, 1.28 M x 138 (rows that share lines) 1 % slower, not taken.
// Small graphs (32 x 138 rows x 138): forward 9.4 us, backward 10.5 + 2.8, where the host takes 138.
#include "pack8.h"

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));

enum { ACT_NONE = 0, ACT_RELU = 1, ACT_SILU = 2, ACT_GELU = 3 };

template <int ACT>
__device__ __forceinline__ float act_fwd(float z) {
    if (ACT == ACT_RELU) return z < 0.f ? 0.f : z;              // a NaN stays
    if (ACT == ACT_SILU) return z * __builtin_amdgcn_rcpf(1.f + expf(-z));
    if (ACT == ACT_GELU) return 0.5f * z * (1.f + erff(z * 0.70710678f));
    return z;
}
template <int ACT>
__device__ __forceinline__ float act_bwd(float z) {
    if (ACT == ACT_RELU) return z > 0.f ? 1.f : (z == z ? 0.f : z);
    if (ACT == ACT_SILU) {
        const float s = __builtin_amdgcn_rcpf(1.f + expf(-z));
        return s * fmaf(z, 1.f - s, 1.f);
    }
    if (ACT == ACT_GELU) return fmaf(z * 0.39894228f, expf(-0.5f * z * z), 0.5f * (1.f + erff(z * 0.70710678f)));
    return 1.f;
}

struct GnArgs {
    const float* x; int64_t ldx;
    const int8_t* q; int64_t ldq; const uint8_t* scale; int nb;     // 8-bit form of x (backward pass of a level that kept it)
    const float* g; int64_t ldg;
    int C, groups, per;
    float eps;
    const float* w; const float* b;
    const int32_t* ptr;               // [B + 1] first row of each graph
    const int32_t* order;             // graphs that have rows, by size
    const int4* chunks;               // (graph, first row, end row, -) of row chunks, in the order of the graphs
    const int32_t* first_chunk;       // [listed + 1] first chunk of the k-th graph of that order
    float* out; int64_t ldo;          // out or gx
    double* mean; float* rstd;        // [B, groups]
    int64_t rows;                     // of x, where its 8-bit form is kept
    double2* part;                    // [chunk][C] sums over a chunk's rows, from the first chunk of a larger graph on
    double2* colsum;                  // [rows of colsum][C] column sums (dz * xh, dz): one row per small workgroup, then per large graph
    float2* gsum;                     // [B, groups] mean(a), mean(a * xh)
    int8_t* keep; uint8_t* keep_scale;                              // forward: where the 8-bit form of x goes (leading dimension ldq)
    int n_small, slab, nslabs, pad;   // pad: columns behind the last one that rows of out have for 16-byte access (zeroed)
};

// mean as two fp32 pieces: x - hi is exact where it matters, - lo brings the rest
struct Mean2 { float hi, lo; };
__device__ __forceinline__ Mean2 mean2(double m) {
    Mean2 r;
    r.hi = (float)m;
    r.lo = (float)(m - (double)r.hi);
    if (!(fabsf(r.hi) < 3.0e38f)) r.lo = 0.f;
    return r;
}
// a - mean(a) - xh * mean(a * xh), a = dz * w rounded by itself: where a is its own mean, the mean is the same rounding of the same product,
// and the gradient of a single value is zero, as it is by definition (one rounding of a - mean(a) would leave that of the mean, times
// rstd, which is 316 there).
__device__ __forceinline__ float centred(float dz, float w, float xh, float m1, float m2) { return fmaf(-xh, m2, dz * w - m1); }
__device__ __forceinline__ float normed(float x, Mean2 m, float rs) { return ((x - m.hi) - m.lo) * rs; }

__device__ __forceinline__ float value8(const GnArgs& a, int64_t n, int c) {
    return (float)a.q[n * a.ldq + c] * p8_step(a.scale[n * a.nb + (c >> 5)]);
}

__device__ __forceinline__ void store1(const GnArgs& a, int64_t n, int c, float v) {
    float* p = a.out + n * a.ldo + c;
    p[0] = v;
    if (c == a.C - 1)
        for (int i = 1; i <= a.pad; ++i) p[i] = 0.f;
}

// Sums of the columns [0, sc) of red[ty][c] over ty, then of the columns of each group, in a fixed order.  Every thread calls
// it; the column sums are left in red[0][c], the group sums in grp[j].
__device__ __forceinline__ void reduce_slab(double2* red, double2* grp, int sc, int ty_n, int per, int nt, bool active, int tx, int ty) {
    int s = 1;
    while (s < ty_n) s <<= 1;
    for (s >>= 1; s > 0; s >>= 1) {
        __syncthreads();
        if (active && ty < s && ty + s < ty_n) {
            double2 u = red[ty * sc + tx];
            const double2 v = red[(ty + s) * sc + tx];
            u.x += v.x; u.y += v.y;
            red[ty * sc + tx] = u;
        }
    }
    __syncthreads();
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, nw = nt >> 6;
    for (int j = wave; j * per < sc; j += nw) {
        double u = 0.0, v = 0.0;
        for (int c = lane; c < per; c += 64) {
            const double2 t = red[j * per + c];
            u += t.x; v += t.y;
        }
        u = hgv_wave_sum_d(u); v = hgv_wave_sum_d(v);
        if (lane == 0) grp[j] = make_double2(u, v);
    }
    __syncthreads();
}

// What the sums of a (graph, group) are differences from: its first value.
__device__ __forceinline__ double pivot_of(const GnArgs& a, int graph, int j) {
    return (double)a.x[(int64_t)a.ptr[graph] * a.ldx + (int64_t)j * a.per];
}

__device__ __forceinline__ void stats_of(double2 s, double pivot, double count, float eps, double* mean, float* rstd) {
    const double m = s.x / count;
    double var = s.y / count - m * m;
    var = var < 0.0 ? 0.0 : var;                                // rounding only; a NaN stays
    *mean = pivot + m;
    *rstd = (float)(1.0 / sqrt(var + (double)eps));
}

// ---- graphs whose slab fits into registers: one read -------------------------------------------------------------------
// Thread (tx, ty) holds column tx of the slab in rows ty, ty + TY, ... (at most R of them).  A workgroup walks the small graphs
// blockIdx.x, + gridDim.x, ...; in the backward pass it keeps its column sums of dz * xh and dz over all of them, so there is
// one partial row per workgroup whatever the number of graphs.
template <int NT, int R, int ACT, bool BWD, bool Q8>
__global__ __launch_bounds__(NT) void k_gn_small(const GnArgs a) {
    __shared__ double2 red[NT];
    __shared__ double2 grp[NT];
    const int c0 = blockIdx.y * a.slab, sc = min(a.slab, a.C - c0);
    const int ty_n = NT / sc, ty = threadIdx.x / sc, tx = threadIdx.x - ty * sc;
    const bool active = ty < ty_n;
    const int col = c0 + (active ? tx : 0), j = (active ? tx : 0) / a.per;
    const float w = a.w ? a.w[col] : 1.f, b = a.b ? a.b[col] : 0.f;
    double sw = 0.0, sb = 0.0;
    for (int k = blockIdx.x; k < a.n_small; k += gridDim.x) {
        const int graph = a.order[k];
        const int64_t r0 = a.ptr[graph];
        const int n = (int)(a.ptr[graph + 1] - r0);
        const double count = (double)n * a.per;
        float x[R], g[R];
        double s1 = 0.0, s2 = 0.0;
        if (active) {
            const float* px = Q8 ? nullptr : a.x + (r0 + ty) * a.ldx + col;
            const float* pg = BWD ? a.g + (r0 + ty) * a.ldg + col : nullptr;
#pragma unroll
            for (int i = 0; i < R; ++i) {
                const int r = ty + i * ty_n;
                x[i] = 0.f;
                if (r < n) {
                    x[i] = Q8 ? value8(a, r0 + r, col) : *px;
                    if (BWD) g[i] = *pg;
                }
                if (!Q8) px += ty_n * a.ldx;
                if (BWD) pg += ty_n * a.ldg;
            }
        }
        Mean2 m; float rs;
        if (!BWD) {
            const double pivot = n > 0 ? pivot_of(a, graph, c0 / a.per + j) : 0.0;
            if (active) {
#pragma unroll
                for (int i = 0; i < R; ++i)
                    if (ty + i * ty_n < n) {
                        const double v = (double)x[i] - pivot;
                        s1 += v; s2 = fma(v, v, s2);
                    }
                red[ty * sc + tx] = make_double2(s1, s2);
            }
            reduce_slab(red, grp, sc, ty_n, a.per, NT, active, tx, ty);
            double mean;
            stats_of(grp[j], pivot, count, a.eps, &mean, &rs);
            m = mean2(mean);
            if (active && ty == 0 && tx == j * a.per && n > 0) {
                a.mean[(int64_t)graph * a.groups + c0 / a.per + j] = mean;
                a.rstd[(int64_t)graph * a.groups + c0 / a.per + j] = rs;
            }
            if (active) {
#pragma unroll
                for (int i = 0; i < R; ++i) {
                    const int r = ty + i * ty_n;
                    if (r < n) store1(a, r0 + r, col, act_fwd<ACT>(fmaf(normed(x[i], m, rs), w, b)));
                }
            }
        } else if (n > 0) {                                     // n is the same for the whole workgroup
            m = mean2(a.mean[(int64_t)graph * a.groups + c0 / a.per + j]);
            rs = a.rstd[(int64_t)graph * a.groups + c0 / a.per + j];
            if (active) {
#pragma unroll
                for (int i = 0; i < R; ++i)
                    if (ty + i * ty_n < n) {
                        x[i] = normed(x[i], m, rs);
                        g[i] *= act_bwd<ACT>(fmaf(x[i], w, b));
                        s1 += (double)g[i]; s2 = fma((double)g[i], (double)x[i], s2);
                    }
                sb += s1; sw += s2;
                red[ty * sc + tx] = make_double2(s1 * (double)w, s2 * (double)w);
            }
            reduce_slab(red, grp, sc, ty_n, a.per, NT, active, tx, ty);
            const float m1 = (float)(grp[j].x / count), m2 = (float)(grp[j].y / count);
            if (active && a.out) {
#pragma unroll
                for (int i = 0; i < R; ++i) {
                    const int r = ty + i * ty_n;
                    if (r < n) store1(a, r0 + r, col, rs * centred(g[i], w, x[i], m1, m2));
                }
            }
        }
        __syncthreads();                                        // red and grp are written again
    }
    if (BWD && a.colsum) {
        if (active) red[ty * sc + tx] = make_double2(sw, sb);
        reduce_slab(red, grp, sc, ty_n, a.per, NT, active, tx, ty);
        if (active && ty == 0) a.colsum[(int64_t)blockIdx.x * a.C + col] = red[tx];
    }
}

// ---- larger graphs: sums over row chunks, joined per graph, applied -------------------------------------------------------
template <int VEC, bool Q8>
__device__ __forceinline__ void load_x(const GnArgs& a, int64_t n, int c, float v[VEC]) {
    if (Q8) {
        if (VEC == 4) p8_values4(*(const uint32_t*)(a.q + n * a.ldq + c), a.scale[n * a.nb + (c >> 5)], v);
        else v[0] = value8(a, n, c);
    } else if (VEC == 4) {
        const float4 t = *(const float4*)(a.x + n * a.ldx + c);
        v[0] = t.x; v[VEC > 1 ? 1 : 0] = t.y; v[VEC > 2 ? 2 : 0] = t.z; v[VEC > 3 ? 3 : 0] = t.w;
    } else {
        v[0] = a.x[n * a.ldx + c];
    }
}
template <int VEC>
__device__ __forceinline__ void load_g(const GnArgs& a, int64_t n, int c, float v[VEC]) {
    if (VEC == 4) {
        const float4 t = *(const float4*)(a.g + n * a.ldg + c);
        v[0] = t.x; v[VEC > 1 ? 1 : 0] = t.y; v[VEC > 2 ? 2 : 0] = t.z; v[VEC > 3 ? 3 : 0] = t.w;
    } else {
        v[0] = a.g[n * a.ldg + c];
    }
}

// thread -> (column block, row) of a chunk
struct GnLane { int c, ty, ty_n, tx, tx_n; bool live; };
template <int VEC, bool PACK = false>                           // PACK: eight lanes to a block of 32 columns, also to the last one
__device__ __forceinline__ GnLane gn_lane(const GnArgs& a) {
    GnLane l;
    const int c0 = blockIdx.y * 256 * VEC;
    l.tx_n = min(256, (a.C - c0 + VEC - 1) / VEC);
    if (PACK) l.tx_n = (l.tx_n + 7) & ~7;
    l.ty_n = 256 / l.tx_n;
    l.ty = threadIdx.x / l.tx_n;
    l.tx = threadIdx.x - l.ty * l.tx_n;
    l.c = c0 + l.tx * VEC;
    l.live = l.ty < l.ty_n;
    return l;
}

template <int VEC>
struct GnCols { Mean2 m[VEC]; float rs[VEC], w[VEC], b[VEC]; int j[VEC]; };
template <int VEC>
__device__ __forceinline__ void gn_cols(const GnArgs& a, int graph, int c, GnCols<VEC>& k) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
        const int cc = min(c + i, a.C - 1);
        k.j[i] = cc / a.per;
        k.m[i] = mean2(a.mean[(int64_t)graph * a.groups + k.j[i]]);
        k.rs[i] = a.rstd[(int64_t)graph * a.groups + k.j[i]];
        k.w[i] = a.w ? a.w[cc] : 1.f;
        k.b[i] = a.b ? a.b[cc] : 0.f;
    }
}

// Sums per column of a chunk -> part.  Forward: x - pivot and its square.  Backward: dz and dz * xh (weighted by w when they are joined).
template <int VEC, int ACT, bool BWD, bool Q8>
__global__ __launch_bounds__(256) void k_gn_sums(const GnArgs a, const int chunk0) {
    __shared__ double2 red[256 * VEC];
    const GnLane l = gn_lane<VEC>(a);
    const int4 ch = a.chunks[chunk0 + blockIdx.x];
    double s1[VEC], s2[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) s1[i] = s2[i] = 0.0;
    if (l.live) {
        GnCols<VEC> k;
        double pivot[VEC];
        if (BWD) gn_cols<VEC>(a, ch.x, l.c, k);
        else {
#pragma unroll
            for (int i = 0; i < VEC; ++i) pivot[i] = pivot_of(a, ch.x, min(l.c + i, a.C - 1) / a.per);
        }
#pragma unroll 4
        for (int n = ch.y + l.ty; n < ch.z; n += l.ty_n) {
            float v[VEC];
            load_x<VEC, Q8>(a, n, l.c, v);
            if (BWD) {
                float g[VEC];
                load_g<VEC>(a, n, l.c, g);
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    const float xh = normed(v[i], k.m[i], k.rs[i]);
                    const float dz = g[i] * act_bwd<ACT>(fmaf(xh, k.w[i], k.b[i]));
                    s1[i] += (double)dz; s2[i] = fma((double)dz, (double)xh, s2[i]);
                }
            } else {
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    const double d = (double)v[i] - pivot[i];
                    s1[i] += d; s2[i] = fma(d, d, s2[i]);
                }
            }
        }
#pragma unroll
        for (int i = 0; i < VEC; ++i) red[(l.ty * l.tx_n + l.tx) * VEC + i] = make_double2(s1[i], s2[i]);
    }
    int s = 1;
    while (s < l.ty_n) s <<= 1;
    const int width = l.tx_n * VEC;
    for (s >>= 1; s > 0; s >>= 1) {
        __syncthreads();
        if (l.live && l.ty < s && l.ty + s < l.ty_n) {
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                double2 u = red[l.ty * width + l.tx * VEC + i];
                const double2 v = red[(l.ty + s) * width + l.tx * VEC + i];
                u.x += v.x; u.y += v.y;
                red[l.ty * width + l.tx * VEC + i] = u;
            }
        }
    }
    if (l.live && l.ty == 0) {
#pragma unroll
        for (int i = 0; i < VEC; ++i)
            if (l.c + i < a.C) a.part[(int64_t)blockIdx.x * a.C + l.c + i] = red[l.tx * VEC + i];
    }
}

// One workgroup per (large graph, slab of whole groups): adds the sums of the graph's chunks and forms the group's statistics
// (forward) or the two means of the backward pass and the graph's row of column sums.
template <bool BWD>
__global__ __launch_bounds__(1024) void k_gn_join(const GnArgs a, const int chunk0, const int colrow0) {
    __shared__ double2 red[1024];
    __shared__ double2 grp[1024];
    const int k = a.n_small + blockIdx.x, graph = a.order[k];
    const int ch0 = a.first_chunk[k] - chunk0, ch1 = a.first_chunk[k + 1] - chunk0;
    const double count = (double)(a.ptr[graph + 1] - a.ptr[graph]) * a.per;
    const int c0 = blockIdx.y * a.slab, sc = min(a.slab, a.C - c0);
    double2 total = make_double2(0.0, 0.0);
    if (sc <= 1024) {
        const int ty_n = 1024 / sc, ty = threadIdx.x / sc, tx = threadIdx.x - ty * sc;
        const bool active = ty < ty_n;
        double u = 0.0, v = 0.0;
        if (active) {
#pragma unroll 4
            for (int c = ch0 + ty; c < ch1; c += ty_n) {
                const double2 t = a.part[(int64_t)c * a.C + c0 + tx];
                u += t.x; v += t.y;
            }
            red[ty * sc + tx] = make_double2(u, v);
        }
        if (BWD) {
            // column sums first (unweighted), then the weighted group sums
            int s = 1;
            while (s < ty_n) s <<= 1;
            for (s >>= 1; s > 0; s >>= 1) {
                __syncthreads();
                if (active && ty < s && ty + s < ty_n) {
                    red[ty * sc + tx].x += red[(ty + s) * sc + tx].x;
                    red[ty * sc + tx].y += red[(ty + s) * sc + tx].y;
                }
            }
            if (active && ty == 0) {
                const double2 t = red[tx];
                if (a.colsum) a.colsum[(int64_t)(colrow0 + blockIdx.x) * a.C + c0 + tx] = make_double2(t.y, t.x);
                const double w = a.w ? (double)a.w[c0 + tx] : 1.0;
                red[tx] = make_double2(t.x * w, t.y * w);
            }
            reduce_slab(red, grp, sc, 1, a.per, 1024, active, tx, ty);
        } else {
            reduce_slab(red, grp, sc, ty_n, a.per, 1024, active, tx, ty);
        }
        const int j = threadIdx.x;
        if (j < sc / a.per) total = grp[j];
    } else {                                                    // one group wider than the workgroup: all of it belongs to one sum
        double u = 0.0, v = 0.0;
        for (int c = threadIdx.x; c < sc; c += 1024) {
            double p = 0.0, q = 0.0;
            for (int r = ch0; r < ch1; ++r) {
                const double2 t = a.part[(int64_t)r * a.C + c0 + c];
                p += t.x; q += t.y;
            }
            if (BWD && a.colsum) a.colsum[(int64_t)(colrow0 + blockIdx.x) * a.C + c0 + c] = make_double2(q, p);
            const double w = BWD && a.w ? (double)a.w[c0 + c] : 1.0;
            u += p * w; v += q * w;
        }
        red[threadIdx.x] = make_double2(u, v);
        reduce_slab(red, grp, 1024, 1, 1024, 1024, true, threadIdx.x, 0);
        if (threadIdx.x == 0) total = grp[0];
    }
    const int j = threadIdx.x;
    if (j < sc / a.per) {
        const int64_t at = (int64_t)graph * a.groups + c0 / a.per + j;
        if (BWD) a.gsum[at] = make_float2((float)(total.x / count), (float)(total.y / count));
        else stats_of(total, pivot_of(a, graph, c0 / a.per + j), count, a.eps, a.mean + at, a.rstd + at);
    }
}

// Streaming stores (the output does not push out what is read again: 8 bundled graphs 60 -> 51 us), and the chunks from the last to
// the first, since the last ones read by the sums are the ones still in the memory-side cache (1.28 M x 138: 2 %).  PACK: the 8-bit
// form of x on the way.
template <int VEC, int ACT, bool BWD, bool Q8, bool PACK = false>
__global__ __launch_bounds__(256) void k_gn_apply(const GnArgs a, const int chunk0) {
    static_assert(!PACK || (VEC == 4 && !BWD && !Q8), "packs x where it is read in 16 bytes");
    const GnLane l = gn_lane<VEC, PACK>(a);
    if (!l.live) return;                                        // whole blocks of eight lanes leave: the maxima below stay inside one
    const int4 ch = a.chunks[chunk0 + (int)(gridDim.x - 1 - blockIdx.x)];
    GnCols<VEC> k;
    gn_cols<VEC>(a, ch.x, l.c, k);
    float m1[VEC], m2[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
        if (BWD) {
            const float2 t = a.gsum[(int64_t)ch.x * a.groups + k.j[i]];
            m1[i] = t.x; m2[i] = t.y;
        }
    }
    const bool stored = !PACK || l.c < a.C;
#pragma unroll 1
    for (int n = ch.y + l.ty; n < ch.z; n += l.ty_n) {
        float v[VEC], o[VEC];
        if (stored) {
            load_x<VEC, Q8>(a, n, l.c, v);
        } else {
#pragma unroll
            for (int i = 0; i < VEC; ++i) v[i] = 0.f;
        }
        if (PACK) {
            float p[4];
            uint32_t m = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                p[i] = l.c + i < a.C ? v[VEC > i ? i : 0] : 0.f;
                m = max(m, __float_as_uint(p[i]) & 0x7fffffffu);
            }
            const int byte = p8_byte(p8_max8(m));
            const uint32_t w = p8_quantise4(p, byte);
            if (l.c < a.ldq) __builtin_nontemporal_store(w, (uint32_t*)(a.keep + (int64_t)n * a.ldq + l.c));
            if ((threadIdx.x & 7) == 0) a.keep_scale[(int64_t)n * a.nb + (l.c >> 5)] = (uint8_t)byte;
        }
        if (BWD) {
            float g[VEC];
            load_g<VEC>(a, n, l.c, g);
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                const float xh = normed(v[i], k.m[i], k.rs[i]);
                const float dz = g[i] * act_bwd<ACT>(fmaf(xh, k.w[i], k.b[i]));
                o[i] = k.rs[i] * centred(dz, k.w[i], xh, m1[i], m2[i]);
            }
        } else {
#pragma unroll
            for (int i = 0; i < VEC; ++i) o[i] = act_fwd<ACT>(fmaf(normed(v[i], k.m[i], k.rs[i]), k.w[i], k.b[i]));
        }
        if (VEC == 4) {
#pragma unroll
            for (int i = 0; i < VEC; ++i)
                if (l.c + i >= a.C) o[i] = 0.f;                 // pad columns
            const f32x4 t = {o[0], o[VEC > 1 ? 1 : 0], o[VEC > 2 ? 2 : 0], o[VEC > 3 ? 3 : 0]};
            if (stored) __builtin_nontemporal_store(t, (f32x4*)(a.out + (int64_t)n * a.ldo + l.c));
        } else {
            store1(a, n, l.c, o[0]);
        }
    }
}

// gw, gb: the column sums' rows added in order.
__global__ __launch_bounds__(1024) void k_gn_affine(const double2* __restrict__ colsum, const int rows, const int C, float* __restrict__ gw,
                                                    float* __restrict__ gb) {
    __shared__ double2 red[1024];
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5, c = blockIdx.x * 32 + tx;
    double u = 0.0, v = 0.0;
    if (c < C) {
#pragma unroll 4
        for (int r = ty; r < rows; r += 32) {
            const double2 t = colsum[(int64_t)r * C + c];
            u += t.x; v += t.y;
        }
    }
    red[threadIdx.x] = make_double2(u, v);
    for (int s = 16; s > 0; s >>= 1) {
        __syncthreads();
        if (ty < s) {
            red[threadIdx.x].x += red[threadIdx.x + 32 * s].x;
            red[threadIdx.x].y += red[threadIdx.x + 32 * s].y;
        }
    }
    if (ty == 0 && c < C) {
        if (gw) gw[c] = (float)red[tx].x;
        if (gb) gb[c] = (float)red[tx].y;
    }
}

// ---- host side --------------------------------------------------------------------------------------------------------
constexpr int SMALL_R = 16;                                     // rows that a thread of k_gn_small holds
constexpr int SMALL_WGS = 2048;                                 // workgroups of it per slab

int gn_slab(int C, int per) {                                   // whole groups, at least 32 columns
    const int m = per >= 32 ? 1 : (32 + per - 1) / per;
    return min(C, m * per);
}
// Rows up to which a graph takes k_gn_small: what 1024 threads hold.
int gn_small_rows(int C, int per) {
    const int slab = gn_slab(C, per);
    return slab > 1024 ? 0 : 1024 / slab * SMALL_R;
}

template <int ACT, bool BWD, bool Q8>
int gn_launch(const GnArgs& a, int listed, int small_rows, int chunk0, int chunk1, float* gw, float* gb, hipStream_t stream) {
    const int small_wgs = min(a.n_small, SMALL_WGS);
    if (a.n_small > 0) {
        const dim3 grid((unsigned)small_wgs, (unsigned)a.nslabs);
        if (a.slab <= 256 && small_rows <= 256 / a.slab * SMALL_R)
            hipLaunchKernelGGL((k_gn_small<256, SMALL_R, ACT, BWD, Q8>), grid, dim3(256), 0, stream, a);
        else if (a.slab <= 512 && small_rows <= 512 / a.slab * SMALL_R)
            hipLaunchKernelGGL((k_gn_small<512, SMALL_R, ACT, BWD, Q8>), grid, dim3(512), 0, stream, a);
        else
            hipLaunchKernelGGL((k_gn_small<1024, SMALL_R, ACT, BWD, Q8>), grid, dim3(1024), 0, stream, a);
    }
    const bool vec = (Q8 || (hgv_aligned(a.x, 16) && a.ldx % 4 == 0 && a.ldx >= (a.C + 3) / 4 * 4)) &&
                     (!BWD || (hgv_aligned(a.g, 16) && a.ldg % 4 == 0 && a.ldg >= (a.C + 3) / 4 * 4)) &&
                     (!a.out || (hgv_aligned(a.out, 16) && a.ldo % 4 == 0 && a.ldo >= (a.C + 3) / 4 * 4));
    const unsigned slabs = (unsigned)hgv_cdiv(a.C, vec ? 1024 : 256);
    // The 8-bit form: with the last pass where that reads every row (320 000 rows forward: 20 columns 50 -> 46 us, 138 columns
    // 127 -> 110, 256 columns 248 -> 197), else by itself.
    const bool keeps = !BWD && a.keep && vec && a.n_small == 0;
    if (!BWD && a.keep && !keeps) {
        const int rc = hgv_pack8(a.x, a.ldx, a.rows, a.C, a.keep, a.ldq, a.keep_scale, stream);
        if (rc) return rc;
    }
    if (listed > a.n_small) {
        const dim3 grid((unsigned)(chunk1 - chunk0), slabs);
        if (vec) hipLaunchKernelGGL((k_gn_sums<4, ACT, BWD, Q8>), grid, dim3(256), 0, stream, a, chunk0);
        else hipLaunchKernelGGL((k_gn_sums<1, ACT, BWD, Q8>), grid, dim3(256), 0, stream, a, chunk0);
        hipLaunchKernelGGL(k_gn_join<BWD>, dim3((unsigned)(listed - a.n_small), (unsigned)a.nslabs), dim3(1024), 0, stream, a, chunk0,
                           small_wgs);
        if (a.out) {
            if (!BWD && keeps) hipLaunchKernelGGL((k_gn_apply<4, ACT, false, false, true>), grid, dim3(256), 0, stream, a, chunk0);
            else if (vec) hipLaunchKernelGGL((k_gn_apply<4, ACT, BWD, Q8>), grid, dim3(256), 0, stream, a, chunk0);
            else hipLaunchKernelGGL((k_gn_apply<1, ACT, BWD, Q8>), grid, dim3(256), 0, stream, a, chunk0);
        }
    }
    if (BWD && a.colsum)
        hipLaunchKernelGGL(k_gn_affine, dim3((unsigned)hgv_cdiv(a.C, 32)), dim3(1024), 0, stream, a.colsum,
                           small_wgs + listed - a.n_small, a.C, gw, gb);
    HGV_CHECK_LAUNCH(BWD ? "group_norm_bwd" : "group_norm_fwd");
    return HGV_OK;
}

int gn_check(const GnArgs& a, int num_graphs, int listed, int n_small, int small_rows, int chunk0, int chunk1, const char* what) {
    HGV_REQUIRE(a.C > 0 && a.groups > 0 && a.C % a.groups == 0, HGV_EINVAL, "%s: %d columns in %d groups", what, a.C, a.groups);
    HGV_REQUIRE(listed >= 0 && listed <= num_graphs && n_small >= 0 && n_small <= listed && chunk0 >= 0 && chunk1 - chunk0 >= listed - n_small, HGV_EINVAL, "%s: bad graph counts", what);
    HGV_REQUIRE(a.ptr && a.order && a.chunks && a.first_chunk && a.mean && a.rstd, HGV_EINVAL, "%s: null buffer", what);
    HGV_REQUIRE(n_small == 0 || small_rows <= gn_small_rows(a.C, a.per), HGV_EINVAL,
                "%s: graphs of %d rows do not fit the one-read kernel", what, small_rows);
    HGV_REQUIRE(hgv_cdiv(a.C, 256) <= 65535, HGV_EUNSUPPORTED, "%s: too many columns", what);
    return HGV_OK;
}

}  // namespace

extern "C" int hgv_group_norm_small_rows(int C, int groups) {
    return C > 0 && groups > 0 && C % groups == 0 ? gn_small_rows(C, C / groups) : 0;
}

extern "C" size_t hgv_group_norm_ws(int64_t n_chunks, int num_graphs, int listed, int n_small, int C, int groups, int backward) {
    size_t n = hgv_align256((size_t)n_chunks * C * sizeof(double2));
    if (backward) {
        n += hgv_align256((size_t)(min(n_small, SMALL_WGS) + listed - n_small) * C * sizeof(double2));
        n += hgv_align256((size_t)num_graphs * groups * sizeof(float2));
    }
    return n + 256;
}

static int gn_fwd(const float* x, int64_t ldx, int C, int groups, int act, float eps, const float* w, const float* b,
                                  const int32_t* ptr, const int32_t* order, const int32_t* chunks, const int32_t* first_chunk,
                                  int num_graphs, int listed, int n_small, int small_rows, int chunk0, int chunk1,
                                  int64_t rows, int8_t* q, int64_t ldq, uint8_t* scale, float* out, int64_t ldo, double* mean, float* rstd, void* ws, size_t ws_bytes, hipStream_t stream) {
    GnArgs a = {};
    a.x = x; a.ldx = ldx; a.C = C; a.groups = groups; a.per = groups > 0 ? C / groups : 0; a.eps = eps; a.w = w; a.b = b;
    a.ptr = ptr; a.order = order; a.chunks = (const int4*)chunks; a.first_chunk = first_chunk; a.out = out; a.ldo = ldo;
    a.mean = mean; a.rstd = rstd; a.n_small = n_small;
    a.rows = rows; a.keep = q; a.ldq = ldq; a.keep_scale = scale; a.nb = (C + 31) / 32;
    const int rc = gn_check(a, num_graphs, listed, n_small, small_rows, chunk0, chunk1, "group_norm_fwd");
    if (rc) return rc;
    HGV_REQUIRE(x && out && ldx >= C && ldo >= C, HGV_EINVAL, "group_norm_fwd: null buffer or bad leading dimension");
    HGV_REQUIRE(ws_bytes >= hgv_group_norm_ws(chunk1 - chunk0, num_graphs, listed, n_small, C, groups, 0) && hgv_aligned(ws, 256), HGV_EWORKSPACE,
                "group_norm_fwd: workspace too small or misaligned");
    a.pad = C % 4 && a.out && a.ldo >= (C + 3) / 4 * 4 ? 4 - C % 4 : 0;
    a.slab = gn_slab(C, a.per); a.nslabs = (int)hgv_cdiv(C, a.slab);
    HGV_REQUIRE(a.nslabs <= 65535, HGV_EUNSUPPORTED, "group_norm_fwd: too many columns");
    a.part = (double2*)ws;
    switch (act) {
        case ACT_NONE: return gn_launch<ACT_NONE, false, false>(a, listed, small_rows, chunk0, chunk1, nullptr, nullptr, stream);
        case ACT_RELU: return gn_launch<ACT_RELU, false, false>(a, listed, small_rows, chunk0, chunk1, nullptr, nullptr, stream);
        case ACT_SILU: return gn_launch<ACT_SILU, false, false>(a, listed, small_rows, chunk0, chunk1, nullptr, nullptr, stream);
        case ACT_GELU: return gn_launch<ACT_GELU, false, false>(a, listed, small_rows, chunk0, chunk1, nullptr, nullptr, stream);
    }
    hgv_set_error("group_norm_fwd: unknown activation %d", act);
    return HGV_EINVAL;
}

extern "C" int hgv_group_norm_fwd(const float* x, int64_t ldx, int C, int groups, int act, float eps, const float* w, const float* b,
                                  const int32_t* ptr, const int32_t* order, const int32_t* chunks, const int32_t* first_chunk,
                                  int num_graphs, int listed, int n_small, int small_rows, int chunk0, int chunk1,
                                  float* out, int64_t ldo, double* mean, float* rstd, void* ws, size_t ws_bytes, hipStream_t stream) {
    return gn_fwd(x, ldx, C, groups, act, eps, w, b, ptr, order, chunks, first_chunk, num_graphs, listed, n_small, small_rows, chunk0, chunk1,
                  0, nullptr, 0, nullptr, out, ldo, mean, rstd, ws, ws_bytes, stream);
}

extern "C" int hgv_group_norm_fwd8(const float* x, int64_t ldx, int C, int groups, int act, float eps, const float* w, const float* b,
                                   const int32_t* ptr, const int32_t* order, const int32_t* chunks, const int32_t* first_chunk,
                                   int num_graphs, int listed, int n_small, int small_rows, int chunk0, int chunk1, int64_t rows,
                                   int8_t* q, int64_t ldq, uint8_t* scale, float* out, int64_t ldo, double* mean, float* rstd, void* ws,
                                   size_t ws_bytes, hipStream_t stream) {
    HGV_REQUIRE(rows > 0 && q && scale && ldq >= C && ldq % 16 == 0 && ldq <= 32 * (int64_t)((C + 31) / 32) && hgv_aligned(q, 16), HGV_EINVAL,
                "group_norm_fwd8: null / misaligned buffer or bad leading dimension");
    return gn_fwd(x, ldx, C, groups, act, eps, w, b, ptr, order, chunks, first_chunk, num_graphs, listed, n_small, small_rows, chunk0, chunk1,
                  rows, q, ldq, scale, out, ldo, mean, rstd, ws, ws_bytes, stream);
}

template <bool Q8>
static int gn_bwd(int act, const GnArgs& a, int listed, int small_rows, int chunk0, int chunk1, float* gw, float* gb,
                  hipStream_t stream) {
    switch (act) {
        case ACT_NONE: return gn_launch<ACT_NONE, true, Q8>(a, listed, small_rows, chunk0, chunk1, gw, gb, stream);
        case ACT_RELU: return gn_launch<ACT_RELU, true, Q8>(a, listed, small_rows, chunk0, chunk1, gw, gb, stream);
        case ACT_SILU: return gn_launch<ACT_SILU, true, Q8>(a, listed, small_rows, chunk0, chunk1, gw, gb, stream);
        case ACT_GELU: return gn_launch<ACT_GELU, true, Q8>(a, listed, small_rows, chunk0, chunk1, gw, gb, stream);
    }
    hgv_set_error("group_norm_bwd: unknown activation %d", act);
    return HGV_EINVAL;
}

extern "C" int hgv_group_norm_bwd(const float* g, int64_t ldg, const float* x, int64_t ldx, const int8_t* q, int64_t ldq,
                                  const uint8_t* scale, int C, int groups, int act, const float* w, const float* b, const int32_t* ptr,
                                  const int32_t* order, const int32_t* chunks, const int32_t* first_chunk, int num_graphs, int listed,
                                  int n_small, int small_rows, int chunk0, int chunk1, const double* mean,
                                  const float* rstd, float* gx, int64_t ldgx, float* gw, float* gb, void* ws, size_t ws_bytes,
                                  hipStream_t stream) {
    GnArgs a = {};
    a.x = x; a.ldx = ldx; a.q = q; a.ldq = ldq; a.scale = scale; a.nb = (C + 31) / 32; a.g = g; a.ldg = ldg;
    a.C = C; a.groups = groups; a.per = groups > 0 ? C / groups : 0; a.w = w; a.b = b;
    a.ptr = ptr; a.order = order; a.chunks = (const int4*)chunks; a.first_chunk = first_chunk; a.out = gx; a.ldo = ldgx;
    a.mean = (double*)mean; a.rstd = (float*)rstd; a.n_small = n_small;
    const int rc = gn_check(a, num_graphs, listed, n_small, small_rows, chunk0, chunk1, "group_norm_bwd");
    if (rc) return rc;
    HGV_REQUIRE(g && ldg >= C && (!gx || ldgx >= C) && (gx || gw || gb), HGV_EINVAL, "group_norm_bwd: null buffer or bad leading dimension");
    HGV_REQUIRE(q ? (scale && ldq >= C && ldq % 16 == 0 && hgv_aligned(q, 16)) : (x && ldx >= C), HGV_EINVAL,
                "group_norm_bwd: needs x, or its 8-bit form");
    HGV_REQUIRE(ws_bytes >= hgv_group_norm_ws(chunk1 - chunk0, num_graphs, listed, n_small, C, groups, 1) && hgv_aligned(ws, 256), HGV_EWORKSPACE,
                "group_norm_bwd: workspace too small or misaligned");
    a.pad = C % 4 && a.out && a.ldo >= (C + 3) / 4 * 4 ? 4 - C % 4 : 0;
    a.slab = gn_slab(C, a.per); a.nslabs = (int)hgv_cdiv(C, a.slab);
    HGV_REQUIRE(a.nslabs <= 65535, HGV_EUNSUPPORTED, "group_norm_bwd: too many columns");
    char* p = (char*)ws;
    a.part = (double2*)p;
    p += hgv_align256((size_t)(chunk1 - chunk0) * C * sizeof(double2));
    if (gw || gb) a.colsum = (double2*)p;
    p += hgv_align256((size_t)(min(n_small, SMALL_WGS) + listed - n_small) * C * sizeof(double2));
    a.gsum = (float2*)p;
    return q ? gn_bwd<true>(act, a, listed, small_rows, chunk0, chunk1, gw, gb, stream)
             : gn_bwd<false>(act, a, listed, small_rows, chunk0, chunk1, gw, gb, stream);
}
