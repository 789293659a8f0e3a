// Norms before and after a block, with the block's gate, scale and residual, in one pass each way.
//
//   v = norm_after(u) * wa + ba          the block's output, normalised (or v = u)
//   y = r + scale * g * v                g: none, a row for every `gate_rows` rows, or a byte mask
//   n = norm_before(y) * wb + bb         what the next block reads (optional)
//   norm: "layer" (x - mean) / sqrt(var + eps), "rms" x / sqrt(mean(x^2) + eps)
//
// Backward, with a^ and b^ the normalised values, dt = dy + norm_before'(dn):
//   norm'(d) = rstd * (d w - mean(d w) - ^ mean(d w ^))   (the first mean only for "layer")
//   dr = dt;  dg = scale v dt;  dv = scale g dt;  du = norm_after'(dv);  dw = sum_rows d ^;  db = sum_rows d
//
// Bound: HBM.  Every operand is read once and every result written once; a row lives in the registers of the lanes
// that read it (16 lanes up to 128 elements, a wave up to 768, a workgroup up to 4096), y is made again in the
// backward from u and r instead of being read.  Statistics, sums and y are f32; n is taken from the f32 y, not
// from its rounded copy.  Column sums (affine and broadcast-gate gradients) stay in registers over a workgroup's
// rows, then go to the workspace, one row a workgroup, and are added by a second kernel in a fixed order: no atomics.
// Operands are reached through buffer descriptors, for which a place outside a row, or an operand that is not there, is an
// offset out of reach and no branch: with branches round every access, and the scalar registers their masks took, the
// waves spent more time on those than on the rows (45 -> 32 us forward, 113 -> 53 us backward with its column sums for 32,768 x 640 bf16 with
// gate, residual and both norms; 168 and 252 MB, that is 5.3 and 4.8 TB/s).  What the backward still spills are scalar registers (23 to 100,
// the descriptors themselves, into vector lanes), and at widths of 513 to 768 that do not divide into vectors 22 to 30 vector registers: a
// single wave a SIMD would hold them, and is slower (65,536 x 637 bf16: 196 us instead of 174).  16-bit rows beyond 2048 use 12 bytes of scratch
// a lane.
#include "elem.h"

namespace {

constexpr int THREADS = 256;
constexpr int MAX_D = PCLIP_NORM_MAX_D;
// workgroups of a forward, which then take row after row: four a compute unit, two for the widest rows, of which a workgroup has as much
// under way as two others (8192 x 4096 with gate and both norms, bf16: 78 us with two, 97 with four; f32 without a gate 76 and 79)
constexpr int fwd_blocks(int d) { return d > 2048 ? 512 : 1024; }

struct NormGateArgs {
    const void *u, *r, *gate;
    const void *wa, *ba, *wb, *bb;
    void *y, *n;
    float4* stats;                    // [rows] {mean_a, rstd_a, mean_b, rstd_b}
    const void *dy, *dn;
    void *du, *dr, *dg;
    float *part_w, *part_g;           // [blocks][4][d], [gate rows][chunks][d]
    int rows, d, gate_rows;           // gate_rows: rows that share a row of the gate (1: elementwise)
    int gate_kind, after, before, param_f32;
    float scale, eps;
    // division of the rows: a workgroup takes `groups_per_block` whole groups of `group_rows` rows, or (chunks > 1) a
    // chunk of `chunk_rows` rows of one group
    int groups, group_rows, groups_per_block, chunks, chunk_rows;
    int sum_gate;                     // the gate's gradient is a sum over the rows of a group
    int wanted;                       // which affine gradients: bit 0 dwa, 1 dba, 2 dwb, 3 dbb
};

__host__ __device__ __forceinline__ int padded(int d) { return (d + 3) & ~3; }

// every lane's value plus those of the three lanes at its place in the other rows of 16, by exchanging rows between two
// registers: no trip through LDS, which costs 2 to 4 % of the wide rows' backward
__device__ __forceinline__ float add_rows_of_16(float v) {
#ifdef __HIP_DEVICE_COMPILE__
    const auto p = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(p[0]) + __uint_as_float(p[1]);
    const auto q = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(q[0]) + __uint_as_float(q[1]);
#endif
    return v;
}

// sums of two values over the G lanes that hold a row (16, 64, or the whole workgroup), in every lane
template <int G>
__device__ __forceinline__ void row_sum2(float& a, float& b, float (*lds)[2]) {
#define PCLIP_DPP_ADD2(ctrl)                                                                     \
    a += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(a), ctrl, 0xF, 0xF, true)); \
    b += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(b), ctrl, 0xF, 0xF, true))
    PCLIP_DPP_ADD2(0xB1);
    PCLIP_DPP_ADD2(0x4E);
    PCLIP_DPP_ADD2(0x141);
    PCLIP_DPP_ADD2(0x140);
#undef PCLIP_DPP_ADD2
    if constexpr (G >= 64) {
        a = add_rows_of_16(a);
        b = add_rows_of_16(b);
    }
    if constexpr (G == 256) {
        __syncthreads();   // the previous sum's readers are done
        if ((threadIdx.x & 63) == 0) {
            lds[threadIdx.x >> 6][0] = a;
            lds[threadIdx.x >> 6][1] = b;
        }
        __syncthreads();
        a = (lds[0][0] + lds[1][0]) + (lds[2][0] + lds[3][0]);
        b = (lds[0][1] + lds[1][1]) + (lds[2][1] + lds[3][1]);
    }
}

// A row of a wave's operands as the buffer instructions see it: the first byte of the wave's first row, and how far it reaches.
// An operand that is absent reaches nowhere: its loads give zeros and its stores vanish, as they do for lanes whose offset
// lies outside, so neither needs a branch.
constexpr unsigned REACH = 1u << 28, OUTSIDE = 1u << 31;   // an offset of OUTSIDE stays outside when it is divided by an element's size
struct Span { const void* base; unsigned reach; };
__device__ __forceinline__ Span span_of(const void* p, size_t byte) { return {p ? (const char*)p + byte : nullptr, p ? REACH : 0u}; }

// BYTES (1 to 16) of a lane as whole registers
constexpr int words(int bytes) { return bytes > 4 ? bytes / 4 : 1; }
template <int BYTES>
__device__ __forceinline__ void buffer_load(Span s, unsigned off, unsigned* r) {
#ifdef __HIP_DEVICE_COMPILE__   // the host pass has no descriptors
    const auto rsrc = __builtin_amdgcn_make_buffer_rsrc((void*)s.base, 0, s.reach, 0x00020000);
    if constexpr (BYTES == 16) {
        const auto v = __builtin_amdgcn_raw_buffer_load_b128(rsrc, off, 0, 0);
        r[0] = v[0], r[1] = v[1], r[2] = v[2], r[3] = v[3];
    } else if constexpr (BYTES == 8) {
        const auto v = __builtin_amdgcn_raw_buffer_load_b64(rsrc, off, 0, 0);
        r[0] = v[0], r[1] = v[1];
    } else if constexpr (BYTES == 4) {
        r[0] = __builtin_amdgcn_raw_buffer_load_b32(rsrc, off, 0, 0);
    } else if constexpr (BYTES == 2) {
        r[0] = (unsigned short)__builtin_amdgcn_raw_buffer_load_b16(rsrc, off, 0, 0);
    } else {
        r[0] = (unsigned char)__builtin_amdgcn_raw_buffer_load_b8(rsrc, off, 0, 0);
    }
#endif
}
constexpr int PAST_L2 = 2;   // the nt bit: results that nobody reads back soon
template <int BYTES>
__device__ __forceinline__ void buffer_store(Span s, unsigned off, const unsigned* v) {
#ifdef __HIP_DEVICE_COMPILE__
    typedef unsigned __attribute__((ext_vector_type(4))) u4;
    typedef unsigned __attribute__((ext_vector_type(2))) u2;
    const auto rsrc = __builtin_amdgcn_make_buffer_rsrc((void*)s.base, 0, s.reach, 0x00020000);
    if constexpr (BYTES == 16) __builtin_amdgcn_raw_buffer_store_b128(u4{v[0], v[1], v[2], v[3]}, rsrc, off, 0, PAST_L2);
    else if constexpr (BYTES == 8) __builtin_amdgcn_raw_buffer_store_b64(u2{v[0], v[1]}, rsrc, off, 0, PAST_L2);
    else if constexpr (BYTES == 4) __builtin_amdgcn_raw_buffer_store_b32(v[0], rsrc, off, 0, PAST_L2);
    else __builtin_amdgcn_raw_buffer_store_b16((unsigned short)v[0], rsrc, off, 0, PAST_L2);
#endif
}
// element i of a lane's words, and the words of a lane's elements
template <typename T, int V>
__device__ __forceinline__ float element(const unsigned* w, int i) {
    if constexpr (sizeof(T) == 4) return __builtin_bit_cast(float, w[i]);
    else return (float)__builtin_bit_cast(T, (unsigned short)(V == 1 ? w[i] : w[i / 2] >> (i % 2 * 16)));
}
template <typename T>
__device__ __forceinline__ unsigned bits(float x) {
    if constexpr (sizeof(T) == 4) return __builtin_bit_cast(unsigned, x);
    else return __builtin_bit_cast(unsigned short, (T)x);
}

// The elements of one lane: NV vectors of V, vector k at column (k * G + lane) * V.  V is one where rows do not divide into vectors
// or an operand is not aligned to one.
template <typename T, int G, int NV, int V>
struct Row {
    static constexpr int E = NV * V, NG = THREADS / G, ROWS = G < 64 ? 64 / G : 1, BYTES = V * (int)sizeof(T);   // ROWS: of a wave
    static constexpr int W = words(BYTES), WB = words(V);   // registers of a vector, and of a byte mask's
    // whether a row is loaded while the one before it is worked on: two waves a SIMD do not cover the memory's latency by
    // themselves; rows of many registers would not fit twice
    static constexpr bool AHEAD = NV * W <= 8;
    static __device__ __forceinline__ int col(int k) { return (k * G + (int)(threadIdx.x % G)) * V; }
    static __device__ __forceinline__ int in_wave() { return G < 64 ? (int)(threadIdx.x & 63) / G : 0; }
    // byte offsets of the lane's vectors from the wave's first row
    static __device__ __forceinline__ void offsets(int d, unsigned (&off)[NV]) {
#pragma unroll
        for (int k = 0; k < NV; k++) off[k] = col(k) < d ? (unsigned)(in_wave() * d + col(k)) * (unsigned)sizeof(T) : OUTSIDE;
    }
    static __device__ __forceinline__ void load(Span s, const unsigned (&off)[NV], unsigned skip, unsigned (&r)[NV * W]) {
#pragma unroll
        for (int k = 0; k < NV; k++) buffer_load<BYTES>(s, off[k] | skip, r + k * W);
    }
    static __device__ __forceinline__ void store(Span s, const unsigned (&off)[NV], unsigned skip, const float (&x)[E]) {
#pragma unroll
        for (int k = 0; k < NV; k++) {
            unsigned v[W];
#pragma unroll
            for (int i = 0; i < W; i++) v[i] = BYTES / W == 4 && sizeof(T) == 2 ? bits<T>(x[k * V + 2 * i]) | bits<T>(x[k * V + 2 * i + 1]) << 16 : bits<T>(x[k * V + i]);
            buffer_store<BYTES>(s, off[k] | skip, v);
        }
    }
    static __device__ __forceinline__ void widen(const unsigned (&r)[NV * W], float (&x)[E]) {
#pragma unroll
        for (int i = 0; i < E; i++) x[i] = element<T, V>(r + i / V * W, i % V);
    }
    static __device__ __forceinline__ void fill(float (&x)[E], float v) {
#pragma unroll
        for (int i = 0; i < E; i++) x[i] = v;
    }
    // a row of the gate: values of T, or bytes (nonzero = 1)
    struct Gate { unsigned t[NV * W], b[NV * WB]; };
    static __device__ __forceinline__ void load_gate(const NormGateArgs& A, int row0, const unsigned (&off)[NV], unsigned skip, Gate& r) {
        if (A.gate_kind == PCLIP_GATE_BYTES) {
            const Span s = span_of(A.gate, (size_t)row0 * A.d);
#pragma unroll
            for (int k = 0; k < NV; k++) buffer_load<V>(s, (off[k] | skip) / (unsigned)sizeof(T), r.b + k * WB);
        } else if (A.gate_kind == PCLIP_GATE_ROWS) {
            const unsigned first = A.gate_rows == 1 ? (unsigned)row0 : (unsigned)row0 / (unsigned)A.gate_rows;
            const Span s = span_of(A.gate, (size_t)first * A.d * sizeof(T));
            unsigned back = 0;   // the lane's gate row may be an earlier one than its own row's place from the wave's first
            if (ROWS > 1 && A.gate_rows > 1)
                back = (unsigned)(in_wave() - (int)((unsigned)(row0 + in_wave()) / (unsigned)A.gate_rows - first)) * (unsigned)A.d * (unsigned)sizeof(T);
#pragma unroll
            for (int k = 0; k < NV; k++) buffer_load<BYTES>(s, (off[k] | skip) >= OUTSIDE ? OUTSIDE : off[k] - back, r.t + k * W);
        }
    }
    static __device__ __forceinline__ void widen_gate(const NormGateArgs& A, const Gate& r, float (&g)[E]) {
        if (A.gate_kind == PCLIP_GATE_BYTES) {
#pragma unroll
            for (int i = 0; i < E; i++) g[i] = r.b[i / V * WB + i % V / 4] >> (i % V % 4 * 8) & 255u ? 1.f : 0.f;
        } else if (A.gate_kind == PCLIP_GATE_ROWS) {
            widen(r.t, g);
        } else {
            fill(g, 1.f);
        }
    }
    // Affine parameters.  Lanes that take row after row of one place keep theirs in registers when each has a place of its own
    // (G = 256); waves that share the places read them from LDS, as f32 padded to whole vectors, again for each row: in
    // registers they would take a quarter of a lane's, which the column sums need.
    struct Param {
        static constexpr bool OWN = G == 256;
        float own[OWN ? E : 1];
        const float* lds;
        __device__ __forceinline__ void stage(const void* p, bool f32, int d, float other, float* to) {
            if constexpr (OWN) {
#pragma unroll
                for (int k = 0; k < NV; k++)
#pragma unroll
                    for (int i = 0; i < V; i++) own[k * V + i] = at(p, f32, d, other, col(k) + i);
            } else {
                for (int c = threadIdx.x; c < padded(d); c += THREADS) to[c] = at(p, f32, d, other, c);
                lds = to;
            }
        }
        static __device__ __forceinline__ float at(const void* p, bool f32, int d, float other, int c) {
            return !p || c >= d ? other : f32 ? ((const float*)p)[c] : (float)((const T*)p)[c];
        }
        __device__ __forceinline__ void get(int k, int d, float (&x)[V]) const {
            if constexpr (OWN) {
#pragma unroll
                for (int i = 0; i < V; i++) x[i] = own[k * V + i];
            } else if constexpr (V == 1) {
                x[0] = lds[col(k) < d ? col(k) : 0];   // lanes behind the row use any
            } else {
#pragma unroll
                for (int i = 0; i < V; i += 4) {
                    const int c = col(k) + i;
                    const f32x4 v = *(const f32x4*)(lds + (c < d ? c : 0));
#pragma unroll
                    for (int j = 0; j < 4; j++) x[i + j] = v[j];
                }
            }
        }
    };
    static __device__ __forceinline__ void affine(float (&x)[E], float mean, float rstd, const Param& w, const Param& b, int d) {
#pragma unroll
        for (int k = 0; k < NV; k++) {
            float wk[V], bk[V];
            w.get(k, d, wk);
            b.get(k, d, bk);
#pragma unroll
            for (int i = 0; i < V; i++) x[k * V + i] = fmaf((x[k * V + i] - mean) * rstd, wk[i], bk[i]);
        }
    }
    // mean (zero for rms) and 1 / sqrt(mean square of the centred values + eps)
    static __device__ __forceinline__ void stats(const float (&x)[E], int kind, int d, float eps, float& mean, float& rstd, float (*lds)[2]) {
        const float inv = 1.f / (float)d;
        mean = 0.f;
        float s = 0.f, q = 0.f;
        if (kind == PCLIP_NORM_LAYER) {
#pragma unroll
            for (int i = 0; i < E; i++) s += x[i];   // the places behind the row are zero
            row_sum2<G>(s, q, lds);
            mean = s * inv;
        }
        q = 0.f;
        s = 0.f;
#pragma unroll
        for (int k = 0; k < NV; k++) {
            const float m = col(k) < d ? mean : 0.f;   // nothing behind the row is off its mean
#pragma unroll
            for (int i = 0; i < V; i++) {
                const float c = x[k * V + i] - m;
                q = fmaf(c, c, q);
            }
        }
        row_sum2<G>(q, s, lds);
        rstd = 1.f / sqrtf(q * inv + eps);
    }
};

template <typename T, int G, int NV, int V>
__global__ __launch_bounds__(THREADS) void norm_gate_fwd_kernel(const NormGateArgs A) {
    using R = Row<T, G, NV, V>;
    constexpr int E = R::E;
    __shared__ float lds[4][2];
    const int d = A.d, rows = A.rows;
    extern __shared__ __attribute__((aligned(16))) float params[];
    typename R::Param wa, ba, wb, bb;
    wa.stage(A.wa, A.param_f32, d, 1.f, params);
    ba.stage(A.ba, A.param_f32, d, 0.f, params + padded(d));
    wb.stage(A.wb, A.param_f32, d, 1.f, params + 2 * padded(d));
    bb.stage(A.bb, A.param_f32, d, 0.f, params + 3 * padded(d));
    __syncthreads();
    unsigned off[NV];
    R::offsets(d, off);
    unsigned in_u[NV * R::W], in_r[NV * R::W];   // a row as it was read
    typename R::Gate in_g;
    auto skip = [&](int row0) { return R::ROWS > 1 && rows - row0 <= R::in_wave() ? OUTSIDE : 0u; };
    auto load = [&](int row0) {
        const size_t at = (size_t)row0 * d * sizeof(T);
        R::load(span_of(A.u, at), off, skip(row0), in_u);
        R::load(span_of(A.r, at), off, skip(row0), in_r);
        R::load_gate(A, row0, off, skip(row0), in_g);
    };
    const int stride = gridDim.x * R::NG;
    int row0 = blockIdx.x * R::NG + (G == 256 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) * R::ROWS);
    if (R::AHEAD && row0 < rows) load(row0);
    for (; row0 < rows; row0 += stride) {
        asm volatile("" ::: "memory");   // parameters in LDS are read again for each row
        float u[E], y[E], g[E];
        if (!R::AHEAD) load(row0);
        R::widen(in_u, u);
        R::widen(in_r, y);
        R::widen_gate(A, in_g, g);
        if (R::AHEAD && rows - row0 > stride) load(row0 + stride);
        float4 st = make_float4(0.f, 1.f, 0.f, 1.f);
        if (A.after) {
            R::stats(u, A.after, d, A.eps, st.x, st.y, lds);
            R::affine(u, st.x, st.y, wa, ba, d);
        }
#pragma unroll
        for (int k = 0; k < NV; k++) {
            const float scale = R::col(k) < d ? A.scale : 0.f;
#pragma unroll
            for (int i = 0; i < V; i++) y[k * V + i] = fmaf(scale, u[k * V + i] * g[k * V + i], y[k * V + i]);
        }
        const size_t at = (size_t)row0 * d * sizeof(T);
        R::store(span_of(A.y, at), off, skip(row0), y);
        if (A.before) {
            R::stats(y, A.before, d, A.eps, st.z, st.w, lds);
            R::affine(y, st.z, st.w, wb, bb, d);
            R::store(span_of(A.n, at), off, skip(row0), y);
        }
        if (A.stats && threadIdx.x % G == 0 && !skip(row0)) A.stats[row0 + R::in_wave()] = st;
    }
}

// Adds the accumulators of a workgroup's row slots (`buf`: one row of E * G floats a wave) and hands each column's sum
// to `put(column, value)`.  Every thread of the workgroup calls it.
template <typename T, int G, int NV, int V, int E, typename Put>
__device__ __forceinline__ void flush_columns(float (&acc)[E], float* buf, int d, Put put) {
    using R = Row<T, G, NV, V>;
    if constexpr (G == 256) {   // one row at a time: every column has one owner
#pragma unroll
        for (int k = 0; k < NV; k++)
#pragma unroll
            for (int i = 0; i < V; i++)
                if (R::col(k) + i < d) put(R::col(k) + i, acc[k * V + i]);
    } else {
        constexpr int W = G * E;   // columns of a wave's row of buf
        if constexpr (G == 16) {
#pragma unroll
            for (int i = 0; i < R::E; i++) {
                acc[i] += __shfl_xor(acc[i], 16);
                acc[i] += __shfl_xor(acc[i], 32);
            }
        }
        __syncthreads();   // the previous call's readers are done
        if ((threadIdx.x & 63) < G)
#pragma unroll
            for (int k = 0; k < NV; k++)
#pragma unroll
                for (int i = 0; i < V; i++) buf[(threadIdx.x >> 6) * W + R::col(k) + i] = acc[k * V + i];
        __syncthreads();
        for (int c = threadIdx.x; c < d; c += THREADS) put(c, (buf[c] + buf[W + c]) + (buf[2 * W + c] + buf[3 * W + c]));
    }
#pragma unroll
    for (int i = 0; i < R::E; i++) acc[i] = 0.f;
}

template <typename T, int G, int NV, int V>
__global__ __launch_bounds__(THREADS, NV * V > 12 ? 1 : 2) void norm_gate_bwd_kernel(const NormGateArgs A) {
    using R = Row<T, G, NV, V>;
    constexpr int E = R::E;
    __shared__ float lds[4][2];
    __shared__ float buf[G == 256 ? 1 : 4 * G * E];
    const int d = A.d;
    const float inv = 1.f / (float)d;
    float swa[E], sba[E], swb[E], sbb[E], sg[E];
#pragma unroll
    for (int i = 0; i < E; i++) swa[i] = sba[i] = swb[i] = sbb[i] = sg[i] = 0.f;
    extern __shared__ __attribute__((aligned(16))) float params[];
    typename R::Param wa, ba, wb;
    wa.stage(A.wa, A.param_f32, d, 1.f, params);
    ba.stage(A.ba, A.param_f32, d, 0.f, params + padded(d));
    wb.stage(A.wb, A.param_f32, d, 1.f, params + 2 * padded(d));
    __syncthreads();
    const bool before = A.before && A.dn;
    unsigned off[NV];
    R::offsets(d, off);
    unsigned in_u[NV * R::W], in_r[NV * R::W], in_dy[NV * R::W], in_dn[NV * R::W];   // a row as it was read
    typename R::Gate in_g;
    float4 in_st;
    int first = 0, last = 0;
    auto skip = [&](int row0) { return R::ROWS > 1 && last - row0 <= R::in_wave() ? OUTSIDE : 0u; };
    auto load = [&](int row0) {
        const size_t at = (size_t)row0 * d * sizeof(T);
        const unsigned s = skip(row0);
        in_st = make_float4(0.f, 1.f, 0.f, 1.f);
        if (A.stats && !s) in_st = A.stats[row0 + R::in_wave()];
        R::load(span_of(A.u, at), off, s, in_u);
        R::load(span_of(A.dy, at), off, s, in_dy);
        if (before) {
            R::load(span_of(A.dn, at), off, s, in_dn);
            R::load(span_of(A.r, at), off, s, in_r);
        }
        R::load_gate(A, row0, off, s, in_g);
    };
    const int g0 = A.chunks > 1 ? (int)blockIdx.x / A.chunks : (int)blockIdx.x * A.groups_per_block;
    const int g1 = A.chunks > 1 ? g0 + 1 : min(g0 + A.groups_per_block, A.groups);
    for (int grp = g0; grp < g1; grp++) {
        // (group + 1) * group_rows <= rows: no overflow
        first = grp * A.group_rows, last = first + A.group_rows;
        if (A.chunks > 1) {
            const long long from = first + (long long)((int)blockIdx.x % A.chunks) * A.chunk_rows;
            first = (int)min(from, (long long)last);
            last = (int)min(from + A.chunk_rows, (long long)last);
        }
        int row0 = first + (G == 256 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) * R::ROWS);
        if (R::AHEAD && row0 < last) load(row0);
        for (; row0 < last; row0 += R::NG) {
            asm volatile("" ::: "memory");   // parameters in LDS are read again for each row
            float u[E], t[E], g[E], h[E], q[E];
            if (!R::AHEAD) load(row0);
            const float4 st = in_st;
            R::widen(in_u, u);
            R::widen(in_dy, t);
            if (before) {
                R::widen(in_dn, q);
                R::widen(in_r, h);
            }
            R::widen_gate(A, in_g, g);
            if (R::AHEAD && last - row0 > R::NG) load(row0 + R::NG);
            const size_t at = (size_t)row0 * d * sizeof(T);
            const unsigned s = skip(row0);
            float v[E];   // the value that the gate multiplies
            if (A.after) {
#pragma unroll
                for (int k = 0; k < NV; k++) {
                    float wk[V], bk[V];
                    wa.get(k, d, wk);
                    ba.get(k, d, bk);
#pragma unroll
                    for (int j = 0; j < V; j++) {
                        const int i = k * V + j;
                        u[i] = (u[i] - st.x) * st.y;   // from here on the normalised value
                        v[i] = fmaf(u[i], wk[j], bk[j]);
                    }
                }
            } else {
#pragma unroll
                for (int i = 0; i < E; i++) v[i] = u[i];
            }
            if (before) {
                float m1 = 0.f, m2 = 0.f;
#pragma unroll
                for (int k = 0; k < NV; k++) {
                    float wk[V];
                    wb.get(k, d, wk);
#pragma unroll
                    for (int j = 0; j < V; j++) {
                        const int i = k * V + j;
                        h[i] = (fmaf(A.scale, g[i] * v[i], h[i]) - st.z) * st.w;
                        swb[i] = fmaf(q[i], h[i], swb[i]);   // q is zero behind the row
                        sbb[i] += q[i];
                        q[i] *= wk[j];
                        m1 += q[i];
                        m2 = fmaf(q[i], h[i], m2);
                    }
                }
                row_sum2<G>(m1, m2, lds);
                m1 = A.before == PCLIP_NORM_LAYER ? m1 * inv : 0.f;
                m2 *= inv;
#pragma unroll
                for (int i = 0; i < E; i++) t[i] = fmaf(st.w, q[i] - m1 - h[i] * m2, t[i]);
            }
            R::store(span_of(A.dr, at), off, s, t);
            if (A.dg && !A.sum_gate) {
                float e[E];
#pragma unroll
                for (int i = 0; i < E; i++) e[i] = A.scale * v[i] * t[i];
                R::store(span_of(A.dg, at), off, s, e);
            }
            float m1 = 0.f, m2 = 0.f;
#pragma unroll
            for (int k = 0; k < NV; k++) {
                float wk[V];
                wa.get(k, d, wk);
                const float scale = R::col(k) < d ? A.scale : 0.f;   // nothing behind the row enters the sums
#pragma unroll
                for (int j = 0; j < V; j++) {
                    const int i = k * V + j;
                    const float in = scale * t[i];
                    sg[i] = fmaf(v[i], in, sg[i]);
                    t[i] = g[i] * in;                                            // dv
                    swa[i] = fmaf(t[i], u[i], swa[i]);
                    sba[i] += t[i];
                    t[i] *= wk[j];
                    m1 += t[i];
                    m2 = fmaf(t[i], u[i], m2);
                }
            }
            if (A.after) {
                row_sum2<G>(m1, m2, lds);
                m1 = A.after == PCLIP_NORM_LAYER ? m1 * inv : 0.f;
                m2 *= inv;
#pragma unroll
                for (int i = 0; i < E; i++) t[i] = st.y * (t[i] - m1 - u[i] * m2);
            }
            R::store(span_of(A.du, at), off, s, t);
        }
        if (A.sum_gate) {
            float* to = A.part_g + ((size_t)grp * A.chunks + (A.chunks > 1 ? (int)blockIdx.x % A.chunks : 0)) * d;
            T* out = (T*)A.dg + (size_t)grp * d;
            flush_columns<T, G, NV, V>(sg, buf, d, [&](int c, float s) {
                if (A.chunks > 1) to[c] = s;
                else out[c] = (T)s;
            });
        }
    }
    if (A.part_w) {
        float* to = A.part_w + (size_t)blockIdx.x * 4 * d;
        if (A.wanted & 1) flush_columns<T, G, NV, V>(swa, buf, d, [&](int c, float s) { to[c] = s; });
        if (A.wanted & 2) flush_columns<T, G, NV, V>(sba, buf, d, [&](int c, float s) { to[d + c] = s; });
        if (A.wanted & 4) flush_columns<T, G, NV, V>(swb, buf, d, [&](int c, float s) { to[2 * d + c] = s; });
        if (A.wanted & 8) flush_columns<T, G, NV, V>(sbb, buf, d, [&](int c, float s) { to[3 * d + c] = s; });
    }
}

// Column sums of the workspace: blockIdx.y < 4 an affine gradient over the `blocks` workgroups, behind that a gate row
// over its chunks.  64 columns x 16 rows of threads, the 16 added through LDS.
struct ColumnSumArgs {
    const float *part_w, *part_g;
    void* out[4];
    void* dg;
    int blocks, chunks, d, first_y, param_type, type;
};
__device__ __forceinline__ void store_as(void* p, int type, size_t i, float v) {
    if (type == PCLIP_DT_F32) ((float*)p)[i] = v;
    else if (type == PCLIP_DT_BF16) ((__bf16*)p)[i] = (__bf16)v;
    else ((_Float16*)p)[i] = (_Float16)v;
}
__global__ __launch_bounds__(1024) void column_sum_kernel(const ColumnSumArgs A) {
    __shared__ float lds[16][65];
    const int lane = threadIdx.x & 63, part = threadIdx.x >> 6, c = blockIdx.x * 64 + lane, k = blockIdx.y + A.first_y, d = A.d;
    const bool gate = k >= 4;
    if (!gate && !A.out[k]) return;
    const float* p = gate ? A.part_g + (size_t)(k - 4) * A.chunks * d : A.part_w + (size_t)k * d;
    const size_t stride = gate ? (size_t)d : (size_t)4 * d;
    const int count = gate ? A.chunks : A.blocks;
    float s = 0.f;
    if (c < d) {
        float more[8] = {};
        int i = part;
        for (; i + 7 * 16 < count; i += 8 * 16)   // eight loads under way
#pragma unroll
            for (int q = 0; q < 8; q++) more[q] += p[(i + q * 16) * stride + c];
        for (; i < count; i += 16) s += p[i * stride + c];
#pragma unroll
        for (int q = 0; q < 8; q++) s += more[q];
    }
    lds[part][lane] = s;
    __syncthreads();
    if (part == 0 && c < d) {
        s = 0.f;
#pragma unroll
        for (int i = 0; i < 16; i++) s += lds[i][lane];
        if (gate) store_as(A.dg, A.type, (size_t)(k - 4) * d + c, s);
        else store_as(A.out[k], A.param_type, c, s);
    }
}

// Lanes, vectors and their width for a row: the fewest lanes that hold it with at most 12 elements each (the backward keeps five
// column sums of that many registers; 16 only beyond 2048, where nothing smaller holds a row), in 16-byte accesses where that
// wastes less than half of them.
struct Shape { int lanes, vectors, width; };
Shape shape_of(int d, int dtype) {
    const bool wide = dtype != PCLIP_DT_F32;   // 16 bytes are eight elements
    if (d <= 64) return {16, 1, 4};
    if (d <= 128) return wide ? Shape{16, 1, 8} : Shape{16, 2, 4};
    if (d <= 256) return {64, 1, 4};
    if (d <= 512) return wide ? Shape{64, 1, 8} : Shape{64, 2, 4};
    if (d <= 768) return {64, 3, 4};
    if (d <= 1024) return {256, 1, 4};
    if (d <= 2048) return wide ? Shape{256, 1, 8} : Shape{256, 2, 4};
    return wide ? Shape{256, 2, 8} : Shape{256, 4, 4};
}

// How the backward divides the rows over workgroups (see NormGateArgs).  With column sums 512 workgroups, two a compute unit,
// are aimed at: more write more partial sums (1024: 60 us instead of 54 for 32,768 x 640, 39 instead of 30 for 3003 x 1283).
void plan(NormGateArgs& A, int dtype, bool sums, int& blocks) {
    const int slots = THREADS / shape_of(A.d, dtype).lanes;
    const int target = sums ? 512 : 2048;
    A.group_rows = A.sum_gate ? A.gate_rows : A.rows;
    A.groups = A.rows / A.group_rows;
    A.groups_per_block = 1;
    A.chunks = 1;
    A.chunk_rows = A.group_rows;
    if (A.groups >= target) {
        A.groups_per_block = (A.groups + target - 1) / target;
    } else {
        const int want = target / A.groups, most = (A.group_rows + slots - 1) / slots;   // a chunk has a row for every slot at least
        A.chunks = want < most ? want : most;
        A.chunk_rows = (A.group_rows + A.chunks - 1) / A.chunks;
        A.chunks = (A.group_rows + A.chunk_rows - 1) / A.chunk_rows;
    }
    blocks = A.chunks > 1 ? A.groups * A.chunks : (A.groups + A.groups_per_block - 1) / A.groups_per_block;
}

template <typename T, int G, int NV, int V>
int launch(const NormGateArgs& A, bool fwd, int blocks, hipStream_t st) {
    // the affine parameters, where waves share them (see Param): at most 768 of each, below the limit that every kernel has
    const size_t bytes = Row<T, G, NV, V>::Param::OWN ? 0 : (size_t)(fwd ? 4 : 3) * padded(A.d) * sizeof(float);
    if (fwd) norm_gate_fwd_kernel<T, G, NV, V><<<blocks, THREADS, bytes, st>>>(A);
    else norm_gate_bwd_kernel<T, G, NV, V><<<blocks, THREADS, bytes, st>>>(A);
    return PCLIP_OK;
}
template <typename T, int V8>
int launch_width(const NormGateArgs& A, const Shape& s, bool fwd, int blocks, hipStream_t st) {
    // V8: elements of an access of eight; four go in one access, or one by one
    constexpr int V4 = V8 == 1 ? 1 : 4;
    const int each = s.vectors * s.width;
    if (s.lanes == 16) return each == 4 ? launch<T, 16, 4 / V4, V4>(A, fwd, blocks, st) : launch<T, 16, 8 / V8, V8>(A, fwd, blocks, st);
    if (s.lanes == 64)
        return each == 4 ? launch<T, 64, 4 / V4, V4>(A, fwd, blocks, st)
                         : each == 8 ? launch<T, 64, 8 / V8, V8>(A, fwd, blocks, st) : launch<T, 64, 12 / V4, V4>(A, fwd, blocks, st);
    return each == 4 ? launch<T, 256, 4 / V4, V4>(A, fwd, blocks, st)
                     : each == 8 ? launch<T, 256, 8 / V8, V8>(A, fwd, blocks, st) : launch<T, 256, 16 / V8, V8>(A, fwd, blocks, st);
}
// whether every row of every operand begins at a multiple of its vectors' width
template <typename T>
bool in_vectors(const NormGateArgs& A, const Shape& s) {
    const bool bytes = A.gate_kind == PCLIP_GATE_BYTES;
    uintptr_t bits = (uintptr_t)A.u | (uintptr_t)A.r | (uintptr_t)A.y | (uintptr_t)A.n | (uintptr_t)A.dy | (uintptr_t)A.dn | (uintptr_t)A.du | (uintptr_t)A.dr |
                     (uintptr_t)A.dg | (bytes ? (uintptr_t)A.gate * sizeof(T) : (uintptr_t)A.gate);
    return bits % (s.width * sizeof(T)) == 0 && A.d % s.width == 0;
}
template <typename T>
int launch_type(const NormGateArgs& A, int dtype, bool fwd, int blocks, hipStream_t st) {
    const Shape s = shape_of(A.d, dtype);
    return in_vectors<T>(A, s) ? launch_width<T, PclipVec<T>::N>(A, s, fwd, blocks, st) : launch_width<T, 1>(A, s, fwd, blocks, st);
}
int launch_kernel(const NormGateArgs& A, int dtype, bool fwd, int blocks, hipStream_t st) {
    if (dtype == PCLIP_DT_F32) return launch_type<float>(A, dtype, fwd, blocks, st);
    if (dtype == PCLIP_DT_BF16) return launch_type<__bf16>(A, dtype, fwd, blocks, st);
    return launch_type<_Float16>(A, dtype, fwd, blocks, st);
}

int check_common(const char* who, int rows, int d, int dtype, int param_type, const void* gate, int gate_kind, int gate_rows, int after, int before,
                 float eps) {
    PCLIP_REQUIRE(pclip_dtype_ok(dtype), "%s: unknown type %d", who, dtype);
    PCLIP_REQUIRE(param_type == PCLIP_DT_F32 || param_type == dtype, "%s: affine parameters are f32 or of the rows' type", who);
    PCLIP_REQUIRE(rows >= 1 && rows <= 0x7fff0000 && d >= 1 && d <= MAX_D, "%s: rows=%d d=%d (1 <= rows <= 2147418112, 1 <= d <= %d)", who, rows, d, MAX_D);
    PCLIP_REQUIRE(after >= PCLIP_NORM_NONE && after <= PCLIP_NORM_RMS && before >= PCLIP_NORM_NONE && before <= PCLIP_NORM_RMS, "%s: unknown norm", who);
    PCLIP_REQUIRE(gate_kind >= PCLIP_GATE_NONE && gate_kind <= PCLIP_GATE_BYTES && (gate_kind == PCLIP_GATE_NONE || gate), "%s: gate kind and pointer", who);
    PCLIP_REQUIRE(gate_kind != PCLIP_GATE_ROWS || (gate_rows >= 1 && rows % gate_rows == 0), "%s: gate_rows=%d does not divide rows=%d", who, gate_rows, rows);
    PCLIP_REQUIRE(eps >= 0.f, "%s: eps must be zero or more", who);
    return PCLIP_OK;
}

}  // namespace

extern "C" int pclip_norm_gate_fwd(const void* u, const void* r, const void* gate, int gate_kind, int gate_rows, float scale, int after, const void* wa,
                                   const void* ba, int before, const void* wb, const void* bb, int param_type, float eps, int rows, int d, int dtype,
                                   void* y, void* n, float* stats, void* stream) {
    int rc = check_common("norm_gate_fwd", rows, d, dtype, param_type, gate, gate_kind, gate_rows, after, before, eps);
    if (rc) return rc;
    PCLIP_REQUIRE(u && y && (before == PCLIP_NORM_NONE || n), "norm_gate_fwd: null pointer");
    PCLIP_REQUIRE(((uintptr_t)stats & 15) == 0, "norm_gate_fwd: stats must be 16-byte aligned");
    NormGateArgs A = {};
    A.u = u, A.r = r, A.gate = gate, A.wa = wa, A.ba = ba, A.wb = wb, A.bb = bb, A.y = y, A.n = n, A.stats = (float4*)stats;
    A.rows = rows, A.d = d, A.gate_rows = gate_kind == PCLIP_GATE_ROWS ? gate_rows : 1, A.gate_kind = gate_kind, A.after = after, A.before = before;
    A.param_f32 = param_type == PCLIP_DT_F32, A.scale = scale, A.eps = eps;
    const int slots = THREADS / shape_of(d, dtype).lanes;
    const long long want = ((long long)rows + slots - 1) / slots;
    rc = launch_kernel(A, dtype, true, want < fwd_blocks(d) ? (int)want : fwd_blocks(d), (hipStream_t)stream);
    return rc ? rc : pclip_check_launch("norm_gate_fwd");
}

extern "C" int pclip_norm_gate_row(int d, int dtype, int* lanes, int* vectors, int* width) {
    PCLIP_REQUIRE(d >= 1 && d <= MAX_D && pclip_dtype_ok(dtype) && lanes && vectors && width, "norm_gate_row: d=%d or the type, or a null pointer", d);
    const Shape s = shape_of(d, dtype);
    *lanes = s.lanes, *vectors = s.vectors, *width = d % s.width == 0 ? s.width : 1;
    if (*width != s.width) *vectors *= s.width;
    return PCLIP_OK;
}

extern "C" size_t pclip_norm_gate_bwd_workspace_bytes(int rows, int d, int dtype, int gate_rows) {
    if (rows < 1 || rows > 0x7fff0000 || d < 1 || d > MAX_D || !pclip_dtype_ok(dtype) || gate_rows < 0 || (gate_rows && rows % gate_rows)) return 0;
    NormGateArgs A = {};
    A.rows = rows, A.d = d, A.gate_rows = gate_rows ? gate_rows : 1, A.sum_gate = gate_rows > 1;
    int blocks = 0;
    plan(A, dtype, true, blocks);
    return ((size_t)blocks * 4 + (A.chunks > 1 && A.sum_gate ? (size_t)A.groups * A.chunks : 0)) * d * sizeof(float);
}

extern "C" int pclip_norm_gate_bwd(const void* u, const void* r, const void* gate, int gate_kind, int gate_rows, float scale, int after, const void* wa,
                                   const void* ba, int before, const void* wb, const void* bb, int param_type, float eps, int rows, int d, int dtype,
                                   const float* stats, const void* dy, const void* dn, void* du, void* dr, void* dgate, void* dwa, void* dba, void* dwb,
                                   void* dbb, void* ws, size_t ws_bytes, void* stream) {
    int rc = check_common("norm_gate_bwd", rows, d, dtype, param_type, gate, gate_kind, gate_rows, after, before, eps);
    if (rc) return rc;
    PCLIP_REQUIRE(u && (dy || dn), "norm_gate_bwd: null pointer");
    PCLIP_REQUIRE((after == PCLIP_NORM_NONE && before == PCLIP_NORM_NONE) || stats, "norm_gate_bwd: the forward's statistics are needed");
    PCLIP_REQUIRE(((uintptr_t)stats & 15) == 0, "norm_gate_bwd: stats must be 16-byte aligned");
    PCLIP_REQUIRE(!dgate || gate_kind == PCLIP_GATE_ROWS, "norm_gate_bwd: a byte mask has no gradient");
    PCLIP_REQUIRE((!dwa || after) && (!dba || after) && (!dwb || before) && (!dbb || before), "norm_gate_bwd: affine gradient of a norm that is not there");
    NormGateArgs A = {};
    A.u = u, A.r = r, A.gate = gate, A.wa = wa, A.ba = ba, A.wb = wb, A.bb = bb, A.stats = (float4*)stats, A.dy = dy, A.dn = dn, A.du = du, A.dr = dr;
    A.dg = dgate, A.rows = rows, A.d = d, A.gate_rows = gate_kind == PCLIP_GATE_ROWS ? gate_rows : 1, A.gate_kind = gate_kind, A.after = after;
    A.before = before, A.param_f32 = param_type == PCLIP_DT_F32, A.scale = scale, A.eps = eps, A.sum_gate = dgate && A.gate_rows > 1;
    A.wanted = (dwa ? 1 : 0) | (dba ? 2 : 0) | (dwb ? 4 : 0) | (dbb ? 8 : 0);
    const bool affine = A.wanted != 0;
    int blocks = 0;
    plan(A, dtype, affine || A.sum_gate, blocks);
    const bool gate_parts = A.sum_gate && A.chunks > 1;
    const size_t w_floats = affine ? (size_t)blocks * 4 * d : 0, need = (w_floats + (gate_parts ? (size_t)A.groups * A.chunks * d : 0)) * sizeof(float);
    PCLIP_REQUIRE(need == 0 || (ws && ws_bytes >= need), "norm_gate_bwd: workspace too small (%zu bytes, need %zu)", ws_bytes, need);
    A.part_w = affine ? (float*)ws : nullptr;
    A.part_g = gate_parts ? (float*)ws + w_floats : nullptr;
    rc = launch_kernel(A, dtype, false, blocks, (hipStream_t)stream);
    if (rc) return rc;
    if (affine || gate_parts) {
        ColumnSumArgs S = {};
        S.part_w = A.part_w, S.part_g = A.part_g, S.out[0] = dwa, S.out[1] = dba, S.out[2] = dwb, S.out[3] = dbb, S.dg = dgate;
        S.blocks = blocks, S.chunks = A.chunks, S.d = d, S.first_y = affine ? 0 : 4, S.param_type = param_type, S.type = dtype;
        const int ny = (affine ? 4 : 0) + (gate_parts ? A.groups : 0);
        column_sum_kernel<<<dim3((d + 63) / 64, ny), 1024, 0, (hipStream_t)stream>>>(S);
    }
    return pclip_check_launch("norm_gate_bwd");
}
