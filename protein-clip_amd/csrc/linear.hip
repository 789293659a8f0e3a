// Linear layer with bias, activation and residual in its epilogue, and its backward.
//
//   z = x W^T + b,  y = act(z) + r;   dz = dy * act'(z),  dx = dz W,  dW = dz^T x,  db = sum_rows dz
//
// All three products are D[i][j] = sum_k P(i,k) Q(j,k) on the matrix cores (16x16x32 for bf16 / f16, 16x16x4 for f32),
// with f32 sums, and differ in which way P and Q lie in memory: along k (rows x, W, dz in the forward and dx) or along
// i / j (W in dx; dz and x in dW).
#include "elem.h"
#include <math.h>
#include <type_traits>

namespace {

// ---- element types on the matrix cores ------------------------------------------------------
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

template <typename T> struct Mfma;   // Frag: 16 bytes, the k values of one row that a lane feeds to one step
template <> struct Mfma<__bf16> {
    typedef bf16x8 Frag;
    static __device__ __forceinline__ f32x4 step(Frag a, Frag b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};
template <> struct Mfma<_Float16> {
    typedef f16x8 Frag;
    static __device__ __forceinline__ f32x4 step(Frag a, Frag b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
};
template <> struct Mfma<float> {
    typedef f32x4 Frag;
    static __device__ __forceinline__ f32x4 step(Frag a, Frag b, f32x4 c) {
#pragma unroll
        for (int t = 0; t < 4; t++) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[t], b[t], c, 0, 0, 0);
        return c;
    }
};

// ---- tiles in LDS -----------------------------------------------------------------------------
// A tile holds ROWS rows (i or j) of 128 bytes of k (64 16-bit or 32 f32 values), in 16-byte chunks.
//   along k:  chunk (row, c) at row * 128 + ((c ^ row % 8) * 16)
//   along i:  k rows of ROWS elements; chunks permuted by k so that the four k rows which a fragment's read touches
//             at once lie in different banks
// The exchange keeps both the writes (8 lanes a 128-byte row) and the fragment reads (16 rows, or 4 k rows, a step)
// off each other's banks.
template <typename T> constexpr int KSTEP = 128 / (int)sizeof(T);   // k values of a tile

constexpr unsigned DIRECT_RANGE = 1u << 30;   // bytes that a buffer descriptor reaches: more than a tile spans (256 rows of 65536 f32)
// 16 bytes a lane from base + offset to lds + 16 * lane; zeros from DIRECT_RANGE on.  base and lds are the same for the wave.
__device__ __forceinline__ void load_direct(const void* base, unsigned offset, char* lds) {
#ifdef __HIP_DEVICE_COMPILE__   // the host pass has no descriptor type
    const auto rsrc = __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, DIRECT_RANGE, 0x00020000);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (__attribute__((address_space(3))) void*)lds, 16, offset, 0, 0, 0);
#endif
}

constexpr int VMCNT_0 = 0x0F70;   // s_waitcnt: no vector memory access under way; the other counters as they are

template <typename T, int ROWS, bool ALONG_K>
struct Tile {
    static constexpr int V = PclipVec<T>::N;
    static constexpr int CHUNKS = ROWS * 8;               // of 16 bytes
    static constexpr int ICH = ROWS / V;                  // along i: chunks of a k row
    typedef typename Mfma<T>::Frag Frag;

    static __device__ __forceinline__ int swizzle_i(int k) {
        if constexpr (sizeof(T) == 2) return (((k & 3) | ((k >> 1) & 4)) << 1) & (ICH - 1);
        else return (((k >> 2) & 3) << 2) & (ICH - 1);
    }
    // byte offset of chunk number c, and the (row, k) of its first element within the tile
    static __device__ __forceinline__ int slot(int c, int& row, int& k) {
        if constexpr (ALONG_K) {
            row = c >> 3;
            k = (c & 7) * V;
            return row * 128 + (((c & 7) ^ (row & 7)) << 4);
        } else {
            k = c / ICH;
            const int ch = c % ICH;
            row = ch * V;
            return k * ROWS * (int)sizeof(T) + ((ch ^ swizzle_i(k)) << 4);
        }
    }
    // the fragment of rows i0 .. i0 + 15 at k step kk: lane l holds row l % 16, group l / 16 of the step's k values
    static __device__ __forceinline__ Frag frag(const char* lds, int i0, int kk, int lane) {
        const int r = lane & 15, q = lane >> 4;
        if constexpr (ALONG_K) {
            const int row = i0 + r;
            return *(const Frag*)(lds + row * 128 + (((kk * 4 + q) ^ (row & 7)) << 4));
        } else if constexpr (sizeof(T) == 2) {
            // two transposing reads of 4 k rows x 16 elements: the lane gives the address of 4 elements of k row
            // 8q + 4j + r / 4 and receives the 4 k values of its own element
            union { s16x4 h[2]; Frag f; } u;
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const int k = kk * 32 + q * 8 + j * 4 + (r >> 2), i = i0 + (r & 3) * 4;
                const char* p = lds + k * ROWS * 2 + (((i >> 3) ^ swizzle_i(k)) << 4) + (i & 4) * 2;
                u.h[j] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)p);
            }
            return u.f;
        } else {
            Frag f;
#pragma unroll
            for (int t = 0; t < 4; t++) {
                const int k = kk * 16 + q * 4 + t, i = i0 + r;
                f[t] = *(const float*)(lds + k * ROWS * 4 + (((i >> 2) ^ swizzle_i(k)) << 4) + (i & 3) * 4);
            }
            return f;
        }
    }
    // chunk c of the tile whose first row is i0 and first k is k0: elements outside rows x k are zero
    static __device__ __forceinline__ u32x4 fetch_edge(const T* p, int ld, int i0, int rows, long long k0, long long k_end, int c) {
        int row, k;
        slot(c, row, k);
        const long long kk = k0 + k;
        const int i = i0 + row;
        const long long valid = ALONG_K ? (i < rows ? k_end - kk : 0) : (kk < k_end ? rows - i : 0);
        const T* at = ALONG_K ? p + (long long)i * ld + kk : p + kk * ld + i;
        PclipPack<T, V> a;
#pragma unroll
        for (int e = 0; e < V; e++) a.v[e] = e < valid ? at[e] : (T)0.f;
        return __builtin_bit_cast(u32x4, a);
    }
    // Inside the matrix a chunk's address is the tile's (the same for all lanes, kept in scalar registers) plus this offset,
    // which no step changes.  Rows behind the last one read the last one again when they lie along k: nothing of them is stored.
    static __device__ __forceinline__ unsigned offset(int ld, int i0, int rows, int c) {
        int row, k;
        slot(c, row, k);
        if (ALONG_K) row = min(row, rows - 1 - i0);
        return (unsigned)(ALONG_K ? row * ld + k : k * ld + row) * (unsigned)sizeof(T);
    }
    static __device__ __forceinline__ const char* origin(const T* p, int ld, int i0, long long k0) {
        return (const char*)(ALONG_K ? p + (long long)i0 * ld + k0 : p + k0 * ld + i0);
    }
    // Straight to LDS, 16 bytes a lane in the order of the lanes: place c of the tile takes the chunk that slot() puts there.
    static __device__ __forceinline__ int direct_k(int c) { return ALONG_K ? ((c & 7) ^ ((c >> 3) & 7)) * V : c / ICH; }
    static __device__ __forceinline__ unsigned direct_offset(int ld, int i0, int rows, int c) {
        const int k = direct_k(c), row = ALONG_K ? c >> 3 : ((c % ICH) ^ swizzle_i(c / ICH)) * V;
        return i0 + row < rows ? (unsigned)(ALONG_K ? row * ld + k : k * ld + row) * (unsigned)sizeof(T) : DIRECT_RANGE;
    }
    static __device__ __forceinline__ bool inside(int i0, int rows) { return ALONG_K || i0 + ROWS <= rows; }
};

// ---- activations --------------------------------------------------------------------------------
// act(z) and its slope.  f32 results use the library's erf and exp.  For 16-bit results the Gaussian tail is
// Phi(-a) = exp(-a^2 / 2) * P(1 / (1 + 0.3 a)), P a polynomial fitted to erfcx(a / sqrt 2) / 2 by reweighted least
// squares over 0 <= a <= 13: 1.9e-6 relative error, a hundredth of an f16 half step, in one exp and one reciprocal,
// and z Phi(z) = max(z, 0) - a Phi(-a), Phi(z) + z phi(z) = exp(-a^2 / 2) (P - a / sqrt(2 pi)) or one minus that.
// Arguments are cut off where only their product with a factor that has vanished remains, so that an infinite z has the
// limits of value and slope; a NaN passes through the factor.
template <bool EXACT, int ACT>
__device__ __forceinline__ float activate(float z, float& slope) {
    if constexpr (ACT == PCLIP_ACT_RELU) {
        slope = z <= 0.f ? 0.f : 1.f;   // a NaN passes, both ways
        return z <= 0.f ? 0.f : z;
    } else if constexpr (ACT == PCLIP_ACT_GELU && EXACT) {
        const float phi = 0.5f * erfcf(z * -0.70710678118654752f);
        slope = fmaf(fminf(fmaxf(z, -40.f), 40.f) * 0.39894228040143268f, expf(-0.5f * z * z), phi);
        return fmaxf(z, -40.f) * phi;
    } else if constexpr (ACT == PCLIP_ACT_GELU) {
        const float a = fminf(fabsf(z), 40.f), t = __builtin_amdgcn_rcpf(fmaf(0.3f, a, 1.f));
        const float e = __builtin_amdgcn_exp2f(z * -0.72134752044448170f * z);
        float p = -0.0845887363f;
        p = fmaf(p, t, 0.240555853f);
        p = fmaf(p, t, -0.0486187227f);
        p = fmaf(p, t, 0.164744467f);
        p = fmaf(p, t, 0.106712937f);
        p = fmaf(p, t, 0.121272907f);
        p = fmaf(p, t, -7.96368695e-05f);
        const float w = e * fmaf(-0.39894228040143268f, a, p);
        slope = z < 0.f ? w : 1.f - w;
        return fmaf(-a, p * e, fmaxf(z, 0.f));
    } else if constexpr (ACT == PCLIP_ACT_SILU) {
        float s;
        if constexpr (EXACT) s = 1.f / (1.f + expf(-z));
        else s = __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(z * -1.44269504088896341f));
        const float y = fmaxf(z, -100.f) * s;
        slope = fmaf(fminf(y, 100.f), 1.f - s, s);
        return y;
    } else {
        slope = 1.f;
        return z;
    }
}

// The slope is kept for the backward with the precision of a product's operand at every size, since the gradients of units that lie far
// out rest on small slopes: in f32 for f32 and f16 operands, for bf16 as a 16-bit float of 11 bits (three more than dz keeps), times 2^15, which
// puts slopes down to 2^-29 (gelu at -6.6, silu at -23) among its normal numbers and those up to 1.13 below its largest.  16-bit fixed
// point, which was 1e-5 off near one, was 3 % off at gelu's -4 and zero from -5 on; f16 operands want more bits near one than a
// 16-bit float has (their error would rise from 2.9e-4 to 3.6e-4).
template <typename T> struct SlopeFormat { typedef float Type; static constexpr float SCALE = 1.f; };
template <> struct SlopeFormat<__bf16> { typedef _Float16 Type; static constexpr float SCALE = 32768.f; };
template <typename T> using SlopeOf = typename SlopeFormat<T>::Type;

template <typename T, int V>
__device__ __forceinline__ void store_slope(SlopeOf<T>* p, int valid, float (&v)[V]) {
#pragma unroll
    for (int i = 0; i < V; i++) v[i] *= SlopeFormat<T>::SCALE;
    stream_f32<SlopeOf<T>, V>(p, valid, v);
}

// ---- the product -----------------------------------------------------------------------------------
// what becomes of the sums: below EPI_STORE the forward's epilogue with that activation
enum { EPI_STORE = PCLIP_ACT_SILU + 1, EPI_SLAB };

struct GemmArgs {
    const void *P, *Q;
    int ldp, ldq, I, J;
    long long K, k_split;           // contraction length, and the part of one workgroup (a multiple of KSTEP)
    int tiles_i, tiles_j, splits, blocks;   // blocks: tiles of all splits
    const void *bias, *residual;    // forward
    void *out, *slope;
    float *slab, *row_sum;          // EPI_SLAB: [splits][I][J], [splits][I]; slab NULL (one split): straight into out and slope
    bool sum_rows;                  // EPI_SLAB: the sums over P's rows are wanted, too
};

// The rows' sums as one more column of the product, of ones: the first half of a wave's rows, or the second.  (`first` comes
// from a scalar: matrix instructions run whatever the lanes' mask says, so no branch around them may be the lanes' own.)
template <typename T, int FI>
__device__ __forceinline__ void add_rows(const typename Mfma<T>::Frag (&fp)[FI], typename Mfma<T>::Frag one, bool first, f32x4 (&ones)[FI / 2]) {
    if (first) {
#pragma unroll
        for (int i = 0; i < FI / 2; i++) ones[i] = Mfma<T>::step(one, fp[i], ones[i]);
    } else {
#pragma unroll
        for (int i = 0; i < FI / 2; i++) ones[i] = Mfma<T>::step(one, fp[FI / 2 + i], ones[i]);
    }
}

// f32 products are summed in runs of RUN steps (256 k values), whose sums are added: one chain over 2560 k values ends up 1e-6 off, runs
// 3e-7, for some twenty registers a 64 x 64 tile and a few hundredths of the time.  16-bit results do not show it.
constexpr int RUN = 8;
template <typename T, int FI, int FJ>
struct Runs {
    static constexpr bool ON = sizeof(T) == 4;
    f32x4 total[ON ? FI : 1][ON ? FJ : 1], total_ones[ON ? FI / 2 : 1];
    int step = 0;
    __device__ __forceinline__ Runs() {
        if constexpr (ON)
#pragma unroll
            for (int i = 0; i < FI; i++) {
                total_ones[i / 2] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int j = 0; j < FJ; j++) total[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
            }
    }
    static __device__ __forceinline__ void move(f32x4& total, f32x4& acc, bool last) {
        total += acc;
        acc = last ? total : f32x4{0.f, 0.f, 0.f, 0.f};
    }
    __device__ __forceinline__ void end_of_step(f32x4 (&acc)[FI][FJ], f32x4 (&ones)[FI / 2], bool last) {
        if constexpr (ON) {
            if (++step % RUN && !last) return;
#pragma unroll
            for (int i = 0; i < FI; i++) {
                if (i % 2 == 0) move(total_ones[i / 2], ones[i / 2], last);
#pragma unroll
                for (int j = 0; j < FJ; j++) move(total[i][j], acc[i][j], last);
            }
        }
    }
};

// A launch has fewer than 2^32 threads, and a column of 2^31 rows has more tiles than that: workgroups lie in planes of PLANE (a
// multiple of eight, so that the order below goes on over their border), of which the last may hold some that have no tile.
constexpr int PLANE = 1 << 23;
__device__ __forceinline__ int workgroup() { return (int)(blockIdx.y * PLANE + blockIdx.x); }

// Workgroups go to the eight XCDs in turn; give each XCD a run of neighbouring tiles, which share rows of P or Q in its L2.
__device__ __forceinline__ int xcd_order(int b, int n) {
    const int xcd = b & 7, q = n >> 3, r = n & 7;
    return xcd * q + min(xcd, r) + (b >> 3);
}

// between the writes and the reads of LDS by which the lanes of a wave exchange values, and before the next writes
__device__ __forceinline__ void wave_exchange() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// bias, activation, slope and residual of V sums in one row of the result, `left` of them inside it
template <typename T, int EPI, int V>
__device__ __forceinline__ void epilogue(const GemmArgs& A, size_t at, const float (&bias)[V], int left, float (&v)[V]) {
    float slope[V];
#pragma unroll
    for (int e = 0; e < V; e++) v[e] = activate<sizeof(T) == 4, EPI>(v[e] + bias[e], slope[e]);
    if constexpr (EPI == PCLIP_ACT_RELU && std::is_same_v<T, _Float16>) {
        // the backward reads the slope from the output: a value above zero that rounds to zero becomes -0 (bfloat16 reaches
        // as far down as the f32 sums do)
#pragma unroll
        for (int e = 0; e < V; e++) v[e] = v[e] > 0.f && v[e] <= 0x1p-25f ? -0.f : v[e];
    }
    if (A.slope) store_slope<T, V>((SlopeOf<T>*)A.slope + at, left, slope);
    if (A.residual) {
        float res[V];
        load_f32<T, V>((const T*)A.residual + at, left, res);
#pragma unroll
        for (int e = 0; e < V; e++) v[e] += res[e];
    }
}

// What a wave does with its accumulators: rows from i0, columns from j0 on.
template <typename T, int FI, int FJ, int EPI>
__device__ __forceinline__ void finish(const GemmArgs& A, f32x4 (&acc)[FI][FJ], f32x4 (&ones)[FI / 2], bool sum_rows, char* lds, int i0, int j0, int split) {
    const int lane = threadIdx.x & 63;
    // a lane holds, of every 16 x 16 tile, row i = lane % 16 and the four columns from j = 4 * (lane / 16) on
    if constexpr (EPI == EPI_SLAB) {
#pragma unroll
        for (int fi = 0; fi < FI; fi++) {
            const int i = i0 + fi * 16 + (lane & 15);
            if (i >= A.I) continue;
#pragma unroll
            for (int fj = 0; fj < FJ; fj++) {
                const int j = j0 + fj * 16 + (lane >> 4) * 4;
                float v[4];
#pragma unroll
                for (int e = 0; e < 4; e++) v[e] = acc[fi][fj][e];
                if (j >= A.J) continue;
                if (A.slab) store_f32<float, 4>(A.slab + ((size_t)split * A.I + i) * A.J + j, A.J - j, v);
                else store_f32<T, 4>((T*)A.out + (size_t)i * A.J + j, A.J - j, v);
            }
            const bool first = (threadIdx.x >> 6 & 1) == 0;   // the column of waves, see add_rows
            if (sum_rows && lane < 16 && first == (fi < FI / 2)) {
                if (A.slab) A.row_sum[(size_t)split * A.I + i] = ones[fi % (FI / 2)][0];
                else ((T*)A.slope)[i] = (T)ones[fi % (FI / 2)][0];
            }
        }
    } else {
        // 16 rows at a time through LDS (a wave's own part of it), after which a lane holds the V columns of one 16-byte access and
        // neighbouring lanes neighbouring ones: whole lines are written, and read of the residual.  Only lanes of one wave exchange values,
        // whose LDS accesses are executed in order: wave_exchange keeps the compiler to that order, and no instruction comes of it
        constexpr int V = PclipVec<T>::N, WC = FJ * 16, PITCH = WC + 4, LANES = WC / V, ROWS = 64 / LANES;
        __syncthreads();
        float* own = (float*)lds + (threadIdx.x >> 6) * 16 * PITCH;
        const int c = (lane % LANES) * V, j = j0 + c, left = A.J - j;
        float bias[V];
        if (EPI < EPI_STORE) {
#pragma unroll
            for (int e = 0; e < V; e++) bias[e] = 0.f;
            if (A.bias) load_f32<T, V>((const T*)A.bias + j, left, bias);
        }
#pragma unroll
        for (int fi = 0; fi < FI; fi++) {
#pragma unroll
            for (int fj = 0; fj < FJ; fj++) *(f32x4*)(own + (lane & 15) * PITCH + fj * 16 + (lane >> 4) * 4) = acc[fi][fj];
            wave_exchange();
#pragma unroll
            for (int first = 0; first < 16; first += ROWS) {
                const int row = first + lane / LANES, i = i0 + fi * 16 + row;
                float v[V];
#pragma unroll
                for (int e = 0; e < V; e += 4) *(f32x4*)(v + e) = *(const f32x4*)(own + row * PITCH + c + e);
                if (i >= A.I || left <= 0) continue;
                const size_t at = (size_t)i * A.J + j;
                if constexpr (EPI < EPI_STORE) epilogue<T, EPI, V>(A, at, bias, left, v);
                stream_f32<T, V>((T*)A.out + at, left, v);
            }
            wave_exchange();
        }
    }
}

template <typename T, int BI, int BJ, int WI, int WJ, bool PK, bool QK, int EPI>
__global__ __launch_bounds__(64 * WI * WJ, 2) void gemm_kernel(const GemmArgs A) {
    typedef Tile<T, BI, PK> TP;
    typedef Tile<T, BJ, QK> TQ;
    typedef typename Mfma<T>::Frag Frag;
    constexpr int N = 64 * WI * WJ, NP = TP::CHUNKS / N, NQ = TQ::CHUNKS / N;
    constexpr int FI = BI / WI / 16, FJ = BJ / WJ / 16, BYTES = (BI + BJ) * 128;
    extern __shared__ __attribute__((aligned(16))) char lds[];

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    if (workgroup() >= A.blocks) return;
    int b = xcd_order(workgroup(), A.blocks);
    const int tj = b % A.tiles_j;
    b /= A.tiles_j;
    const int ti = b % A.tiles_i, split = b / A.tiles_i;
    const int i0 = ti * BI, j0 = tj * BJ;
    const int wi = (wave / WJ) * (BI / WI), wj = (wave % WJ) * (BJ / WJ);
    const long long k_first = split * A.k_split, k_end = k_first + A.k_split < A.K ? k_first + A.k_split : A.K;
    const T *P = (const T*)A.P, *Q = (const T*)A.Q;

    u32x4 rp[NP], rq[NQ];
    unsigned op[NP], oq[NQ];
#pragma unroll
    for (int n = 0; n < NP; n++) op[n] = TP::offset(A.ldp, i0, A.I, tid + n * N);
#pragma unroll
    for (int n = 0; n < NQ; n++) oq[n] = TQ::offset(A.ldq, j0, A.J, tid + n * N);
    const bool p_inside = TP::inside(i0, A.I), q_inside = TQ::inside(j0, A.J);
    auto fetch = [&](long long k0) {
        const bool whole = k0 + KSTEP<T> <= k_end;
        if (whole && p_inside) {
            const char* at = TP::origin(P, A.ldp, i0, k0);
#pragma unroll
            for (int n = 0; n < NP; n++) rp[n] = __builtin_bit_cast(u32x4, *(const PclipPack<T, TP::V>*)(at + op[n]));
        } else {
#pragma unroll
            for (int n = 0; n < NP; n++) rp[n] = TP::fetch_edge(P, A.ldp, i0, A.I, k0, k_end, tid + n * N);
        }
        if (whole && q_inside) {
            const char* at = TQ::origin(Q, A.ldq, j0, k0);
#pragma unroll
            for (int n = 0; n < NQ; n++) rq[n] = __builtin_bit_cast(u32x4, *(const PclipPack<T, TQ::V>*)(at + oq[n]));
        } else {
#pragma unroll
            for (int n = 0; n < NQ; n++) rq[n] = TQ::fetch_edge(Q, A.ldq, j0, A.J, k0, k_end, tid + n * N);
        }
    };
    f32x4 acc[FI][FJ], ones[FI / 2];
#pragma unroll
    for (int i = 0; i < FI; i++) {
        ones[i / 2] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < FJ; j++) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    Runs<T, FI, FJ> runs;
    Frag one;
#pragma unroll
    for (int e = 0; e < PclipVec<T>::N; e++) one[e] = (T)1.f;
    const bool sum_rows = EPI == EPI_SLAB && A.sum_rows && tj == 0;   // each column of waves half of its rows

    fetch(k_first);
    int buf = 0;
    for (long long k = k_first; k < k_end; k += KSTEP<T>) {
        char *lp = lds + buf * BYTES, *lq = lp + BI * 128;
        int row, kk;
#pragma unroll
        for (int n = 0; n < NP; n++) *(u32x4*)(lp + TP::slot(tid + n * N, row, kk)) = rp[n];
#pragma unroll
        for (int n = 0; n < NQ; n++) *(u32x4*)(lq + TQ::slot(tid + n * N, row, kk)) = rq[n];
        __syncthreads();   // the other buffer's readers were done before they came here
        if (k + KSTEP<T> < k_end) fetch(k + KSTEP<T>);
#pragma unroll
        for (int s = 0; s < 2; s++) {
            Frag fp[FI], fq[FJ];
#pragma unroll
            for (int i = 0; i < FI; i++) fp[i] = TP::frag(lp, wi + i * 16, s, lane);
#pragma unroll
            for (int j = 0; j < FJ; j++) fq[j] = TQ::frag(lq, wj + j * 16, s, lane);
#pragma unroll
            for (int i = 0; i < FI; i++)
#pragma unroll
                for (int j = 0; j < FJ; j++) acc[i][j] = Mfma<T>::step(fq[j], fp[i], acc[i][j]);
            if (sum_rows) add_rows<T, FI>(fp, one, wj == 0, ones);
        }
        runs.end_of_step(acc, ones, k + KSTEP<T> >= k_end);
        buf ^= 1;
    }

    finish<T, FI, FJ, EPI>(A, acc, ones, sum_rows, lds, i0 + wi, j0 + wj, split);
}

// The same product for operands whose rows begin at multiples of 16 bytes: tiles go from memory to LDS directly.  One buffer of
// LDS is enough, because a wave takes all its fragments of a step into registers first; the next tile is on its way while
// the matrix cores work, and two or three workgroups share a compute unit.  Chunks outside the matrix are read at an offset
// beyond the descriptor's range, which writes zeros.  Bound by the matrix cores and the reads of LDS (a 64 x 64 part of a
// tile reads 16 KB for 32 matrix instructions, 128 x 64 24 KB for 64): 65,536 x 2560 -> 640 bf16 220 us, 978 TFLOP/s; dW 269 us,
// 797; 16,384 x 1280 -> 1280 54.5 us, 986.  The staged form: 541 at 16,383 x 1283 -> 1279.
template <typename T, int BI, int BJ, int WI, int WJ, bool PK, bool QK, int EPI>
__global__ __launch_bounds__(64 * WI * WJ, 2) void gemm_direct_kernel(const GemmArgs A) {
    typedef Tile<T, BI, PK> TP;
    typedef Tile<T, BJ, QK> TQ;
    typedef typename Mfma<T>::Frag Frag;
    constexpr int N = 64 * WI * WJ, NP = TP::CHUNKS / N, NQ = TQ::CHUNKS / N;
    constexpr int FI = BI / WI / 16, FJ = BJ / WJ / 16;
    extern __shared__ __attribute__((aligned(16))) char lds[];

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    if (workgroup() >= A.blocks) return;
    int b = xcd_order(workgroup(), A.blocks);
    const int tj = b % A.tiles_j;
    b /= A.tiles_j;
    const int ti = b % A.tiles_i, split = b / A.tiles_i;
    const int i0 = ti * BI, j0 = tj * BJ;
    const int wi = (wave / WJ) * (BI / WI), wj = (wave % WJ) * (BJ / WJ);
    const long long k_first = split * A.k_split, k_end = k_first + A.k_split < A.K ? k_first + A.k_split : A.K;
    const T *P = (const T*)A.P, *Q = (const T*)A.Q;

    unsigned op[NP], oq[NQ];
#pragma unroll
    for (int n = 0; n < NP; n++) op[n] = TP::direct_offset(A.ldp, i0, A.I, tid + n * N);
#pragma unroll
    for (int n = 0; n < NQ; n++) oq[n] = TQ::direct_offset(A.ldq, j0, A.J, tid + n * N);
    auto fetch = [&](long long k0) {
        const long long left = k_end - k0;
        const void *at_p = TP::origin(P, A.ldp, i0, k0), *at_q = TQ::origin(Q, A.ldq, j0, k0);
        char *lp = lds + wave * 1024, *lq = lp + BI * 128;
        if (left >= KSTEP<T>) {
#pragma unroll
            for (int n = 0; n < NP; n++) load_direct(at_p, op[n], lp + n * N * 16);
#pragma unroll
            for (int n = 0; n < NQ; n++) load_direct(at_q, oq[n], lq + n * N * 16);
        } else {
#pragma unroll
            for (int n = 0; n < NP; n++) load_direct(at_p, TP::direct_k(tid + n * N) < left ? op[n] : DIRECT_RANGE, lp + n * N * 16);
#pragma unroll
            for (int n = 0; n < NQ; n++) load_direct(at_q, TQ::direct_k(tid + n * N) < left ? oq[n] : DIRECT_RANGE, lq + n * N * 16);
        }
    };
    f32x4 acc[FI][FJ], ones[FI / 2];
#pragma unroll
    for (int i = 0; i < FI; i++) {
        ones[i / 2] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < FJ; j++) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    Runs<T, FI, FJ> runs;
    Frag one;
#pragma unroll
    for (int e = 0; e < PclipVec<T>::N; e++) one[e] = (T)1.f;
    const bool sum_rows = EPI == EPI_SLAB && A.sum_rows && tj == 0;   // each column of waves half of its rows

    fetch(k_first);
    for (long long k = k_first; k < k_end; k += KSTEP<T>) {
        __builtin_amdgcn_s_waitcnt(VMCNT_0);   // this wave's part of the tile has arrived in LDS (the barrier's own fence waits for it as well)
        __syncthreads();   // every wave's part of the tile is there
        Frag fp[2][FI], fq[2][FJ];
#pragma unroll
        for (int s = 0; s < 2; s++) {
#pragma unroll
            for (int j = 0; j < FJ; j++) fq[s][j] = TQ::frag(lds + BI * 128, wj + j * 16, s, lane);
#pragma unroll
            for (int i = 0; i < FI; i++) fp[s][i] = TP::frag(lds, wi + i * 16, s, lane);
        }
        __syncthreads();   // and in every wave's registers: LDS may be written again
        if (k + KSTEP<T> < k_end) fetch(k + KSTEP<T>);
#pragma unroll
        for (int s = 0; s < 2; s++) {
#pragma unroll
            for (int i = 0; i < FI; i++)
#pragma unroll
                for (int j = 0; j < FJ; j++) acc[i][j] = Mfma<T>::step(fq[s][j], fp[s][i], acc[i][j]);
            if (sum_rows) add_rows<T, FI>(fp[s], one, wj == 0, ones);
        }
        runs.end_of_step(acc, ones, k + KSTEP<T> >= k_end);
    }
    finish<T, FI, FJ, EPI>(A, acc, ones, sum_rows, lds, i0 + wi, j0 + wj, split);
}

// The forward's and dx's split contraction: the slabs of the splits added in order, then the epilogue.  A thread takes four columns of a row.
template <typename T, int EPI>
__global__ __launch_bounds__(256) void join_kernel(const GemmArgs A) {
    const int vecs = (A.J + 3) / 4;
    const long long n = (long long)blockIdx.x * 256 + threadIdx.x;
    if (n >= (long long)A.I * vecs) return;
    const int i = (int)(n / vecs), j = (int)(n % vecs) * 4, left = A.J - j;
    const size_t at = (size_t)i * A.J + j, slab = (size_t)A.I * A.J;
    float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int k = 0; k < A.splits; k++) {
        float part[4];
        load_f32<float, 4>(A.slab + k * slab + at, left, part);
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] += part[e];
    }
    if constexpr (EPI < EPI_STORE) {
        float bias[4] = {0.f, 0.f, 0.f, 0.f};
        if (A.bias) load_f32<T, 4>((const T*)A.bias + j, left, bias);
        epilogue<T, EPI, 4>(A, at, bias, left, v);
    }
    stream_f32<T, 4>((T*)A.out + at, left, v);
}

// out[e] = sum over the splits' slabs in a fixed order, rounded once; blocks behind those of the weight's gradient sum the bias's.
// A workgroup takes 16 x 4 elements in 16 parts of the splits, of the bias's few elements and many splits 4 x 4 in 64 parts.
struct SlabSum {
    const float* slab[2];
    void* out[2];
    long long n[2];
    int splits[2], blocks;   // blocks: of the first sum
};
constexpr int SUM_LANES[2] = {16, 4};
template <typename T>
__global__ __launch_bounds__(256) void slab_sum_kernel(const SlabSum A) {
    __shared__ float lds[256][4];
    const int which = (int)blockIdx.x >= A.blocks, lanes = which ? SUM_LANES[1] : SUM_LANES[0], parts = 256 / lanes, splits = A.splits[which];
    const int lane = threadIdx.x % lanes, part = threadIdx.x / lanes;
    const long long n = A.n[which], e = (((long long)blockIdx.x - (which ? A.blocks : 0)) * lanes + lane) * 4, left = n - e;
    const int valid = left < 4 ? (int)left : 4;
    float s[4] = {0.f, 0.f, 0.f, 0.f};
    if (valid > 0)
#pragma unroll 4
        for (int k = part; k < splits; k += parts) {
            float v[4];
            load_f32<float, 4>(A.slab[which] + (size_t)k * n + e, valid, v);
#pragma unroll
            for (int c = 0; c < 4; c++) s[c] += v[c];
        }
    for (int o = 128; o >= lanes; o >>= 1) {
#pragma unroll
        for (int c = 0; c < 4; c++) lds[threadIdx.x][c] = s[c];
        __syncthreads();
        if ((int)threadIdx.x < o)
#pragma unroll
            for (int c = 0; c < 4; c++) s[c] += lds[threadIdx.x + o][c];
        __syncthreads();
    }
    if (part == 0 && valid > 0) store_f32<T, 4>((T*)A.out[which] + e, valid, s);
}

// Bound by memory: 1.0 GB for 65,536 x 2560 bf16 in 204 us, 4.9 TB/s (before the column sums were added: 180-197 us, with one access under
// way instead of four 245).
// dz = dy * slope, or dy where the output is not +0, rounded to the operands' type: a choice, since the matrix cores take no wider operand
// beside a 16-bit one.  It leaves dx and dW 1.4 times as far from the exact ones as one rounding at the end would (bf16 0.0024 instead of
// 0.0017 in the 2-norm, f16 0.00029 and 0.00021); a second 16-bit part of dz would halve the rate of both products, half of the time of
// a training pass.  And the column sums of the unrounded products, from which the
// bias's gradient comes (the rounded ones would bring it the errors of M roundings).  `lanes` neighbouring threads take a row's
// vectors, 256 / lanes rows at once; a workgroup takes `rows` rows of its columns, with four accesses of each operand under way.
struct SlopeArgs {
    const void *dy, *saved;
    void *dz, *db;        // dz: NULL when only the sums are wanted; db: written when one workgroup holds all rows
    float* sums;          // [workgroups over the rows][N], or NULL when no sums are wanted or db takes them
    int M, N, lanes, rows;
};
// HOW: what dy is multiplied by; S: its type
enum { BY_SLOPE, BY_OUTPUT, BY_NOTHING };   // BY_NOTHING: dz is dy and not written, only the sums are wanted (S is not read)
template <typename T, typename S, int HOW>
__global__ __launch_bounds__(256) void slope_kernel(const SlopeArgs A) {
    constexpr int V = PclipVec<T>::N, AHEAD = 4;
    typedef PclipPack<T, V> Pack;
    typedef PclipPack<S, V> Saved;
    typedef std::conditional_t<sizeof(S) == 4, unsigned, unsigned short> Bits;
    __shared__ float lds[256][V + 1];
    const int c = ((int)blockIdx.x * A.lanes + (int)threadIdx.x % A.lanes) * V, valid = A.N - c, step = 256 / A.lanes;
    const int begin = (int)blockIdx.y * A.rows, end = A.M - begin > A.rows ? begin + A.rows : A.M;
    const T* dy = (const T*)A.dy;
    const S* saved = (const S*)A.saved;
    T* dz = (T*)A.dz;
    float sum[V];
#pragma unroll
    for (int i = 0; i < V; i++) sum[i] = 0.f;
    auto product = [](T d, S s) {
        if constexpr (HOW == BY_NOTHING) return (float)d;
        else if constexpr (HOW == BY_OUTPUT) return __builtin_bit_cast(Bits, s) == 0 ? 0.f : (float)d;   // zero only at +0; NaN, and -0 (see finish), pass
        else return (float)d * ((float)s * (1.f / SlopeFormat<T>::SCALE));
    };
    int row = begin + (int)threadIdx.x / A.lanes;
    // the last vector of a row that does not divide into vectors is read from V columns before the row's end on, and what
    // it shares with the one before is left out (rows shorter than a vector go element by element)
    const int twice = valid >= V ? 0 : V - valid;
    if (valid > 0 && A.N >= V) {
        const int from = c - twice;
        auto use = [&](const Pack& d, const Saved& s, size_t at) {
            float x[V];
#pragma unroll
            for (int i = 0; i < V; i++) {
                x[i] = product(d.v[i], s.v[i]);
                sum[i] += x[i];
            }
            if (HOW == BY_NOTHING || !dz) return;
            if (twice == 0) {
                store_f32<T, V>(dz + at, V, x);
            } else {
#pragma unroll
                for (int i = 1; i < V; i++)
                    if (i >= twice) dz[at + i] = (T)x[i];
            }
        };
        for (; end - row > (AHEAD - 1) * step; row += AHEAD * step) {
            Pack d[AHEAD];
            Saved s[AHEAD];
#pragma unroll
            for (int q = 0; q < AHEAD; q++) {
                const size_t at = (size_t)(row + q * step) * A.N + from;
                d[q] = *(const Pack*)(dy + at);
                if constexpr (HOW != BY_NOTHING) s[q] = *(const Saved*)(saved + at);
            }
#pragma unroll
            for (int q = 0; q < AHEAD; q++) use(d[q], s[q], (size_t)(row + q * step) * A.N + from);
        }
        for (; row < end; row += step) {
            const size_t at = (size_t)row * A.N + from;
            if constexpr (HOW == BY_NOTHING) use(*(const Pack*)(dy + at), Saved{}, at);
            else use(*(const Pack*)(dy + at), *(const Saved*)(saved + at), at);
        }
#pragma unroll
        for (int i = 0; i < V; i++) {   // the columns from c on come first
            float moved = sum[i];
#pragma unroll
            for (int k = 1; k < V; k++)
                if (twice == k && i + k < V) moved = sum[i + k];
            sum[i] = moved;
        }
    } else if (valid > 0) {
        for (; row < end; row += step)
#pragma unroll
            for (int i = 0; i < V; i++)
                if (i < valid) {
                    const size_t at = (size_t)row * A.N + c + i;
                    const float x = HOW == BY_NOTHING ? (float)dy[at] : product(dy[at], saved[at]);
                    sum[i] += x;
                    if (HOW != BY_NOTHING && dz) dz[at] = (T)x;
                }
    }
    if (!A.sums && !A.db) return;
#pragma unroll
    for (int i = 0; i < V; i++) lds[threadIdx.x][i] = sum[i];
    __syncthreads();
    if ((int)threadIdx.x < A.lanes && valid > 0) {
        for (int t = A.lanes; t < 256; t += A.lanes)
#pragma unroll
            for (int i = 0; i < V; i++) sum[i] += lds[threadIdx.x + t][i];
        if (A.db) store_f32<T, V>((T*)A.db + c, valid, sum);
        else store_f32<float, V>(A.sums + (size_t)blockIdx.y * A.N + c, valid, sum);
    }
}

// ---- host side -----------------------------------------------------------------------------------------
template <typename T, int BI, int BJ, bool DIRECT, bool PK, bool QK, int EPI>
int launch_tile(GemmArgs A, hipStream_t st) {
    static PclipLdsLimit limit;
    constexpr size_t bytes = (DIRECT ? 1 : 2) * (size_t)(BI + BJ) * 128;
    const void* fn;
    if constexpr (DIRECT) fn = (const void*)&gemm_direct_kernel<T, BI, BJ, 2, 2, PK, QK, EPI>;
    else fn = (const void*)&gemm_kernel<T, BI, BJ, 2, 2, PK, QK, EPI>;
    const int rc = pclip_ensure_lds(limit, fn, bytes, "linear");
    if (rc) return rc;
    A.tiles_i = (A.I + BI - 1) / BI;
    A.tiles_j = (A.J + BJ - 1) / BJ;
    const long long blocks = (long long)A.tiles_i * A.tiles_j * A.splits;
    PCLIP_REQUIRE(blocks <= 0x7fffffffll, "linear: too many tiles (%lld)", blocks);
    A.blocks = (int)blocks;
    const dim3 grid(A.blocks < PLANE ? A.blocks : PLANE, (unsigned)((blocks + PLANE - 1) / PLANE));
    if constexpr (DIRECT) gemm_direct_kernel<T, BI, BJ, 2, 2, PK, QK, EPI><<<grid, 256, bytes, st>>>(A);
    else gemm_kernel<T, BI, BJ, 2, 2, PK, QK, EPI><<<grid, 256, bytes, st>>>(A);
    return PCLIP_OK;
}

long long tiles(long long i, long long j, int bi, int bj) { return ((i + bi - 1) / bi) * ((j + bj - 1) / bj); }

template <typename T, bool DIRECT, bool PK, bool QK, int EPI>
int launch_size(const GemmArgs& A, int bi, int bj, hipStream_t st) {
    if constexpr (DIRECT && EPI != EPI_SLAB && sizeof(T) == 2)
        if (bi == 256) return launch_tile<T, 256, 128, DIRECT, PK, QK, EPI>(A, st);
    if constexpr ((EPI == EPI_SLAB && DIRECT) || sizeof(T) == 2)   // f32 rows go in small tiles only, see launch_rows and row_plan
        if (bi >= 128) return launch_tile<T, 128, 128, DIRECT, PK, QK, EPI>(A, st);
    return launch_tile<T, 64, 64, DIRECT, PK, QK, EPI>(A, st);
}
// whether every row of both operands begins at a multiple of 16 bytes
template <typename T>
bool direct(const void* P, const void* Q, int ldp, int ldq) {
    const uintptr_t bits = (uintptr_t)P | (uintptr_t)Q | (uintptr_t)ldp * sizeof(T) | (uintptr_t)ldq * sizeof(T);
    return (bits & 15) == 0;
}
template <typename T, bool PK, bool QK, int EPI>
int launch_product(const GemmArgs& A, int bi, int bj, hipStream_t st) {
    return direct<T>(A.P, A.Q, A.ldp, A.ldq) ? launch_size<T, true, PK, QK, EPI>(A, bi, bj, st) : launch_size<T, false, PK, QK, EPI>(A, bi, bj, st);
}

// Forward and dx: the tile whose workgroups are done first.  A compute unit's share is its number of workgroups times the tile's
// area, over what the tile reaches of the matrix cores when several share a unit (16-bit: 256 x 128 a little more than
// 128 x 128, 64 x 64 0.62 of it: 232, 241 and 371 us for 65,536 x 640 -> 2560) and 0.6 of that for one alone, which waits for its own
// loads (4096 x 2560 -> 640: 39 us with one 128 x 128 tile on some units, 31 with three of 64 x 64).  16,384 x 1280 -> 1280: 3 * 256 x 128
// tiles a unit 63 us, 5 * 128 x 128 56 us.  f32 products wait for the matrix cores whatever the tile, so they take the smallest,
// which divides most evenly and leaves room for the runs' sums (8192 x 640 -> 640: 54.5 us, 123 of 154 TFLOP/s).
int row_tile(int I, int J, int dtype) {
    if (dtype == PCLIP_DT_F32) return 64;
    int best = 64;
    double least = 0.0;
    for (int bi : {64, 128, 256}) {
        const int bj = bi == 64 ? 64 : 128;
        const double each = (double)((tiles(I, J, bi, bj) + 255) / 256), reach = (bi == 64 ? 0.62 : bi == 128 ? 1.0 : 1.03) * (each == 1.0 ? 0.6 : 1.0);
        const double cost = each * bi * bj / reach;
        if (bi == 64 || cost < least) best = bi, least = cost;
    }
    return best;
}
// How often the contraction of an f32 product over the rows is split.  A 64 x 64 tile keeps a compute unit busy for 0.5 to 0.65 us a step of 32 k values,
// so few tiles, or some more than divide evenly over the 256 units, leave much of the device idle; splits cost a second launch and two
// passes over their sums.  In microseconds: rounds of tiles x steps x 0.6, and 4 + 8 ns a tile and split.  Unsplit and split:
// 1 x 2560 -> 2560 54 and 15 (library 8), 37 x 2369 -> 1280 62 and 15 (10), 1040 x 2560 -> 320 56 and 27 (24), 1108 x 2560 -> 640 56 and 43 (34),
// 4096 x 2560 -> 640 128 and 116 (114); 300 x 320 -> 320 9.3 and 10.0, 704 x 1280 -> 2560 46 and 54: not split.
struct Split { int splits, k_split; };
Split row_split(int I, int J, int K, int dtype) {
    Split best = {1, (K + 63) / 64 * 64};
    if (dtype != PCLIP_DT_F32) return best;
    const long long t = tiles(I, J, 64, 64);
    const int steps = (K + 31) / 32;
    if (t > 2048) return best;   // eight rounds and more: the last one weighs little
    double least = (double)((t + 255) / 256) * steps * 0.6;
    for (int s = 2; s <= 24 && s * 4 <= steps; s++) {   // four steps at least
        const int per = (steps + s - 1) / s;
        const double cost = (double)((t * s + 255) / 256) * per * 0.6 + 4.0 + 0.008 * (double)(t * s);
        if (cost < least) best = {(steps + per - 1) / per, per * 32}, least = cost;
    }
    return best;
}
size_t split_bytes(int I, int J, int K, int dtype) {
    const int s = row_split(I, J, K, dtype).splits;
    return s > 1 ? pclip_align_up((size_t)s * I * J * sizeof(float), 256) : 0;
}

// slab: split_bytes of scratch, or NULL: in one
template <typename T, bool PK, bool QK, int EPI>
int launch_rows(GemmArgs A, float* slab, hipStream_t st) {
    constexpr int DTYPE = sizeof(T) == 4 ? PCLIP_DT_F32 : PCLIP_DT_BF16;
    A.splits = 1, A.k_split = (A.K + 63) / 64 * 64;
    if constexpr (sizeof(T) == 4) {
        const Split s = row_split(A.I, A.J, (int)A.K, DTYPE);
        if (slab && s.splits > 1) {
            A.splits = s.splits, A.k_split = s.k_split, A.slab = slab;
            const int rc = launch_product<T, PK, QK, EPI_SLAB>(A, 64, 64, st);
            if (rc) return rc;
            join_kernel<T, EPI><<<(unsigned)(((long long)A.I * ((A.J + 3) / 4) + 255) / 256), 256, 0, st>>>(A);
            return PCLIP_OK;
        }
    }
    const int best = row_tile(A.I, A.J, DTYPE);
    return launch_product<T, PK, QK, EPI>(A, best, best == 64 ? 64 : 128, st);
}

// The product over the rows (dW): tile size, the number of splits and their length.  The tile is 128 x 128, or 64 x 64 where a side is
// no longer, and for f32 with few tiles: 16 waves then share a compute unit instead of 8 (4096 x 640 -> 128: 16 us instead
// of 22; 16,384 x 1280 -> 1280, a hundred tiles: 711 instead of 493), and where f32 operands are staged, whose fetched registers and the
// runs' sums of a 128 x 128 tile do not fit (spilled, 16,383 x 1283 -> 1279 846 us instead of 674; 600 x 2049 -> 2047 120 instead of 79).
struct RowPlan { int tile, splits; long long k_split; };
RowPlan row_plan(int M, int K, int N, int dtype, bool staged) {
    const bool f32 = dtype == PCLIP_DT_F32;
    const int step = f32 ? 32 : 64, tile = K > 64 && N > 64 && !(f32 && (staged || tiles(N, K, 128, 128) <= 16)) ? 128 : 64;
    const long long t = tiles(N, K, tile, tile), steps = ((long long)M + step - 1) / step;
    // two workgroups a compute unit, in one round; of the small staged tiles four, and eight in rounds where the tiles alone leave the last
    // round half empty (16,383 x 1283 -> 1279: 980 us with two, 817 with four, 674 with eight; 16,384 x 1281 -> 200: 154, 144, 143)
    long long s = (!(f32 && staged) ? 512 : t > 256 ? 2048 : 1024) / t;
    if (s > (steps + 3) / 4) s = (steps + 3) / 4;   // four steps a workgroup at least
    if (s < 1) s = 1;
    const long long per = (steps + s - 1) / s;
    return {tile, (int)((steps + per - 1) / per), per * step};
}

template <typename T>
int forward(const GemmArgs& A, int act, float* slab, hipStream_t st) {
    if (act == PCLIP_ACT_NONE) return launch_rows<T, true, true, PCLIP_ACT_NONE>(A, slab, st);
    if (act == PCLIP_ACT_RELU) return launch_rows<T, true, true, PCLIP_ACT_RELU>(A, slab, st);
    if (act == PCLIP_ACT_GELU) return launch_rows<T, true, true, PCLIP_ACT_GELU>(A, slab, st);
    return launch_rows<T, true, true, PCLIP_ACT_SILU>(A, slab, st);
}

// how slope_kernel divides M x N: lanes a row, workgroups over the columns and over the rows (of 64 rows at least), rows of each
struct SlopePlan { int lanes, over_n, over_m, rows; };
SlopePlan slope_plan(int M, int N, int dtype) {
    const int V = dtype == PCLIP_DT_F32 ? 4 : 8, vecs = (N + V - 1) / V;
    int lanes = 1;
    while (lanes < vecs && lanes < 64) lanes *= 2;
    const int over_n = (vecs + lanes - 1) / lanes;
    long long rows = ((long long)M * over_n + 2047) / 2048;   // eight workgroups a compute unit
    if (rows < 64) rows = 64;
    return {lanes, over_n, (int)((M + rows - 1) / rows), (int)rows};
}

// where the parts of the workspace lie; `input`: dx is wanted, `product`: dW, `bias_alone`: db without it
struct BackwardLayout { size_t sums, dx, slab, row_sum, bytes; };   // dz at 0
BackwardLayout backward_layout(int M, int K, int N, int dtype, int act, bool input, bool product, bool bias_alone, bool staged) {
    BackwardLayout L = {};
    if (act != PCLIP_ACT_NONE) L.sums = pclip_align_up((size_t)M * N * pclip_dtype_size(dtype), 256);
    L.dx = L.sums;
    if (act != PCLIP_ACT_NONE || bias_alone) {
        const SlopePlan s = slope_plan(M, N, dtype);
        L.dx += s.over_m > 1 ? pclip_align_up((size_t)s.over_m * N * sizeof(float), 256) : 0;
    }
    L.slab = L.dx + (input ? split_bytes(M, K, N, dtype) : 0);
    if (!product) {
        L.bytes = L.slab;
        return L;
    }
    const RowPlan p = row_plan(M, K, N, dtype, staged);
    L.row_sum = L.slab + (p.splits > 1 ? pclip_align_up((size_t)p.splits * N * K * sizeof(float), 256) : 0);
    L.bytes = L.row_sum + (p.splits > 1 && act == PCLIP_ACT_NONE ? (size_t)p.splits * N * sizeof(float) : 0);
    return L;
}

template <typename T>
int backward(const T* x, const T* w, const T* dy, const void* saved, int is_output, int M, int K, int N, int dtype, int act, T* dx, T* dw, T* db, char* ws,
             size_t ws_bytes, hipStream_t st) {
    const bool bias_alone = db && !dw;
    const bool staged = !direct<T>(act == PCLIP_ACT_NONE ? dy : (const T*)ws, x, N, K);
    const BackwardLayout L = backward_layout(M, K, N, dtype, act, dx, dw, bias_alone, staged);
    if (L.bytes > ws_bytes) return pclip_fail(PCLIP_EINVAL, "linear_bwd: workspace too small (%zu bytes, need %zu)", ws_bytes, L.bytes);
    const RowPlan p = row_plan(M, K, N, dtype, staged);
    SlabSum S = {};
    const T* dz = dy;
    if (act != PCLIP_ACT_NONE || bias_alone) {
        const SlopePlan s = slope_plan(M, N, dtype);
        SlopeArgs A = {dy, saved, dx || dw ? ws : nullptr, nullptr, nullptr, M, N, s.lanes, s.rows};
        if (db && s.over_m == 1) A.db = db;
        else if (db) A.sums = (float*)(ws + L.sums), S.slab[1] = A.sums, S.out[1] = db, S.n[1] = N, S.splits[1] = s.over_m;
        const dim3 grid(s.over_n, s.over_m);
        if (act == PCLIP_ACT_NONE) slope_kernel<T, T, BY_NOTHING><<<grid, 256, 0, st>>>(A);
        else if (is_output) slope_kernel<T, T, BY_OUTPUT><<<grid, 256, 0, st>>>(A);
        else slope_kernel<T, SlopeOf<T>, BY_SLOPE><<<grid, 256, 0, st>>>(A);
        if (act != PCLIP_ACT_NONE) dz = (const T*)ws;
    }
    if (dx) {
        GemmArgs A = {};
        A.P = dz, A.Q = w, A.ldp = N, A.ldq = K, A.I = M, A.J = K, A.K = N, A.out = dx;
        const int rc = launch_rows<T, true, false, EPI_STORE>(A, (float*)(ws + L.dx), st);
        if (rc) return rc;
    }
    if (dw) {
        const bool sum_here = db && act == PCLIP_ACT_NONE;   // dz is dy, exactly: its sums ride on the product
        GemmArgs A = {};
        A.P = dz, A.Q = x, A.ldp = N, A.ldq = K, A.I = N, A.J = K, A.K = M, A.k_split = p.k_split, A.splits = p.splits;
        A.sum_rows = sum_here;
        if (p.splits == 1) {
            A.out = dw, A.slope = sum_here ? db : nullptr;
        } else {
            A.slab = (float*)(ws + L.slab), A.row_sum = (float*)(ws + L.row_sum);
            S.slab[0] = A.slab, S.out[0] = dw, S.n[0] = (long long)N * K, S.splits[0] = p.splits, S.blocks = (int)((S.n[0] + 4 * SUM_LANES[0] - 1) / (4 * SUM_LANES[0]));
            if (sum_here) S.slab[1] = A.row_sum, S.out[1] = db, S.n[1] = N, S.splits[1] = p.splits;
        }
        const int rc = launch_product<T, false, false, EPI_SLAB>(A, p.tile, p.tile, st);
        if (rc) return rc;
    }
    const int blocks = S.blocks + (S.out[1] ? (N + 4 * SUM_LANES[1] - 1) / (4 * SUM_LANES[1]) : 0);
    if (blocks) slab_sum_kernel<T><<<blocks, 256, 0, st>>>(S);
    return PCLIP_OK;
}

int check_sizes(const char* who, int M, int K, int N, int dtype, int act) {
    PCLIP_REQUIRE(pclip_dtype_ok(dtype), "%s: unknown type %d", who, dtype);
    PCLIP_REQUIRE(M >= 1 && M <= 0x7fff0000 && K >= 1 && N >= 1 && K <= PCLIP_LINEAR_MAX_DIM && N <= PCLIP_LINEAR_MAX_DIM, "%s: M=%d K=%d N=%d (1 <= M <= 2147418112, 1 <= K, N <= %d)", who, M, K,
                  N, PCLIP_LINEAR_MAX_DIM);
    PCLIP_REQUIRE(act >= PCLIP_ACT_NONE && act <= PCLIP_ACT_SILU, "%s: unknown activation %d", who, act);
    return PCLIP_OK;
}

}  // namespace

extern "C" size_t pclip_linear_fwd_workspace_bytes(int M, int K, int N, int dtype) {
    if (check_sizes("linear_fwd", M, K, N, dtype, 0)) return 0;
    return split_bytes(M, N, K, dtype);
}

extern "C" int pclip_linear_fwd_ws(const void* x, const void* w, const void* bias, const void* residual, int M, int K, int N, int dtype, int activation,
                                   void* y, void* slope, void* ws, size_t ws_bytes, void* stream) {
    int rc = check_sizes("linear_fwd", M, K, N, dtype, activation);
    if (rc) return rc;
    PCLIP_REQUIRE(x && w && y, "linear_fwd: null pointer");
    const size_t need = ws ? split_bytes(M, N, K, dtype) : 0;
    PCLIP_REQUIRE(ws_bytes >= need, "linear_fwd: workspace too small (%zu bytes, need %zu)", ws_bytes, need);
    PCLIP_REQUIRE(((uintptr_t)ws & 15) == 0, "linear_fwd: the workspace must be 16-byte aligned");
    GemmArgs A = {};
    A.P = x, A.Q = w, A.ldp = K, A.ldq = K, A.I = M, A.J = N, A.K = K;
    A.bias = bias, A.residual = residual, A.out = y, A.slope = slope;
    hipStream_t st = (hipStream_t)stream;
    if (dtype == PCLIP_DT_F32) rc = forward<float>(A, activation, (float*)ws, st);
    else if (dtype == PCLIP_DT_BF16) rc = forward<__bf16>(A, activation, nullptr, st);
    else rc = forward<_Float16>(A, activation, nullptr, st);
    return rc ? rc : pclip_check_launch("linear_fwd");
}

extern "C" int pclip_linear_fwd(const void* x, const void* w, const void* bias, const void* residual, int M, int K, int N, int dtype, int activation,
                                void* y, void* slope, void* stream) {
    return pclip_linear_fwd_ws(x, w, bias, residual, M, K, N, dtype, activation, y, slope, nullptr, 0, stream);
}

extern "C" int pclip_linear_tile(int M, int K, int N, int dtype, int product, int aligned) {
    if (check_sizes("linear_tile", M, K, N, dtype, 0)) return 0;
    if (product == 2) return row_plan(M, K, N, dtype, !aligned).tile;
    const int tile = row_tile(M, product ? K : N, dtype);
    return !aligned && tile == 256 ? 128 : tile;   // see launch_size
}

extern "C" size_t pclip_linear_bwd_workspace_bytes(int M, int K, int N, int dtype, int activation) {
    if (check_sizes("linear_bwd", M, K, N, dtype, activation)) return 0;
    size_t most = 0;   // whichever gradients are wanted, at whatever addresses
    for (int k = 0; k < 3; k++) {
        const size_t bytes = backward_layout(M, K, N, dtype, activation, true, k > 0, k == 0, k == 2).bytes;
        if (bytes > most) most = bytes;
    }
    return most;
}

extern "C" int pclip_linear_bwd(const void* x, const void* w, const void* dy, const void* saved, int saved_is_output, int M, int K, int N, int dtype,
                                int activation, void* dx, void* dw, void* db, void* ws, size_t ws_bytes, void* stream) {
    int rc = check_sizes("linear_bwd", M, K, N, dtype, activation);
    if (rc) return rc;
    PCLIP_REQUIRE(dy && (!dx || w) && (!dw || x), "linear_bwd: null pointer");
    PCLIP_REQUIRE(x || !db || !dx || activation != PCLIP_ACT_NONE, "linear_bwd: dx and db of a layer without activation in one call needs x");
    PCLIP_REQUIRE(activation == PCLIP_ACT_NONE || saved, "linear_bwd: what the forward saved is needed");
    PCLIP_REQUIRE(!saved_is_output || activation == PCLIP_ACT_RELU, "linear_bwd: only relu's slope can be read from the output");
    PCLIP_REQUIRE(((uintptr_t)ws & 15) == 0, "linear_bwd: the workspace must be 16-byte aligned");
    hipStream_t st = (hipStream_t)stream;
#define PCLIP_LINEAR_BWD(T)                                                                                                                         backward<T>((const T*)x, (const T*)w, (const T*)dy, saved, saved_is_output, M, K, N, dtype, activation, (T*)dx, (T*)dw, (T*)db, (char*)ws, ws ? ws_bytes : 0, st)
    if (dtype == PCLIP_DT_F32) rc = PCLIP_LINEAR_BWD(float);
    else if (dtype == PCLIP_DT_BF16) rc = PCLIP_LINEAR_BWD(__bf16);
    else rc = PCLIP_LINEAR_BWD(_Float16);
#undef PCLIP_LINEAR_BWD
    return rc ? rc : pclip_check_launch("linear_bwd");
}
