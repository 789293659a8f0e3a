// Global gradient norm over many tensors, and clipping.
//
//   N = sqrt(sum_t sum_i x_ti^2),   out_ti = x_ti * min(1, max_norm / (N + eps))
//
// Two passes over the data are unavoidable (the factor needs every element), so the bound is memory: read twice,
// written once.  The tensors travel as a table in the kernel's arguments, TENSORS of them a launch, each cut into
// chunks of CHUNK elements that the workgroups take in turn; a call on a hundred tensors is one launch a pass, and
// nothing is copied to the device, so a captured graph replays it as it stands.
//
// Squares are summed in f64: f32 squares of gradients beyond 1.8e19 would overflow and those below 1e-23 vanish, and
// the conversion and multiply-add cost an eighth of the time the memory needs.  The order of summation is fixed by
// the table alone: the same tensors give the same bits on every call and on every rank.
#include "elem.h"
#include <math.h>

namespace {

constexpr int TENSORS = 120;          // entries of one launch's table: 29 bytes each, below the 4 KB of kernel arguments
constexpr int CHUNK = 8192;           // elements of one chunk: 256 threads, 16 bytes each, 4 (16-bit) or 8 (f32) times
constexpr int MAX_BLOCKS = 2048;      // workgroups of a launch, eight a compute unit
constexpr int SELF_SUM = 256;         // up to this many partial sums every workgroup of the second pass adds them itself
constexpr int THREADS = 256;

struct ClipTable {
    const void* src[TENSORS];
    void* dst[TENSORS];
    long long numel[TENSORS];
    unsigned first[TENSORS];          // first chunk of the tensor
    unsigned char type[TENSORS];      // source type | destination type << 4
    int n;
    unsigned chunks;
};
static_assert(sizeof(ClipTable) <= 4000, "kernel arguments");

// tensor that holds chunk c (the last one whose first chunk is not behind c; every tensor has a chunk)
__device__ __forceinline__ int tensor_of(const ClipTable& tab, unsigned c) {
    int lo = 0, hi = tab.n - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (tab.first[mid] <= c) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

__device__ __forceinline__ double block_sum(double v, double* lds) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    const double s = (lds[0] + lds[1]) + (lds[2] + lds[3]);
    __syncthreads();
    return s;
}

template <typename T>
__device__ __forceinline__ void chunk_squares(const T* p, int len, double& s0, double& s1) {
    constexpr int V = PclipVec<T>::N;
#pragma unroll 4
    for (int i = threadIdx.x * V; i < len; i += THREADS * V) {
        float x[V];
        load_f32<T, V>(p + i, len - i, x);
#pragma unroll
        for (int k = 0; k < V; k += 2) {
            s0 = fma((double)x[k], (double)x[k], s0);
            s1 = fma((double)x[k + 1], (double)x[k + 1], s1);
        }
    }
}

__global__ __launch_bounds__(THREADS) void grad_squares_kernel(const ClipTable tab, double* __restrict__ partial) {
    __shared__ double lds[4];
    double s0 = 0.0, s1 = 0.0;
    for (unsigned c = blockIdx.x; c < tab.chunks; c += gridDim.x) {
        const int t = tensor_of(tab, c);
        const long long off = (long long)(c - tab.first[t]) * CHUNK, left = tab.numel[t] - off;
        const int len = left < CHUNK ? (int)left : CHUNK, type = tab.type[t] & 15;
        if (type == PCLIP_DT_F32) chunk_squares((const float*)tab.src[t] + off, len, s0, s1);
        else if (type == PCLIP_DT_BF16) chunk_squares((const __bf16*)tab.src[t] + off, len, s0, s1);
        else chunk_squares((const _Float16*)tab.src[t] + off, len, s0, s1);
    }
    const double s = block_sum(s0 + s1, lds);
    if (threadIdx.x == 0) partial[blockIdx.x] = s;
}

__global__ __launch_bounds__(THREADS) void grad_norm_kernel(const double* __restrict__ partial, int n, float* __restrict__ norm) {
    __shared__ double lds[4];
    double s = 0.0;
    for (int i = threadIdx.x; i < n; i += THREADS) s += partial[i];
    s = block_sum(s, lds);
    if (threadIdx.x == 0) *norm = (float)sqrt(s);
}

template <typename S, typename D>
__device__ __forceinline__ void chunk_scale(const S* p, D* q, int len, float factor) {
    constexpr int V = sizeof(S) == 2 && sizeof(D) == 2 ? 8 : 4;
#pragma unroll 4
    for (int i = threadIdx.x * V; i < len; i += THREADS * V) {
        float x[V];
        load_f32<S, V>(p + i, len - i, x);
#pragma unroll
        for (int k = 0; k < V; k++) x[k] *= factor;
        store_f32<D, V>(q + i, len - i, x);
    }
}
template <typename S>
__device__ __forceinline__ void chunk_scale_to(const S* p, void* dst, long long off, int type, int len, float factor) {
    if (type == PCLIP_DT_F32) chunk_scale(p, (float*)dst + off, len, factor);
    else if (type == PCLIP_DT_BF16) chunk_scale(p, (__bf16*)dst + off, len, factor);
    else chunk_scale(p, (_Float16*)dst + off, len, factor);
}

// Second pass.  n_partial <= SELF_SUM: the partial sums are added here, by every workgroup in the same order (no launch
// between the passes); otherwise n_partial is 0 and *norm holds the norm.  The chunks are taken from the last to the
// first: what the first pass read last is still in the 256 MB last-level cache.
__global__ __launch_bounds__(THREADS) void grad_scale_kernel(const ClipTable tab, const double* __restrict__ partial, int n_partial, float max_norm,
                                                             float eps, float* norm) {
    __shared__ double lds[4];
    float total;
    if (n_partial > 0) {
        total = (float)sqrt(block_sum((int)threadIdx.x < n_partial ? partial[threadIdx.x] : 0.0, lds));
        if (blockIdx.x == 0 && threadIdx.x == 0) *norm = total;
    } else {
        total = *norm;
    }
    const float ratio = max_norm / (total + eps);
    const float factor = ratio >= 1.f ? 1.f : ratio;   // NaN stays NaN
    for (unsigned k = blockIdx.x; k < tab.chunks; k += gridDim.x) {
        const unsigned c = tab.chunks - 1 - k;
        const int t = tensor_of(tab, c);
        if (factor == 1.f && tab.src[t] == tab.dst[t]) continue;   // in place, not clipped: x * 1 is x
        const long long off = (long long)(c - tab.first[t]) * CHUNK, left = tab.numel[t] - off;
        const int len = left < CHUNK ? (int)left : CHUNK, from = tab.type[t] & 15, to = tab.type[t] >> 4;
        if (from == PCLIP_DT_F32) chunk_scale_to((const float*)tab.src[t] + off, tab.dst[t], off, to, len, factor);
        else if (from == PCLIP_DT_BF16) chunk_scale_to((const __bf16*)tab.src[t] + off, tab.dst[t], off, to, len, factor);
        else chunk_scale_to((const _Float16*)tab.src[t] + off, tab.dst[t], off, to, len, factor);
    }
}

// The next launch's table, from tensor `at` on; false when no tensor with elements is left.
bool fill_table(ClipTable& tab, int& at, int n, const void* const* src, const int64_t* numel, const int* src_type, void* const* dst,
                const int* dst_type) {
    tab.n = 0;
    tab.chunks = 0;
    for (; at < n && tab.n < TENSORS; at++) {
        if (numel[at] == 0) continue;
        const int k = tab.n++;
        tab.src[k] = src[at];
        tab.dst[k] = dst ? dst[at] : nullptr;
        tab.numel[k] = numel[at];
        tab.first[k] = tab.chunks;
        tab.type[k] = (unsigned char)(src_type[at] | ((dst ? dst_type[at] : 0) << 4));
        tab.chunks += (unsigned)((numel[at] + CHUNK - 1) / CHUNK);
    }
    return tab.n > 0;
}

int launches_of(int n) { return (n + TENSORS - 1) / TENSORS; }

}  // namespace

extern "C" size_t pclip_grad_clip_workspace_bytes(int n) {
    if (n < 1) return 0;
    return (size_t)launches_of(n) * MAX_BLOCKS * sizeof(double);
}

extern "C" int pclip_grad_clip(const void* const* src, const int64_t* numel, const int* src_type, void* const* dst, const int* dst_type, int n,
                               float max_norm, float eps, float* norm, void* ws, size_t ws_bytes, void* stream) {
    PCLIP_REQUIRE(src && numel && src_type && norm && ws && (!dst || dst_type), "grad_clip: null pointer");
    PCLIP_REQUIRE(n >= 1 && n <= (1 << 20), "grad_clip: n=%d tensors (1 to 1048576)", n);
    PCLIP_REQUIRE(!dst || max_norm >= 0.f, "grad_clip: max_norm must be zero or more");
    PCLIP_REQUIRE(!dst || (eps >= 0.f && eps < INFINITY), "grad_clip: eps must be zero or more and finite");
    PCLIP_REQUIRE(ws_bytes >= pclip_grad_clip_workspace_bytes(n), "grad_clip: workspace too small (%zu bytes)", ws_bytes);
    long long total = 0;
    for (int i = 0; i < n; i++) {
        PCLIP_REQUIRE(numel[i] >= 0 && numel[i] <= (1ll << 42), "grad_clip: tensor %d has %lld elements", i, (long long)numel[i]);
        PCLIP_REQUIRE(pclip_dtype_ok(src_type[i]) && (!dst || pclip_dtype_ok(dst_type[i])), "grad_clip: tensor %d has an unknown type", i);
        PCLIP_REQUIRE(numel[i] == 0 || (src[i] && (!dst || dst[i])), "grad_clip: tensor %d: null pointer", i);
        PCLIP_REQUIRE(!dst || numel[i] == 0 || src[i] != dst[i] || src_type[i] == dst_type[i], "grad_clip: tensor %d: in place with two types", i);
        total += numel[i];
        PCLIP_REQUIRE(total <= (1ll << 43), "grad_clip: more than 2^43 elements in one call");   // chunk numbers have 31 bits
    }
    hipStream_t st = (hipStream_t)stream;
    double* partial = (double*)ws;
    ClipTable tab;
    int at = 0, sums = 0;
    while (fill_table(tab, at, n, src, numel, src_type, dst, dst_type)) {
        const int grid = tab.chunks < (unsigned)MAX_BLOCKS ? (int)tab.chunks : MAX_BLOCKS;
        grad_squares_kernel<<<grid, THREADS, 0, st>>>(tab, partial + sums);
        sums += grid;
    }
    const bool self = dst && sums > 0 && sums <= SELF_SUM;
    if (!self) grad_norm_kernel<<<1, THREADS, 0, st>>>(partial, sums, norm);
    if (dst) {
        at = 0;
        while (fill_table(tab, at, n, src, numel, src_type, dst, dst_type)) {
            const int grid = tab.chunks < (unsigned)MAX_BLOCKS ? (int)tab.chunks : MAX_BLOCKS;
            grad_scale_kernel<<<grid, THREADS, 0, st>>>(tab, partial, self ? sums : 0, max_norm, eps, norm);
        }
    }
    return pclip_check_launch("grad_clip");
}
