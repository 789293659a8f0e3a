// Global gradient norm over many tensors, and clipping.
//
//   N = sqrt(sum_t sum_i x_ti^2),   out_ti = x_ti * min(1, max_norm / (N + eps))
//
// Two passes over the data are unavoidable (the factor needs every element), so the bound is memory: read twice,
// written once.  The tensors are described by a table, each cut into chunks of CHUNK elements; a workgroup takes a run of
// neighbouring chunks, so it searches the table once.  Up to TENSORS tensors the table travels in the kernels' arguments;
// longer ones are written to the workspace first, TENSORS entries a launch, and each pass is one launch all the
// same (five tables of 120 tensors in turn left the device half empty at every end: 118 -> 77 us for the first pass over
// the 490 tensors of a 30-layer trunk in bf16, 3.9 TB/s; the second, into f32, 192 us, 4.6 TB/s).  Nothing is
// copied from the host, so a captured graph replays it as it stands.
//
// Squares are summed in f64: f32 squares of gradients beyond 1.8e19 would overflow and those below 1e-23 vanish, and
// the conversion and multiply-add cost an eighth of the time the memory needs.  The order of summation is fixed by
// the table alone: the same tensors give the same bits on every call and on every rank.
#include "elem.h"
#include <math.h>

namespace {

constexpr int TENSORS = 120;          // entries of a table in the arguments: 29 bytes each, below the 4 KB of kernel arguments
constexpr int CHUNK = 8192;           // elements of one chunk: 256 threads, 16 bytes each, 4 (16-bit) or 8 (f32) times
constexpr int MAX_BLOCKS = 2048;      // workgroups of a launch, eight a compute unit
constexpr int SELF_SUM = 256;         // up to this many partial sums every workgroup of the second pass adds them itself
constexpr int THREADS = 256;

struct Entry {
    const void* src;
    void* dst;
    long long numel;
    int type;                         // source type | destination type << 4
};
// a table in the kernel's arguments
struct ClipTable {
    const void* src[TENSORS];
    void* dst[TENSORS];
    long long numel[TENSORS];
    unsigned first[TENSORS];          // first chunk of the tensor
    unsigned char type[TENSORS];
    int n;
    unsigned chunks;
    __device__ __forceinline__ unsigned first_of(int t) const { return first[t]; }
    __device__ __forceinline__ Entry entry(int t) const { return {src[t], dst[t], numel[t], type[t]}; }
};
static_assert(sizeof(ClipTable) <= 4000, "kernel arguments");
// a table in the workspace
struct ClipTableView {
    Entry* entries;
    unsigned* first;
    int n;
    unsigned chunks;
    __device__ __forceinline__ unsigned first_of(int t) const { return first[t]; }
    __device__ __forceinline__ Entry entry(int t) const { return entries[t]; }
};

__global__ __launch_bounds__(128) void table_kernel(const ClipTable part, ClipTableView view, int at, unsigned first_chunk) {
    const int t = threadIdx.x;
    if (t >= part.n) return;
    view.entries[at + t] = part.entry(t);
    view.first[at + t] = first_chunk + part.first[t];
}

// tensor that holds chunk c (the last one whose first chunk is not behind c; every tensor has a chunk): 64 places compared at once
template <typename Table>
__device__ __forceinline__ int tensor_of(const Table& tab, unsigned c) {
    const int lane = threadIdx.x & 63;
    int lo = 0, len = tab.n;
    while (len > 1) {
        const int step = (len + 63) >> 6, at = lane * step;
        const int k = __popcll(__ballot(at < len && tab.first_of(lo + (at < len ? at : 0)) <= c)) - 1;   // the first is never behind c
        lo += k * step;
        len = min(step, len - k * step);
    }
    return __builtin_amdgcn_readfirstlane(lo);
}
// calls work(entry, offset, length) for the workgroup's run of chunks; `backwards`: from the last to the first
template <typename Table, typename Work>
__device__ __forceinline__ void for_chunks(const Table& tab, bool backwards, Work work) {
    const unsigned per = (tab.chunks + gridDim.x - 1) / gridDim.x, b = backwards ? gridDim.x - 1 - blockIdx.x : blockIdx.x;
    const unsigned begin = min(b * per, tab.chunks), end = min(begin + per, tab.chunks);
    if (begin == end) return;
    int t = tensor_of(tab, begin);
    Entry e = tab.entry(t);
    unsigned first = tab.first_of(t);
    for (unsigned c = begin; c < end; c++) {
        while (t + 1 < tab.n && tab.first_of(t + 1) <= c) {
            e = tab.entry(++t);
            first = tab.first_of(t);
        }
        const long long off = (long long)(c - first) * CHUNK, left = e.numel - off;
        work(e, off, left < CHUNK ? (int)left : CHUNK);
    }
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

template <typename Table>
__global__ __launch_bounds__(THREADS) void grad_squares_kernel(const Table tab, double* __restrict__ partial) {
    __shared__ double lds[4];
    double s0 = 0.0, s1 = 0.0;
    for_chunks(tab, false, [&](const Entry& e, long long off, int len) {
        const int type = e.type & 15;
        if (type == PCLIP_DT_F32) chunk_squares((const float*)e.src + off, len, s0, s1);
        else if (type == PCLIP_DT_BF16) chunk_squares((const __bf16*)e.src + off, len, s0, s1);
        else chunk_squares((const _Float16*)e.src + off, len, s0, s1);
    });
    const double s = block_sum(s0 + s1, lds);
    if (threadIdx.x == 0) partial[blockIdx.x] = s;
}

__global__ __launch_bounds__(THREADS) void grad_norm_kernel(const double* __restrict__ partial, int n, float* __restrict__ norm) {
    __shared__ double lds[4];
    double s = 0.0;
#pragma unroll 8
    for (int i = threadIdx.x; i < n; i += THREADS) s += partial[i];
    s = block_sum(s, lds);
    if (threadIdx.x == 0) *norm = (float)sqrt(s);
}

template <typename S, typename D>
__device__ __forceinline__ void chunk_scale(const S* p, D* q, int len, float factor) {
    constexpr int V = sizeof(S) == 2 && sizeof(D) == 2 ? 8 : 4;   // at most 16 bytes each way, so that lines are written whole
#pragma unroll 4
    for (int i = threadIdx.x * V; i < len; i += THREADS * V) {
        float x[V];
        load_f32<S, V>(p + i, len - i, x);
#pragma unroll
        for (int k = 0; k < V; k++) x[k] *= factor;
        stream_f32<D, V>(q + i, len - i, x);
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
// first: what the first pass read last is still in the 256 MB last-level cache.  Results go past the L2.
template <typename Table>
__global__ __launch_bounds__(THREADS) void grad_scale_kernel(const Table tab, const double* __restrict__ partial, int n_partial, float max_norm, float eps,
                                                             float* norm) {
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
    for_chunks(tab, true, [&](const Entry& e, long long off, int len) {
        if (factor == 1.f && e.src == e.dst) return;   // in place, not clipped: x * 1 is x
        const int from = e.type & 15, to = e.type >> 4;
        if (from == PCLIP_DT_F32) chunk_scale_to((const float*)e.src + off, e.dst, off, to, len, factor);
        else if (from == PCLIP_DT_BF16) chunk_scale_to((const __bf16*)e.src + off, e.dst, off, to, len, factor);
        else chunk_scale_to((const _Float16*)e.src + off, e.dst, off, to, len, factor);
    });
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

size_t partial_bytes() { return MAX_BLOCKS * sizeof(double); }

// both passes over one table
template <typename Table>
void run(const Table& tab, bool scale, float max_norm, float eps, float* norm, double* partial, hipStream_t st) {
    const unsigned per = (tab.chunks + MAX_BLOCKS - 1) / MAX_BLOCKS;
    const int grid = (int)((tab.chunks + per - 1) / per);
    grad_squares_kernel<<<grid, THREADS, 0, st>>>(tab, partial);
    const bool self = scale && grid <= SELF_SUM;
    if (!self) grad_norm_kernel<<<1, THREADS, 0, st>>>(partial, grid, norm);
    if (scale) grad_scale_kernel<<<grid, THREADS, 0, st>>>(tab, partial, self ? grid : 0, max_norm, eps, norm);
}

}  // namespace

extern "C" size_t pclip_grad_clip_workspace_bytes(int n) {
    if (n < 1) return 0;
    return partial_bytes() + (n > TENSORS ? (size_t)n * (sizeof(Entry) + sizeof(unsigned)) : 0);
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
    PCLIP_REQUIRE(((uintptr_t)ws & 7) == 0, "grad_clip: the workspace must be 8-byte aligned");
    hipStream_t st = (hipStream_t)stream;
    double* partial = (double*)ws;
    ClipTable tab;
    int at = 0;
    if (!fill_table(tab, at, n, src, numel, src_type, dst, dst_type)) {   // no elements at all
        grad_norm_kernel<<<1, THREADS, 0, st>>>(partial, 0, norm);
    } else if (at == n) {
        run(tab, dst != nullptr, max_norm, eps, norm, partial, st);
    } else {
        ClipTableView view = {};
        view.entries = (Entry*)((char*)ws + partial_bytes());
        view.first = (unsigned*)(view.entries + n);
        do {
            table_kernel<<<1, 128, 0, st>>>(tab, view, view.n, view.chunks);
            view.n += tab.n;
            view.chunks += tab.chunks;
        } while (fill_table(tab, at, n, src, numel, src_type, dst, dst_type));
        run(view, dst != nullptr, max_norm, eps, norm, partial, st);
    }
    return pclip_check_launch("grad_clip");
}
