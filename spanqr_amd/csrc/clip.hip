// clip.hip -- the norm over many tensors and their clipped copies.
//
//   norm = sqrt(sum over all tensors of g^2),  out = g min(1, max_norm / norm)
//
// Bound by memory: the gradients are read once for the norm and once more for the copies (from the memory-side cache
// where they fit its 256 MB; the second pass runs backwards, so that it begins with what was read last). Two launches
// for each TABLE tensors: the tensors' addresses travel in the kernel's arguments, so there is no table to upload and a
// captured graph keeps them. Work is cut into CHUNK elements, whatever tensor they are of; a workgroup takes every
// gridDim-th chunk and leaves one partial sum, and with one table every workgroup of the second pass adds all partial
// sums itself, in the same order, instead of waiting for a third launch. Squares are added in fp64: no order of additions
// matters to the fp32 result's rounding, and gradients whose squares leave fp32's range keep their norm.
// 470 million bf16 gradients into fp32: the squares in 160 us (5.8 TB/s, part of it from the cache), the copies in 470
// (6.0 TB/s), 636 together; what has to move, read once and written once, would take 588 at a copy's 4.8 TB/s.
#include "elements.h"
#include "host.h"

using namespace spanqr_dev;
using spanqr_host::error;
using spanqr_host::launched;

namespace {

constexpr int TABLE = 112;          // tensors a launch (its arguments stay below 4 KB)
constexpr int THREADS = 256;
constexpr int CHUNK = THREADS * 32; // elements
constexpr int MAX_PARTS = 4096;     // partial sums of a table

struct Table {
    const void* src[TABLE];
    void* dst[TABLE];
    unsigned long n[TABLE];         // elements
    uint32_t first[TABLE + 1];      // the tensor's first chunk; [count] their number
    uint8_t type[TABLE], out[TABLE];
    int count;
};

// the tensor of a chunk
__device__ __forceinline__ int tensor_of(const Table& t, uint32_t chunk) {
    int lo = 0, hi = t.count;       // first[lo] <= chunk < first[hi]
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (t.first[mid] <= chunk)
            lo = mid;
        else
            hi = mid;
    }
    return lo;
}

// W neighbouring elements at the element's own alignment. A wavefront's access has no gaps if it is 16 bytes a lane at
// most: 4 elements where fp32 is read or written, else 8.
template <typename T, int W>
struct Vector {
    typedef T type __attribute__((ext_vector_type(W), aligned(sizeof(T))));
};

template <typename T>
__device__ __forceinline__ double squares(const T* p, unsigned long n, unsigned long at) {
    double sum = 0.0;
    if (n - at >= CHUNK) {   // all loads at once
        constexpr int W = 16 / sizeof(T), PIECES = CHUNK / THREADS / W;
        typedef typename Vector<T, W>::type V;
        V k[PIECES];
#pragma unroll
        for (int c = 0; c < PIECES; ++c) k[c] = *(const V*)(p + at + (unsigned long)W * (threadIdx.x + c * THREADS));
#pragma unroll
        for (int c = 0; c < PIECES; ++c)
#pragma unroll
            for (int i = 0; i < W; ++i) sum = fma((double)(float)k[c][i], (double)(float)k[c][i], sum);
        return sum;
    }
    for (unsigned long i = at + 8ul * threadIdx.x; i < n; i += 8ul * THREADS) {
        float f[8];
        load8(p + i, n - i >= 8 ? 8 : (int)(n - i), f);
#pragma unroll
        for (int k = 0; k < 8; ++k) sum = fma((double)f[k], (double)f[k], sum);
    }
    return sum;
}

__global__ __launch_bounds__(THREADS) void k_squares(const Table t, double* part) {
    __shared__ double slot[THREADS / 64];
    double sum = 0.0;
    for (uint32_t chunk = blockIdx.x; chunk < t.first[t.count]; chunk += gridDim.x) {
        const int i = tensor_of(t, chunk);
        const unsigned long at = (unsigned long)(chunk - t.first[i]) * CHUNK;
        if (t.type[i] == SPANQR_BF16)
            sum += squares((const bf16*)t.src[i], t.n[i], at);
        else if (t.type[i] == SPANQR_FP16)
            sum += squares((const fp16*)t.src[i], t.n[i], at);
        else
            sum += squares((const float*)t.src[i], t.n[i], at);
    }
    sum = reduce_threads<THREADS, Sum>(sum, slot);
    if (threadIdx.x == 0) part[blockIdx.x] = sum;
}

// the norm from the partial sums, the same in every workgroup that computes it
__device__ __forceinline__ double norm_of(const double* part, int parts) {
    __shared__ double slot[THREADS / 64];
    double sum = 0.0;
    int i = threadIdx.x;
    for (; i + 7 * THREADS < parts; i += 8 * THREADS) {   // (eight loads together)
        double v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = part[i + k * THREADS];
#pragma unroll
        for (int k = 0; k < 8; ++k) sum += v[k];
    }
    for (; i < parts; i += THREADS) sum += part[i];
    return sqrt(reduce_threads<THREADS, Sum>(sum, slot));
}

// square (or null): the squared norm, as the one partial sum of the second pass
__global__ __launch_bounds__(THREADS) void k_norm(const double* part, int parts, float* norm, double* square) {
    const double v = norm_of(part, parts);
    if (threadIdx.x == 0) {
        *norm = (float)v;
        if (square != nullptr) *square = v * v;
    }
}

template <bool STREAM, typename T, typename O>
__device__ __forceinline__ void scaled(const T* p, O* out, unsigned long n, unsigned long at, float f) {
    if (n - at >= CHUNK) {
        constexpr int W = sizeof(T) == 4 || sizeof(O) == 4 ? 4 : 8, PIECES = CHUNK / THREADS / W;
        typedef typename Vector<T, W>::type V;
        typedef typename Vector<O, W>::type X;
        V k[PIECES];
#pragma unroll
        for (int c = 0; c < PIECES; ++c) {
            const V* from = (const V*)(p + at + (unsigned long)W * (threadIdx.x + c * THREADS));
            k[c] = STREAM ? __builtin_nontemporal_load(from) : *from;
        }
#pragma unroll
        for (int c = 0; c < PIECES; ++c) {
            X v;
#pragma unroll
            for (int i = 0; i < W; ++i) v[i] = (O)((float)k[c][i] * f);
            X* to = (X*)(out + at + (unsigned long)W * (threadIdx.x + c * THREADS));
            if (STREAM)
                __builtin_nontemporal_store(v, to);
            else
                *to = v;
        }
        return;
    }
    float v[8];
    for (unsigned long i = at + 8ul * threadIdx.x; i < n; i += 8ul * THREADS) {
        const int k = n - i >= 8 ? 8 : (int)(n - i);
        load8(p + i, k, v);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] *= f;
        store8(out + i, k, v);
    }
}

template <bool STREAM, typename T>
__device__ __forceinline__ void scaled_to(const T* p, void* out, int type, unsigned long n, unsigned long at, float f) {
    if (type == SPANQR_BF16)
        scaled<STREAM>(p, (bf16*)out, n, at, f);
    else if (type == SPANQR_FP16)
        scaled<STREAM>(p, (fp16*)out, n, at, f);
    else
        scaled<STREAM>(p, (float*)out, n, at, f);
}

// STREAM: past the caches
template <bool STREAM>
__global__ __launch_bounds__(THREADS) void k_clip(const Table t, const double* part, int parts, float max_norm,
                                                  float* norm) {
    const double v = norm_of(part, parts);
    if (norm != nullptr && blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)v;
    // NaN stays NaN; an infinite norm gives 0 (and NaN where the element is infinite)
    const float f = v <= (double)max_norm ? 1.0f : (float)((double)max_norm / v);
    const uint32_t chunks = t.first[t.count];
    for (uint32_t k = blockIdx.x; k < chunks; k += gridDim.x) {
        const uint32_t chunk = chunks - 1 - k;
        const int i = tensor_of(t, chunk);
        if (f == 1.0f && t.src[i] == t.dst[i]) continue;   // in place and within the bound: nothing changes
        const unsigned long at = (unsigned long)(chunk - t.first[i]) * CHUNK;
        if (t.type[i] == SPANQR_BF16)
            scaled_to<STREAM>((const bf16*)t.src[i], t.dst[i], t.out[i], t.n[i], at, f);
        else if (t.type[i] == SPANQR_FP16)
            scaled_to<STREAM>((const fp16*)t.src[i], t.dst[i], t.out[i], t.n[i], at, f);
        else
            scaled_to<STREAM>((const float*)t.src[i], t.dst[i], t.out[i], t.n[i], at, f);
    }
}

unsigned at_most(uint32_t chunks, unsigned most) { return chunks < most ? chunks : most; }

// What passes through the memory-side cache (256 MB) finds nothing there afterwards: then the second pass leaves the
// cache to the gradients it has still to read. In us for both passes, past the caches and otherwise: 940 MB of bf16
// gradients and their fp32 copies (three tables) 636 and 700, 46 MB of fp32 gradients and their copies 40 and 38.
constexpr unsigned long CACHE = 256ul << 20;

unsigned long chunks_of(unsigned long n) { return (n + CHUNK - 1) / CHUNK; }

// Fills the next table from tensor `i` on (empty tensors left out); returns the next tensor
int fill(Table& t, int i, int n, const void* const* src, void* const* dst, const long* numel, const int* type,
         const int* out) {
    t.count = 0;
    t.first[0] = 0;
    for (; i < n && t.count < TABLE; ++i) {
        if (numel[i] == 0) continue;
        const unsigned long end = t.first[t.count] + chunks_of((unsigned long)numel[i]);
        if (end >= 1ul << 31) break;   // chunks of a table are counted in 32 bits
        const int k = t.count++;
        t.src[k] = src[i];
        t.dst[k] = dst == nullptr ? nullptr : dst[i];
        t.n[k] = (unsigned long)numel[i];
        t.type[k] = (uint8_t)type[i];
        t.out[k] = (uint8_t)(out == nullptr ? type[i] : out[i]);
        t.first[k + 1] = (uint32_t)end;
    }
    return i;
}

int check(const char* what, int n, const long* numel) {
    if (n < 0 || (n > 0 && numel == nullptr)) return error(SPANQR_EINVAL, "%s: bad arguments", what);
    for (int i = 0; i < n; ++i)
        if (numel[i] < 0 || numel[i] > 1l << 42) return error(SPANQR_EINVAL, "%s: tensor %d has %ld elements", what, i, numel[i]);
    return SPANQR_OK;
}

bool known(int type) { return type == SPANQR_BF16 || type == SPANQR_FP16 || type == SPANQR_FP32; }

// for any tables that fill() makes of n tensors
long workspace_of(int n) { return 8l * MAX_PARTS * (n / TABLE + 1) + 8; }

int enqueue(const char* what, int n, const void* const* src, const long* numel, const int* type, void* const* dst,
            const int* out, float max_norm, float* norm, void* workspace, long workspace_bytes, hipStream_t st) {
    const int rc = check(what, n, numel);
    if (rc != SPANQR_OK) return rc;
    if (norm == nullptr || workspace == nullptr || (n > 0 && (src == nullptr || type == nullptr)))
        return error(SPANQR_EINVAL, "%s: a missing pointer", what);
    if (workspace_bytes < workspace_of(n)) return error(SPANQR_EINVAL, "%s: the workspace needs %ld bytes", what, workspace_of(n));
    for (int i = 0; i < n; ++i) {
        if (!known(type[i]) || (out != nullptr && !known(out[i]))) return error(SPANQR_EINVAL, "%s: tensor %d: unknown type", what, i);
        if (numel[i] > 0 && (src[i] == nullptr || (dst != nullptr && dst[i] == nullptr)))
            return error(SPANQR_EINVAL, "%s: tensor %d: a missing pointer", what, i);
    }
    double *square = (double*)workspace, *part = square + 1;
    int parts = 0, tables = 0;
    unsigned long bytes = 0;
    Table t;
    for (int i = 0; i < n;) {
        i = fill(t, i, n, src, dst, numel, type, out);
        if (t.count == 0) break;
        for (int k = 0; k < t.count; ++k) bytes += t.n[k] * (t.type[k] == SPANQR_FP32 ? 4 : 2);
        const unsigned grid = at_most(t.first[t.count], MAX_PARTS);
        k_squares<<<grid, THREADS, 0, st>>>(t, part + parts);
        parts += (int)grid;
        ++tables;
    }
    if (dst == nullptr || tables != 1) {
        k_norm<<<1, THREADS, 0, st>>>(part, parts, norm, square);
        if (dst == nullptr || parts == 0) return launched(what);
        part = square, parts = 1, norm = nullptr;
    }
    for (int i = 0; i < n;) {
        const bool first = i == 0;
        i = fill(t, i, n, src, dst, numel, type, out);
        if (t.count == 0) break;
        // (with many partial sums to add in each, fewer workgroups)
        const unsigned grid = at_most(t.first[t.count], parts > 1 ? 2048 : 8192);
        if (bytes > CACHE)
            k_clip<true><<<grid, THREADS, 0, st>>>(t, part, parts, max_norm, first ? norm : nullptr);
        else
            k_clip<false><<<grid, THREADS, 0, st>>>(t, part, parts, max_norm, first ? norm : nullptr);
    }
    return launched(what);
}

}  // namespace

extern "C" {

long spanqr_grad_norm_workspace(int n) {
    return n < 0 ? error(SPANQR_EINVAL, "grad_norm: n = %d", n) : workspace_of(n);
}

int spanqr_grad_norm(int n, const void* const* grads, const long* numel, const int* type, float* norm, void* workspace,
                     long workspace_bytes, void* stream) {
    return enqueue("grad_norm", n, grads, numel, type, nullptr, nullptr, 0.0f, norm, workspace, workspace_bytes,
                   (hipStream_t)stream);
}

int spanqr_clip_grad_norm(int n, const void* const* grads, const long* numel, const int* type, void* const* out,
                          const int* out_type, float max_norm, float* norm, void* workspace, long workspace_bytes,
                          void* stream) {
    if (n > 0 && (out == nullptr || out_type == nullptr)) return error(SPANQR_EINVAL, "clip_grad_norm: a missing pointer");
    if (!(max_norm >= 0.0f)) return error(SPANQR_EINVAL, "clip_grad_norm: max_norm = %g", (double)max_norm);
    return enqueue("clip_grad_norm", n, grads, numel, type, n > 0 ? out : nullptr, out_type, max_norm, norm, workspace,
                   workspace_bytes, (hipStream_t)stream);
}

}  // extern "C"
