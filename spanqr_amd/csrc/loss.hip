// loss.hip -- softmax cross entropy over a large vocabulary from the hidden states and the head's weights, without
// keeping the logits, and its gradients.
//
//   z = x W^T [N, V],  lse_i = log sum_j exp z_ij,  loss_i = w_i (lse_i - z_i,t_i)      (w_i = 0 where t_i is ignored)
//   G_ij = w_i (exp(z_ij - lse_i) - [j = t_i]),  dx = a G W,  dW = a G^T x      (a = 1, or 1 / tokens that count)
//
// Three products of 2 N H V operations each. The product of the logits ends in its own softmax statistics: for SEG
// neighbouring columns of a token it leaves the maximum m and the sum of exp(z - m), and, where gradients are wanted,
// the exponentials p = exp(z - m) themselves, rounded to the 16-bit type once. One pass over p turns them into G
// (times exp(m - lse), the target's element from its fp32 logit), and G goes into the other two products. So nothing
// is multiplied twice, and what is held is 16 bits an element for as many tokens at a time as the workspace takes.
#include "elements.h"
#include "host.h"

using namespace spanqr_dev;
using spanqr_host::error;
using spanqr_host::launched;

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 fp16x8 __attribute__((ext_vector_type(8)));

constexpr float LOG2E = 1.44269504088896340736f;

__device__ __forceinline__ float exp_of(float x) { return __builtin_amdgcn_exp2f(x * LOG2E); }

template <typename T>
struct Vec;
template <>
struct Vec<bf16> {
    typedef bf16x8 x8;
    __device__ __forceinline__ static f32x4 mfma(x8 a, x8 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    }
};
template <>
struct Vec<fp16> {
    typedef fp16x8 x8;
    __device__ __forceinline__ static f32x4 mfma(x8 a, x8 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
    }
};

constexpr int SEG = 32;          // columns that share a maximum

// G is held in 16 bits; half precision has it times 2^10, so that probabilities down to 2^-34 stay normal or at least
// count (bf16 has fp32's exponents)
template <typename T>
constexpr float g_scale() { return sizeof(T) == 2 && std::is_same<T, fp16>::value ? 1024.0f : 1.0f; }

// C[n][m] = sum over k of A(m, k) B(n, k), for the three products:
//   logits  m = vocabulary (A = W rows),    n = token (B = x rows),   k = hidden
//   dx      m = hidden     (A = W columns), n = token (B = G rows),   k = vocabulary
//   dW      m = hidden     (A = x columns), n = vocabulary (B = G columns), k = token
// With m along the matrix instruction's rows a lane holds neighbouring elements of one row of C.
struct ProductArgs {
    long M, N, K;
    const void *A, *B;
    long lda, ldb;               // elements between rows as they lie in memory
    // logits
    const long* target;          // of token 0 of this piece
    float* zt;                   // the target's logit
    float2* stat;                // [token][segs]: maximum, sum
    long segs;
    void* p;                     // exponentials [token][ldp], or null
    long ldp;
    // dx, dW
    void* C;
    long ldc;
    float* acc;                  // dW over several pieces of the tokens: fp32 sums [N][M], or null
    int add, last;               // add to acc; the last piece writes C
    const float* alpha;
};

enum { LOGITS, OUT };

template <typename T, bool A_ROWS, bool B_ROWS, int EPILOGUE>
__global__ __launch_bounds__(256) void k_product(const ProductArgs q) {
    typedef typename Vec<T>::x8 x8;
    constexpr int LD = 40;
    __shared__ __attribute__((aligned(16))) T As[64 * LD], Bs[64 * LD];
    const long m0 = 64l * blockIdx.x, n0 = 64l * blockIdx.y;
    const int t = threadIdx.x, wave = t >> 6, lane = t & 63, lo = lane & 15, hi = lane >> 4;
    const int wm = 32 * (wave & 1), wn = 32 * (wave >> 1);
    f32x4 c[2][2] = {};
    auto stage = [&](T* S, const T* src, long ld, long rows, long r0, long k0, bool by_rows) {
        if (by_rows) {
            const long r = r0 + (t >> 2), k = k0 + 8 * (t & 3);
            const int n = r >= rows || k >= q.K ? 0 : q.K - k >= 8 ? 8 : (int)(q.K - k);
            for (int i = 0; i < 8; ++i) S[(t >> 2) * LD + 8 * (t & 3) + i] = i < n ? src[r * ld + k + i] : (T)0.0f;
        } else {
            const long k = k0 + (t >> 3), r = r0 + 8 * (t & 7);
            const int n = k >= q.K || r >= rows ? 0 : rows - r >= 8 ? 8 : (int)(rows - r);
            for (int i = 0; i < 8; ++i) S[(8 * (t & 7) + i) * LD + (t >> 3)] = i < n ? src[k * ld + r + i] : (T)0.0f;
        }
    };
    for (long k0 = 0; k0 < q.K; k0 += 32) {
        stage(As, (const T*)q.A, q.lda, q.M, m0, k0, A_ROWS);
        stage(Bs, (const T*)q.B, q.ldb, q.N, n0, k0, B_ROWS);
        __syncthreads();
        x8 a[2], b[2];
        for (int i = 0; i < 2; ++i) {
            a[i] = *reinterpret_cast<const x8*>(&As[(wm + 16 * i + lo) * LD + 8 * hi]);
            b[i] = *reinterpret_cast<const x8*>(&Bs[(wn + 16 * i + lo) * LD + 8 * hi]);
        }
        for (int i = 0; i < 2; ++i)
            for (int j = 0; j < 2; ++j) c[i][j] = Vec<T>::mfma(a[i], b[j], c[i][j]);
        __syncthreads();
    }
    // lane: column n = lo of the product's tile, rows m = 4 hi + 0..3
    for (int j = 0; j < 2; ++j) {
        const long n = n0 + wn + 16 * j + lo;
        if constexpr (EPILOGUE == LOGITS) {
            float m = -INFINITY;
            const long first = m0 + wm;
            for (int i = 0; i < 2; ++i)
                for (int r = 0; r < 4; ++r) {
                    if (first + 16 * i + 4 * hi + r >= q.M) c[i][j][r] = -INFINITY;
                    m = nan_max(m, c[i][j][r]);
                }
            m = nan_max(m, __shfl_xor(m, 16));
            m = nan_max(m, __shfl_xor(m, 32));
            const float base = m == -INFINITY ? 0.0f : m;
            float sum = 0.0f;
            const long tgt = n < q.N ? q.target[n] : -1;
            for (int i = 0; i < 2; ++i)
                for (int r = 0; r < 4; ++r) {
                    const long v = first + 16 * i + 4 * hi + r;
                    if (v == tgt && v < q.M) q.zt[n] = c[i][j][r];
                    const float e = exp_of(c[i][j][r] - base);
                    sum += e;
                    if (q.p != nullptr && n < q.N && v < q.ldp) ((T*)q.p)[n * q.ldp + v] = (T)e;
                }
            sum += __shfl_xor(sum, 16);
            sum += __shfl_xor(sum, 32);
            if (hi == 0 && n < q.N && first < q.M) q.stat[n * q.segs + first / SEG] = make_float2(m, sum);
        } else {
            const float alpha = *q.alpha;
            for (int i = 0; i < 2; ++i)
                for (int r = 0; r < 4; ++r) {
                    const long m = m0 + wm + 16 * i + 4 * hi + r;
                    if (m >= q.M || n >= q.N) continue;
                    float v = c[i][j][r];
                    if (q.acc != nullptr) {
                        if (q.add) v += q.acc[n * q.M + m];
                        q.acc[n * q.M + m] = v;
                    }
                    if (q.last) ((T*)q.C)[n * q.ldc + m] = (T)(v * alpha);
                }
        }
    }
}

// a token's weight: 0 where it is ignored, NaN where its target is no column
__device__ __forceinline__ float weight_of(long target, long ignore, long V, const float* row_weight, long i) {
    if (target == ignore) return 0.0f;
    if (target < 0 || target >= V) return NAN;
    return row_weight == nullptr ? 1.0f : row_weight[i];
}

struct Scalars {
    float alpha;    // what dx and dW are multiplied by
    float per;      // what the sum of the losses is multiplied by
    float w_scale;  // G holds the weights times this (a power of 2: the largest weight to [1, 2))
};

// counts the tokens that are not ignored; one workgroup
__global__ __launch_bounds__(1024) void k_prepare(const long* target, long N, long ignore, int mean, const float* row_weight,
                                                  const float* grad_scale, float g, Scalars* out) {
    __shared__ int slot[16];
    __shared__ float most[16];
    int count = 0;
    float w = 0.0f;
    for (long i = threadIdx.x; i < N; i += 1024) {
        const bool kept = target[i] != ignore;
        count += kept;
        if (kept && row_weight != nullptr) {
            const float a = fabsf(row_weight[i]);
            if (a < INFINITY) w = fmaxf(w, a);
        }
    }
    count = reduce_threads<1024, Sum>(count, slot);
    w = reduce_threads<1024, NanMax>(w, most);
    if (threadIdx.x == 0) {
        const float per = mean ? 1.0f / (float)(count > 0 ? count : 1) : 1.0f;
        float s = 1.0f;
        if (w > 0.0f) s = ldexpf(1.0f, -min(max(ilogbf(w), -100), 100));
        out->per = per;
        out->w_scale = s * g;
        out->alpha = per * (grad_scale == nullptr ? 1.0f : *grad_scale) / (s * g);
    }
}

struct FinishArgs {
    long V, segs, ldp, ignore;
    const long* target;
    const float *row_weight, *zt;
    const float2* stat;
    void* p;                     // or null: the loss alone
    float *loss, *lse;
    const Scalars* scal;
};

// one token a blockIdx.x: lse from the segments' statistics, the loss, and p -> G in the columns of blockIdx.y
template <typename T>
__global__ __launch_bounds__(256) void k_finish(const FinishArgs q) {
    __shared__ float slot[4];
    const long i = blockIdx.x;
    const float2* stat = q.stat + i * q.segs;
    float m = -INFINITY;
    for (long s = threadIdx.x; s < q.segs; s += 256) m = nan_max(m, stat[s].x);
    m = reduce_threads<256, NanMax>(m, slot);
    float sum = 0.0f;
    for (long s = threadIdx.x; s < q.segs; s += 256) sum += stat[s].y * exp_of(stat[s].x - m);
    sum = reduce_threads<256, Sum>(sum, slot);
    const float lse = m + logf(sum);
    const long t = q.target[i];
    const float w = weight_of(t, q.ignore, q.V, q.row_weight, i);
    const bool in = t >= 0 && t < q.V && t != q.ignore;
    const float d = in ? q.zt[i] - lse : w;   // log of the target's probability (or 0, or NaN)
    if (blockIdx.y == 0 && threadIdx.x == 0) {
        q.loss[i] = w == 0.0f ? 0.0f : -w * d;
        if (q.lse != nullptr) q.lse[i] = lse;
    }
    if (q.p == nullptr) return;
    T* p = (T*)q.p + i * q.ldp;
    const float f = w * q.scal->w_scale;
    for (long v = 8l * (threadIdx.x + 256l * blockIdx.y); v < q.ldp; v += 8l * 256 * gridDim.y) {
        float e[8];
        if (w == 0.0f) {
#pragma unroll
            for (int k = 0; k < 8; ++k) e[k] = 0.0f;
        } else {
            load8(p + v, 8, e);
            const float s = v < q.V ? f * exp_of(stat[v / SEG].x - lse) : 0.0f;
#pragma unroll
            for (int k = 0; k < 8; ++k) e[k] = v + k < q.V ? e[k] * s : 0.0f;
            if (in && t >= v && t < v + 8) {
#pragma unroll
                for (int k = 0; k < 8; ++k)
                    if (t == v + k) e[k] = f * expm1f(d);
            }
        }
        store8(p + v, 8, e);
    }
}

// the sum (or mean) of the tokens' losses; one workgroup, a fixed order
__global__ __launch_bounds__(1024) void k_total(const float* loss, long N, const Scalars* scal, float* out) {
    __shared__ double slot[16];
    double sum = 0.0;
    for (long i = threadIdx.x; i < N; i += 1024) sum += (double)loss[i];
    sum = reduce_threads<1024, Sum>(sum, slot);
    if (threadIdx.x == 0) *out = (float)(sum * (double)scal->per);
}

constexpr long MAX_N = 1l << 31, MAX_HV = 1l << 24;

long up(long v, long to) { return (v + to - 1) / to * to; }

// where things lie in the workspace, for `tokens` tokens at a time
struct Layout {
    long scal, loss, zt, stat, p, acc, bytes;
    long segs, ldp;
};
Layout layout_of(long N, long H, long V, int grads, long tokens) {
    Layout l;
    l.segs = (V + SEG - 1) / SEG;
    l.ldp = up(V, 64);
    long at = 0;
    auto take = [&](long bytes) {
        const long was = at;
        at += up(bytes, 256);
        return was;
    };
    l.scal = take(sizeof(Scalars));
    l.loss = take(4 * N);
    l.zt = take(4 * tokens);
    l.stat = take(8 * tokens * l.segs);
    l.p = take(grads ? 2 * tokens * l.ldp : 0);
    l.acc = take((grads & 2) && tokens < N ? 4 * H * V : 0);
    l.bytes = at;
    return l;
}

// most tokens at a time within `most` bytes: all, or a multiple of 256 (at least 256)
long tokens_of(long N, long H, long V, int grads, long most) {
    if (N <= 256 || layout_of(N, H, V, grads, N).bytes <= most) return N;
    const long fixed = layout_of(N, H, V, grads, 0).bytes;
    const long each = 8 * ((V + SEG - 1) / SEG) + (grads ? 2 * up(V, 64) : 0) + 4;
    const long fit = (most - fixed) / each / 256 * 256;
    return fit < 256 ? 256 : fit < N ? fit : N;
}

int check_sizes(int type, long N, long H, long V) {
    if (type != SPANQR_BF16 && type != SPANQR_FP16)
        return error(SPANQR_EINVAL, "linear_cross_entropy: x and W are bf16 or fp16");
    if (N < 0 || N > MAX_N || H < 1 || H > MAX_HV || V < 1 || V > MAX_HV)
        return error(SPANQR_EINVAL, "linear_cross_entropy: N = %ld, H = %ld, V = %ld", N, H, V);
    return SPANQR_OK;
}

struct Call {
    int mean;
    bool reduced;
    long N, H, V;
    const void *x, *w;
    long ldx, ldw;
    const long* target;
    long ignore;
    const float *row_weight, *grad_scale;
    float *loss, *lse;
    void *dx, *dw;
};

template <typename T>
int enqueue(const Call& c, char* ws, long tokens, hipStream_t st) {
    const int grads = (c.dx != nullptr ? 1 : 0) | (c.dw != nullptr ? 2 : 0);
    const Layout l = layout_of(c.N, c.H, c.V, grads, tokens);
    Scalars* scal = (Scalars*)(ws + l.scal);
    float* loss = c.reduced ? (float*)(ws + l.loss) : c.loss;
    auto grid = [](long M, long N) { return dim3((unsigned)((M + 63) / 64), (unsigned)((N + 63) / 64)); };
    k_prepare<<<1, 1024, 0, st>>>(c.target, c.N, c.ignore, c.mean, c.row_weight, c.grad_scale, g_scale<T>(), scal);
    for (long at = 0; at < c.N; at += tokens) {
        const long n = c.N - at < tokens ? c.N - at : tokens;
        ProductArgs q = {};
        q.M = c.V, q.N = n, q.K = c.H;
        q.A = c.w, q.lda = c.ldw;
        q.B = (const T*)c.x + at * c.ldx, q.ldb = c.ldx;
        q.target = c.target + at;
        q.zt = (float*)(ws + l.zt);
        q.stat = (float2*)(ws + l.stat);
        q.segs = l.segs;
        q.p = grads ? ws + l.p : nullptr;
        q.ldp = l.ldp;
        k_product<T, true, true, LOGITS><<<grid(q.M, q.N), 256, 0, st>>>(q);
        FinishArgs f = {c.V, l.segs, l.ldp, c.ignore, c.target + at, c.row_weight == nullptr ? nullptr : c.row_weight + at,
                        q.zt, q.stat, q.p, loss + at, c.lse == nullptr ? nullptr : c.lse + at, scal};
        const long split = grads ? (n >= 2048 ? 1 : 2048 / n) : 1, most = (l.ldp + 2047) / 2048;
        k_finish<T><<<dim3((unsigned)n, (unsigned)(split < most ? split : most)), 256, 0, st>>>(f);
        if (c.dx != nullptr) {
            ProductArgs d = {};
            d.M = c.H, d.N = n, d.K = c.V;
            d.A = c.w, d.lda = c.ldw;
            d.B = ws + l.p, d.ldb = l.ldp;
            d.C = (T*)c.dx + at * c.H, d.ldc = c.H;
            d.last = 1;
            d.alpha = &scal->alpha;
            k_product<T, false, true, OUT><<<grid(d.M, d.N), 256, 0, st>>>(d);
        }
        if (c.dw != nullptr) {
            ProductArgs d = {};
            d.M = c.H, d.N = c.V, d.K = n;
            d.A = (const T*)c.x + at * c.ldx, d.lda = c.ldx;
            d.B = ws + l.p, d.ldb = l.ldp;
            d.C = c.dw, d.ldc = c.H;
            d.acc = tokens < c.N ? (float*)(ws + l.acc) : nullptr;
            d.add = at > 0, d.last = at + n == c.N;
            d.alpha = &scal->alpha;
            k_product<T, false, false, OUT><<<grid(d.M, d.N), 256, 0, st>>>(d);
        }
    }
    if (c.N == 0 && c.dw != nullptr) {   // no tokens: a product over nothing
        ProductArgs d = {};
        d.M = c.H, d.N = c.V;
        d.C = c.dw, d.ldc = c.H;
        d.last = 1;
        d.alpha = &scal->alpha;
        k_product<T, false, false, OUT><<<grid(d.M, d.N), 256, 0, st>>>(d);
    }
    if (c.reduced) k_total<<<1, 1024, 0, st>>>(loss, c.N, scal, c.loss);
    return launched("linear_cross_entropy");
}

}  // namespace

extern "C" {

long spanqr_linear_cross_entropy_workspace(int type, long N, long H, long V, int grads, long most_bytes) {
    const int rc = check_sizes(type, N, H, V);
    if (rc != SPANQR_OK) return rc;
    return layout_of(N, H, V, grads, tokens_of(N, H, V, grads, most_bytes)).bytes;
}

int spanqr_linear_cross_entropy(int type, int reduction, long N, long H, long V, const void* x, long ldx, const void* w,
                                long ldw, const long* target, long ignore_index, const float* row_weight,
                                const float* grad_scale, float* loss, float* lse, void* dx, void* dw, void* workspace,
                                long workspace_bytes, void* stream) {
    const int rc = check_sizes(type, N, H, V);
    if (rc != SPANQR_OK) return rc;
    if (reduction != SPANQR_REDUCE_NONE && reduction != SPANQR_REDUCE_SUM && reduction != SPANQR_REDUCE_MEAN)
        return error(SPANQR_EINVAL, "linear_cross_entropy: unknown reduction %d", reduction);
    const bool reduced = reduction != SPANQR_REDUCE_NONE;
    if ((N > 0 && (x == nullptr || target == nullptr)) || w == nullptr || workspace == nullptr ||
        (loss == nullptr && (N > 0 || reduced)))
        return error(SPANQR_EINVAL, "linear_cross_entropy: a missing pointer");
    if ((N > 1 && ldx < H) || (V > 1 && ldw < H))
        return error(SPANQR_EINVAL, "linear_cross_entropy: a row stride below H");
    const int grads = (dx != nullptr ? 1 : 0) | (dw != nullptr ? 2 : 0);
    const long tokens = tokens_of(N, H, V, grads, workspace_bytes);
    if (layout_of(N, H, V, grads, tokens).bytes > workspace_bytes)
        return error(SPANQR_EINVAL, "linear_cross_entropy: the workspace needs %ld bytes",
                     layout_of(N, H, V, grads, tokens).bytes);
    const Call c = {reduction == SPANQR_REDUCE_MEAN, reduced, N, H, V, x, w, ldx, ldw, target, ignore_index, row_weight,
                    grad_scale, loss, lse, dx, dw};
    hipStream_t st = (hipStream_t)stream;
    return type == SPANQR_BF16 ? enqueue<bf16>(c, (char*)workspace, tokens, st)
                               : enqueue<fp16>(c, (char*)workspace, tokens, st);
}

}  // extern "C"
