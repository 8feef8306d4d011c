// Global gradient norm over a list of tensors, and clipping by it (hip/ops.py grad_norm / clip_grad_norm / adam).
//   n = scale * sqrt(sum g^2)  or  scale * max |g|;  c = min(1, max_norm / (n + 1e-6));  out = g * (scale * c)
// HBM-bound: g is read for the norm, read again and written for the scaling. The squares are summed in 64 bits (the
// vector unit does that at its fp32 rate, far above what the loads deliver): no gradient that fp32 or bf16 holds overflows
// or vanishes in its square, and the sum of 10^8 terms keeps its last bits. Every workgroup leaves one partial; the
// partials are joined in a fixed order. 64 M fp32 elements: norm 44 us (5.8 TB/s). 60 tensors of 30 M elements, fp32 and
// bf16: norm 27 us (3.0 TB/s: every tensor's last share is rounded up to a workgroup, 1041 of them where 1024 are resident,
// and the shares are equal in elements, not in bytes), scaling 30 us (6 TB/s, its reads from the cache). A matrix with a row
// stride is shared out by whole rows, so one of few wide rows keeps few workgroups busy.
#include <algorithm>
#include <new>

#include "rows.h"

namespace {

using namespace cgn_rows;

constexpr int GN_NT = 512;
constexpr int GN_MAX = 72;         // tensors per launch: their descriptions travel as kernel arguments (below 4 KB)
constexpr int GN_FEW = 8;
constexpr int GN_BLOCKS = 1024;    // partials of a long list of elements: four workgroups per CU
constexpr int64_t GN_CHUNK = 4096;  // elements a workgroup takes at least

struct Seg {
    const void* g;
    void* out;
    long cols, ld, ldo;  // rows > 1: a matrix with row strides ld / ldo; else cols elements in one piece
    int rows, bf16;
};

template <int N>
struct Segs {
    Seg seg[N];
    int first[N + 1];  // first workgroup of every tensor
    int n;
    bool stream;  // the list is past the caches' size (rows.h)
    long chunk;
};

// The part of tensor t that workgroup b of the launch owns: rows [r0, r1) of columns [c0, c1).
struct Span {
    int t, r0, r1;
    long c0, c1;
};

template <int N>
__device__ __forceinline__ Span span_of(const Segs<N>& a, int b) {
    int lo = 0, hi = a.n - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (a.first[mid] <= b)
            lo = mid;
        else
            hi = mid - 1;
    }
    const Seg& s = a.seg[lo];
    const int k = b - a.first[lo];
    Span p;
    p.t = lo;
    if (s.rows > 1) {
        const int per = s.cols >= a.chunk ? 1 : (int)(a.chunk / s.cols);
        p.r0 = k * per;
        p.r1 = s.rows - p.r0 < per ? s.rows : p.r0 + per;
        p.c0 = 0;
        p.c1 = s.cols;
    } else {
        p.r0 = 0;
        p.r1 = 1;
        p.c0 = (long)k * a.chunk;
        p.c1 = s.cols - p.c0 < a.chunk ? s.cols : p.c0 + a.chunk;
    }
    return p;
}

__device__ __forceinline__ double max_nan(double a, double b) { return a > b || a != a ? a : b; }  // NaN wins

template <bool MAX>
__device__ __forceinline__ double join(double a, double b) {
    return MAX ? max_nan(a, b) : a + b;
}

template <bool MAX>
__device__ __forceinline__ double block_join(double v, double* red) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = join<MAX>(v, __shfl_xor(v, o, 64));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = red[0];
#pragma unroll
    for (int w = 1; w < GN_NT / 64; ++w) v = join<MAX>(v, red[w]);
    return v;
}

// A matrix with a row stride whose rows would leave most of a workgroup idle goes element by element; wider ones row by row.
__device__ __forceinline__ bool narrow(const Seg& s) { return s.rows > 1 && s.cols < GN_NT; }

template <typename T, bool MAX>
__device__ __forceinline__ double part_of(const Seg& s, const Span& p) {
    constexpr int E = Piece<T>::E, U = 4;
    double acc[E];
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = 0.0;
    if (narrow(s)) {
        const long n = (long)(p.r1 - p.r0) * s.cols;
        for (long i = threadIdx.x; i < n; i += GN_NT) {
            const double x = (double)Piece<T>::one((const T*)s.g + (p.r0 + i / s.cols) * s.ld + i % s.cols);
            acc[0] = MAX ? max_nan(fabs(x), acc[0]) : acc[0] + x * x;
        }
    } else {
        for (int r = p.r0; r < p.r1; ++r) {
            const T* g = (const T*)s.g + (long)r * s.ld + p.c0;
            const long n = p.c1 - p.c0, nfull = n / E;
            for (long i0 = threadIdx.x; i0 < nfull; i0 += U * GN_NT) {
                Piece<T> q[U];
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    if (i0 + u * GN_NT < nfull)
                        q[u].load(g + (i0 + u * GN_NT) * E);
                    else
                        q[u].fill(0.f);
                }
#pragma unroll
                for (int u = 0; u < U; ++u)
#pragma unroll
                    for (int e = 0; e < E; ++e) {
                        const double x = (double)q[u].get(e);
                        acc[e] = MAX ? max_nan(fabs(x), acc[e]) : acc[e] + x * x;
                    }
            }
            if (threadIdx.x < n - nfull * E) {
                const double x = (double)Piece<T>::one(g + nfull * E + threadIdx.x);
                acc[0] = MAX ? max_nan(fabs(x), acc[0]) : acc[0] + x * x;
            }
        }
    }
    double t = acc[0];
#pragma unroll
    for (int e = 1; e < E; ++e) t = join<MAX>(t, acc[e]);
    return t;
}

template <bool MAX, int N>
__global__ __launch_bounds__(GN_NT) void norm_part_kernel(const Segs<N> a, double* __restrict__ part) {
    __shared__ double red[GN_NT / 64];
    const Span p = span_of(a, blockIdx.x);
    const Seg& s = a.seg[p.t];
    const double v = s.bf16 ? part_of<Bf16, MAX>(s, p) : part_of<float, MAX>(s, p);
    const double t = block_join<MAX>(v, red);
    if (threadIdx.x == 0) part[blockIdx.x] = t;
}

// The norm, and c = min(1, max_norm / (norm + 1e-6)) with NaN kept, from the partials; every thread gets both.
template <bool MAX>
__device__ __forceinline__ void total_of(const double* part, int n, double scale, double max_norm, double* red,
                                         float* norm, float* coef) {
    double v = 0.0;
    for (int i = threadIdx.x; i < n; i += GN_NT) v = join<MAX>(v, part[i]);
    v = block_join<MAX>(v, red);
    const double nrm = (MAX ? v : sqrt(v)) * fabs(scale);
    *norm = (float)nrm;
    *coef = cgn_clip_factor(nrm, max_norm);
}

template <bool MAX>
__global__ __launch_bounds__(GN_NT) void norm_final_kernel(const double* __restrict__ part, int n, double scale,
                                                           double max_norm, float* __restrict__ norm,
                                                           float* __restrict__ coef) {
    __shared__ double red[GN_NT / 64];
    float v, c;
    total_of<MAX>(part, n, scale, max_norm, red, &v, &c);
    if (threadIdx.x == 0) {
        norm[0] = v;
        if (coef) coef[0] = c;
    }
}

template <typename T>
__device__ __forceinline__ void scale_part(const Seg& s, const Span& p, float f, bool stream) {
    constexpr int E = Piece<T>::E, U = 4;
    if (narrow(s)) {
        const long n = (long)(p.r1 - p.r0) * s.cols;
        for (long i = threadIdx.x; i < n; i += GN_NT) {
            const long r = p.r0 + i / s.cols, c = i % s.cols;
            Piece<T>::put((T*)s.out + r * s.ldo + c, Piece<T>::one((const T*)s.g + r * s.ld + c) * f);
        }
        return;
    }
    for (int r = p.r0; r < p.r1; ++r) {
        const T* g = (const T*)s.g + (long)r * s.ld + p.c0;
        T* out = (T*)s.out + (long)r * s.ldo + p.c0;
        const long n = p.c1 - p.c0, nfull = n / E;
        for (long i0 = threadIdx.x; i0 < nfull; i0 += U * GN_NT) {
            Piece<T> q[U];
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (i0 + u * GN_NT < nfull) q[u].load(g + (i0 + u * GN_NT) * E);
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (i0 + u * GN_NT < nfull) {
                    float o[E];
#pragma unroll
                    for (int e = 0; e < E; ++e) o[e] = q[u].get(e) * f;
                    if (stream)
                        Piece<T>::store_stream(out + (i0 + u * GN_NT) * E, o);
                    else
                        Piece<T>::store(out + (i0 + u * GN_NT) * E, o);
                }
        }
        if (threadIdx.x < n - nfull * E)
            Piece<T>::put(out + nfull * E + threadIdx.x, Piece<T>::one(g + nfull * E + threadIdx.x) * f);
    }
}

// Every workgroup joins the partials itself (a few KB from the L2): one launch less than a kernel for it alone. The spans
// are walked backwards: what the norm's pass read last is still in the 256 MB cache.
template <bool MAX, int N>
__global__ __launch_bounds__(GN_NT) void clip_kernel(const Segs<N> a, const double* __restrict__ part, int nparts,
                                                     double scale, double max_norm, float* __restrict__ norm) {
    __shared__ double red[GN_NT / 64];
    float v, c;
    total_of<MAX>(part, nparts, scale, max_norm, red, &v, &c);
    const int b = gridDim.x - 1 - blockIdx.x;
    if (norm && b == 0 && threadIdx.x == 0) norm[0] = v;
    const Span p = span_of(a, b);
    const Seg& s = a.seg[p.t];
    const float f = (float)(scale * (double)c);
    if (f == 1.f && s.out == s.g) return;  // in place and inside the bound: nothing changes
    if (s.bf16)
        scale_part<Bf16>(s, p, f, a.stream);
    else
        scale_part<float>(s, p, f, a.stream);
}

bool segs_ok(const cgn_grad_tensor* t, int n, bool out) {
    for (int i = 0; i < n; ++i) {
        if (t[i].rows < 0 || t[i].rows > 0x7fffffff || t[i].cols < 0) return false;
        if (t[i].rows == 0 || t[i].cols == 0) continue;
        if (!t[i].g || (out && !t[i].out)) return false;
        if (t[i].rows > 1 && (t[i].ld < t[i].cols || (out && t[i].ldo < t[i].cols))) return false;
        const uintptr_t al = t[i].bf16 ? 2 : 4;
        if ((uintptr_t)t[i].g % al || (out && (uintptr_t)t[i].out % al)) return false;
    }
    return true;
}

// Whether no destination shares memory with another destination or with another tensor's gradient (a destination may be
// its own gradient).
bool apart(const cgn_grad_tensor* t, int n) {
    struct Range {
        uintptr_t a, b;
        bool operator<(const Range& o) const { return a < o.a; }
    };
    Range* r = new (std::nothrow) Range[2 * (size_t)n + 1];
    if (!r) return false;
    int m = 0;
    for (int i = 0; i < n; ++i) {
        if (t[i].rows == 0 || t[i].cols == 0) continue;
        const int64_t size = t[i].bf16 ? 2 : 4;
        const uintptr_t o = (uintptr_t)t[i].out, g = (uintptr_t)t[i].g;
        const int64_t lo = t[i].rows > 1 ? t[i].ldo : 0, lg = t[i].rows > 1 ? t[i].ld : 0;
        r[m++] = Range{o, o + (uintptr_t)(((t[i].rows - 1) * lo + t[i].cols) * size)};
        if (g != o || lo != lg) r[m++] = Range{g, g + (uintptr_t)(((t[i].rows - 1) * lg + t[i].cols) * size)};
    }
    std::sort(r, r + m);
    bool ok = true;
    for (int i = 1; i < m && ok; ++i) ok = r[i - 1].b <= r[i].a;
    delete[] r;
    return ok;
}

int64_t chunk_of(const cgn_grad_tensor* t, int n) {
    int64_t total = 0;
    for (int i = 0; i < n; ++i) total += t[i].rows * t[i].cols;
    int64_t c = ((total + GN_BLOCKS - 1) / GN_BLOCKS + 1023) / 1024 * 1024;  // (one tensor: at most GN_BLOCKS of them)
    return c < GN_CHUNK ? GN_CHUNK : c;
}

int64_t blocks_of(const cgn_grad_tensor& t, int64_t chunk) {
    if (t.rows == 0 || t.cols == 0) return 0;
    if (t.rows == 1) return (t.cols + chunk - 1) / chunk;
    const int64_t per = t.cols >= chunk ? 1 : chunk / t.cols;
    return (t.rows + per - 1) / per;
}

// Fills one launch from tensor i on; returns the tensor behind it.
template <int N>
int pack(const cgn_grad_tensor* t, int n, int i, int64_t chunk, Segs<N>* a, int64_t* blocks) {
    a->n = 0;
    a->chunk = chunk;
    a->stream = chunk * GN_BLOCKS * 4 >= STREAM_BYTES;
    *blocks = 0;
    for (; i < n && a->n < N; ++i) {
        const int64_t b = blocks_of(t[i], chunk);
        if (b == 0) continue;
        a->seg[a->n] = Seg{t[i].g, t[i].out, (long)t[i].cols, (long)t[i].ld, (long)t[i].ldo, (int)t[i].rows,
                           t[i].bf16 ? 1 : 0};
        a->first[a->n++] = (int)*blocks;
        *blocks += b;
    }
    a->first[a->n] = (int)*blocks;
    return i;
}

int64_t parts_of(const cgn_grad_tensor* t, int n) {
    const int64_t chunk = chunk_of(t, n);
    int64_t parts = 0;
    for (int i = 0; i < n; ++i) parts += blocks_of(t[i], chunk);
    return parts;
}

template <bool MAX, int N>
int norm_parts_in(hipStream_t s, const cgn_grad_tensor* t, int n, double* part) {
    const int64_t chunk = chunk_of(t, n);
    int64_t done = 0;
    for (int i = 0; i < n;) {
        Segs<N> a;
        int64_t blocks;
        i = pack(t, n, i, chunk, &a, &blocks);
        if (blocks == 0) continue;
        hipLaunchKernelGGL((norm_part_kernel<MAX, N>), dim3((unsigned)blocks), dim3(GN_NT), 0, s, a, part + done);
        CGN_LAUNCH_CHECK();
        done += blocks;
    }
    return CGN_OK;
}

// (a short list's description is a tenth of the kernel arguments that a full one takes)
template <bool MAX>
int norm_parts(hipStream_t s, const cgn_grad_tensor* t, int n, double* part) {
    return n <= GN_FEW ? norm_parts_in<MAX, GN_FEW>(s, t, n, part) : norm_parts_in<MAX, GN_MAX>(s, t, n, part);
}

template <bool MAX>
int run_norm(hipStream_t s, const cgn_grad_tensor* t, int n, double scale, double max_norm, float* norm, float* coef,
             double* part, int parts) {
    const int rc = norm_parts<MAX>(s, t, n, part);
    if (rc != CGN_OK) return rc;
    hipLaunchKernelGGL(norm_final_kernel<MAX>, dim3(1), dim3(GN_NT), 0, s, part, parts, scale, max_norm, norm, coef);
    CGN_LAUNCH_CHECK();
    return CGN_OK;
}

template <bool MAX, int N>
int clip_in(hipStream_t s, const cgn_grad_tensor* t, int n, double scale, double max_norm, float* norm,
            const double* part, int parts) {
    const int64_t chunk = chunk_of(t, n);
    for (int i = 0; i < n;) {
        Segs<N> a;
        int64_t blocks;
        i = pack(t, n, i, chunk, &a, &blocks);
        if (blocks == 0) continue;
        hipLaunchKernelGGL((clip_kernel<MAX, N>), dim3((unsigned)blocks), dim3(GN_NT), 0, s, a, part, parts, scale, max_norm,
                           norm);
        CGN_LAUNCH_CHECK();
        norm = nullptr;  // written once
    }
    return CGN_OK;
}

template <bool MAX>
int run_clip(hipStream_t s, const cgn_grad_tensor* t, int n, double scale, double max_norm, float* norm, double* part,
             int parts) {
    if (parts == 0) return run_norm<MAX>(s, t, n, scale, max_norm, norm, nullptr, part, 0);
    const int rc = norm_parts<MAX>(s, t, n, part);
    if (rc != CGN_OK) return rc;
    return n <= GN_FEW ? clip_in<MAX, GN_FEW>(s, t, n, scale, max_norm, norm, part, parts)
                       : clip_in<MAX, GN_MAX>(s, t, n, scale, max_norm, norm, part, parts);
}

}  // namespace

// One flat fp32 arena: the partials of its sum of squares in part[0 .. *parts), and with `coef` the norm and the factor too.
int cgn_arena_norm(void* stream, const float* g, int64_t n, double scale, double max_norm, float* norm, float* coef,
                   double* part, int* parts) {
    const cgn_grad_tensor t = {g, nullptr, 1, n, 0, 0, 0};
    *parts = (int)parts_of(&t, 1);
    hipStream_t s = (hipStream_t)stream;
    return coef ? run_norm<false>(s, &t, 1, scale, max_norm, norm, coef, part, *parts) : norm_parts<false>(s, &t, 1, part);
}

extern "C" int cgn_grad_norm_workspace(const cgn_grad_tensor* t, int32_t n, int32_t clip, int64_t* bytes) {
    CGN_CHECK_ARG(n >= 0 && bytes && (n == 0 || t) && segs_ok(t, n, clip != 0) && (!clip || apart(t, n)));
    const int64_t parts = parts_of(t, n);
    CGN_CHECK_ARG(parts <= 0x7fffffff);
    *bytes = parts * 8 + 8;
    return CGN_OK;
}

extern "C" int cgn_grad_norm(void* stream, const cgn_grad_tensor* t, int32_t n, int32_t max_abs, double scale, float* norm,
                             void* workspace, int64_t workspace_bytes) {
    int64_t need;
    const int rc = cgn_grad_norm_workspace(t, n, 0, &need);
    if (rc != CGN_OK) return rc;
    CGN_CHECK_ARG(norm && workspace && (uintptr_t)workspace % 8 == 0);
    if (need > workspace_bytes) return CGN_ERR_WORKSPACE;
    const int parts = (int)((need - 8) / 8);
    hipStream_t s = (hipStream_t)stream;
    double* part = (double*)workspace;
    return max_abs ? run_norm<true>(s, t, n, scale, 0.0, norm, nullptr, part, parts)
                   : run_norm<false>(s, t, n, scale, 0.0, norm, nullptr, part, parts);
}

extern "C" int cgn_clip_grads(void* stream, const cgn_grad_tensor* t, int32_t n, int32_t max_abs, double scale,
                              double max_norm, float* norm, void* workspace, int64_t workspace_bytes) {
    int64_t need;
    const int rc = cgn_grad_norm_workspace(t, n, 1, &need);
    if (rc != CGN_OK) return rc;
    CGN_CHECK_ARG(norm && max_norm >= 0.0 && workspace && (uintptr_t)workspace % 8 == 0);
    if (need > workspace_bytes) return CGN_ERR_WORKSPACE;
    const int parts = (int)((need - 8) / 8);
    hipStream_t s = (hipStream_t)stream;
    double* part = (double*)workspace;
    return max_abs ? run_clip<true>(s, t, n, scale, max_norm, norm, part, parts)
                   : run_clip<false>(s, t, n, scale, max_norm, norm, part, parts);
}
