// Losses over sampled tokens, from the [M, V] logits of the vocabulary projection (hip/ops.py token_logp, policy_loss,
// preference_loss). With s = inv_tau, row maximum m and total z = sum exp(s (x - m)):
//   lp = s (x_t - m) - log z,   d(sum c_i lp_i) / dx_iv = c_i s (1[v = t_i] - exp(s (x_iv - m_i)) / z_i)
// m and z are kept apart (not as m s + log z): lp and the probabilities then carry no rounding of a sum that is large
// against them. HBM-bound: two to five flops and one v_exp_f32 per element. One workgroup holds a row in registers, so
// a loss whose row gradient needs nothing but the row (the policy loss) reads the logits once and writes the gradient
// once. Rows of weight zero (the padding of a batch) are not read: their log-probability and gradient are zeros.
#include "rows.h"

namespace {

using namespace cgn_rows;

constexpr float LOG2E = 1.44269504088896340736f;

struct RowArgs {
    const void* logits;
    long ld;
    const int64_t* target;
    const float* weight;  // null: every row counts with 1
    int V;
    float inv_tau;
    const float* dyn_inv_tau;
    float* logp;     // [M], nullable
    double* lp64;    // [M], nullable: for sums over a sentence
    float* stats;    // [M][2] = (m, z), nullable
    // the policy loss (advantage != null)
    const float* advantage;
    const float* old_logp;  // null: the rows were sampled by these very logits (ratio 1)
    const float* ref_logp;  // null: no KL term
    float clip_lo, clip_hi, kl_coef;
    double* row_loss;  // [M]
    float* coef;       // [M], nullable: d loss / d lp of the row
    void* dlogits;     // may be the logits' own buffer
    long ldd;
};

__device__ __forceinline__ float fast_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

// Everything of a row that is one number; called by one thread. Returns d loss / d lp.
template <typename T>
__device__ __forceinline__ float row_scalars(const RowArgs& a, long row, float w, float inv_tau, float m, float z) {
    const int64_t t = a.target[row];
    // (an out-of-range target gives NaN, never an out-of-bounds read)
    const bool in = t >= 0 && t < a.V;
    const double xt = in ? (double)Piece<T>::one((const T*)a.logits + row * a.ld + t) : (double)NAN;
    const double lp = (xt - (double)m) * (double)inv_tau - (double)logf(z);
    if (a.logp) a.logp[row] = (float)lp;
    if (a.lp64) a.lp64[row] = lp * (double)w;
    if (a.stats) {
        a.stats[2 * row] = m;
        a.stats[2 * row + 1] = z;
    }
    if (!a.advantage) return 0.f;
    const float A = a.advantage[row];
    const float ratio = a.old_logp ? expf((float)(lp - (double)a.old_logp[row])) : 1.f;
    const float lim = fminf(fmaxf(ratio, 1.f - a.clip_lo), 1.f + a.clip_hi);
    const bool cut = (A > 0.f && ratio > 1.f + a.clip_hi) || (A < 0.f && ratio < 1.f - a.clip_lo);
    float loss = -(cut ? lim : ratio) * A, g = cut ? 0.f : -ratio * A;
    if (a.ref_logp) {
        // exp(k) - k - 1 and its derivative through expm1: k is small where the two policies agree
        const float k = (float)((double)a.ref_logp[row] - lp), e = expm1f(k);
        loss += a.kl_coef * (e - k);
        g -= a.kl_coef * e;
    }
    a.row_loss[row] = (double)loss * (double)w;
    g *= w;
    if (a.coef) a.coef[row] = g;
    return g;
}

__device__ __forceinline__ void masked_scalars(const RowArgs& a, long row) {
    if (a.logp) a.logp[row] = 0.f;
    if (a.lp64) a.lp64[row] = 0.0;
    if (a.stats) {
        a.stats[2 * row] = 0.f;
        a.stats[2 * row + 1] = 1.f;
    }
    if (a.row_loss) a.row_loss[row] = 0.0;
    if (a.coef) a.coef[row] = 0.f;
}

template <typename T, int NT>
__device__ __forceinline__ void zero_row(T* d, int V) {
    constexpr int E = Piece<T>::E;
    const int nfull = V / E, rem = V % E;
    float o[E];
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = 0.f;
    for (int i = threadIdx.x; i < nfull; i += NT) Piece<T>::store(d + (long)i * E, o);
    if (threadIdx.x < rem) Piece<T>::put(d + nfull * E + threadIdx.x, 0.f);
}

// One workgroup per row, the row in registers (NV 16-byte pieces per thread and one single element of the V % E last).
template <typename T, int NT, int NV>
__global__ __launch_bounds__(NT) void row_kernel(const RowArgs a) {
    constexpr int E = Piece<T>::E;
    __shared__ float red[NT / 64 + 1];
    __shared__ float coef_s;
    const long row = blockIdx.x;
    const float w = a.weight ? a.weight[row] : 1.f;
    T* d = a.dlogits ? (T*)a.dlogits + row * a.ldd : nullptr;
    if (w == 0.f) {
        if (d) zero_row<T, NT>(d, a.V);
        if (threadIdx.x == 0) masked_scalars(a, row);
        return;
    }
    const float inv_tau = a.dyn_inv_tau ? a.dyn_inv_tau[0] : a.inv_tau;
    const T* x = (const T*)a.logits + row * a.ld;
    const int nfull = a.V / E, rem = a.V % E;
    Piece<T> q[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int i = threadIdx.x + j * NT;
        if (i < nfull)
            q[j].load(x + (long)i * E);
        else
            q[j].fill(-INFINITY);
    }
    const float xt = threadIdx.x < rem ? Piece<T>::one(x + nfull * E + threadIdx.x) : -INFINITY;
    float m = xt;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int e = 0; e < E; ++e) m = fmaxf(m, q[j].get(e));
    m = block_max<NT>(m, red);
    const float c2 = inv_tau * LOG2E;
    const float et = fast_exp2((xt - m) * c2);
    float part[E];
#pragma unroll
    for (int e = 0; e < E; ++e) part[e] = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int e = 0; e < E; ++e) part[e] += fast_exp2((q[j].get(e) - m) * c2);
    float z = et;
#pragma unroll
    for (int e = 0; e < E; ++e) z += part[e];
    z = block_sum<NT>(z, red);
    if (threadIdx.x == 0) coef_s = row_scalars<T>(a, row, w, inv_tau, m, z);
    if (!d) return;
    __syncthreads();
    const float c = coef_s * inv_tau, cz = -c / z;
    const int64_t t = a.target[row];
    const int tp = t >= 0 && t < a.V ? (int)t / E : -1, te = (int)t % E;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int i = threadIdx.x + j * NT;
        if (i < nfull) {
            float o[E];
#pragma unroll
            for (int e = 0; e < E; ++e) o[e] = fast_exp2((q[j].get(e) - m) * c2) * cz;
            if (i == tp) {
#pragma unroll
                for (int e = 0; e < E; ++e) o[e] += e == te ? c : 0.f;
            }
            Piece<T>::store(d + (long)i * E, o);
        }
    }
    if (threadIdx.x < rem)
        Piece<T>::put(d + nfull * E + threadIdx.x, et * cz + (tp == nfull && te == (int)threadIdx.x ? c : 0.f));
}

// A row too long for the registers of a workgroup: running maximum and total per thread, joined at the end.
template <typename T, int NT>
__global__ __launch_bounds__(NT) void row_stream_kernel(const RowArgs a) {
    constexpr int E = Piece<T>::E;
    __shared__ float red[NT / 64 + 1];
    const long row = blockIdx.x;
    const float w = a.weight ? a.weight[row] : 1.f;
    if (w == 0.f) {
        if (threadIdx.x == 0) masked_scalars(a, row);
        return;
    }
    const float inv_tau = a.dyn_inv_tau ? a.dyn_inv_tau[0] : a.inv_tau;
    const float c2 = inv_tau * LOG2E;
    const T* x = (const T*)a.logits + row * a.ld;
    const int nfull = a.V / E, rem = a.V % E;
    constexpr int U = 4;  // pieces in flight
    float m = -INFINITY, z = 0.f;
    for (int i0 = threadIdx.x; i0 < nfull; i0 += U * NT) {
        Piece<T> q[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (i0 + u * NT < nfull)
                q[u].load(x + (long)(i0 + u * NT) * E);
            else
                q[u].fill(-INFINITY);
        }
        float mx = m;
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int e = 0; e < E; ++e) mx = fmaxf(mx, q[u].get(e));
        const float base = mx == -INFINITY ? 0.f : mx;  // (nothing but -inf so far: every term is zero)
        z *= fast_exp2((m - base) * c2);
        m = mx;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            float p = 0.f;
#pragma unroll
            for (int e = 0; e < E; ++e) p += fast_exp2((q[u].get(e) - base) * c2);
            z += p;
        }
    }
    const float xt = threadIdx.x < rem ? Piece<T>::one(x + nfull * E + threadIdx.x) : -INFINITY;
    const float mb = block_max<NT>(fmaxf(m, xt), red);
    const float mine = m == -INFINITY && z == 0.f ? 0.f : z * fast_exp2((m - mb) * c2);
    z = block_sum<NT>(mine + fast_exp2((xt - mb) * c2), red);
    if (threadIdx.x == 0) row_scalars<T>(a, row, w, inv_tau, mb, z);
}

struct GradArgs {
    const void* logits;
    long ld;
    const int64_t* target;
    const float* weight;  // nullable
    int V;
    float inv_tau;
    const float* dyn_inv_tau;
    const float* stats;  // [M][2]
    const float* coef;   // [M]
    const float* scale;  // nullable: one factor on the device (the gradient of the loss itself)
    void* dlogits;       // may be the logits' own buffer: every element is read and written by one thread
    long ldd;
};

template <typename T, int NT>
__global__ __launch_bounds__(NT) void row_grad_kernel(const GradArgs a) {
    constexpr int E = Piece<T>::E;
    const long row = blockIdx.x;
    T* d = (T*)a.dlogits + row * a.ldd;
    if (a.weight && a.weight[row] == 0.f) {
        zero_row<T, NT>(d, a.V);
        return;
    }
    const float inv_tau = a.dyn_inv_tau ? a.dyn_inv_tau[0] : a.inv_tau;
    const float c2 = inv_tau * LOG2E, m = a.stats[2 * row], z = a.stats[2 * row + 1];
    const float c = a.coef[row] * (a.scale ? a.scale[0] : 1.f) * inv_tau, cz = -c / z;
    const T* x = (const T*)a.logits + row * a.ld;
    const int nfull = a.V / E, rem = a.V % E;
    const int64_t t = a.target[row];
    const int tp = t >= 0 && t < a.V ? (int)t / E : -1, te = (int)t % E;
    constexpr int U = 4;
    for (int i0 = threadIdx.x; i0 < nfull; i0 += U * NT) {
        Piece<T> q[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (i0 + u * NT < nfull) q[u].load(x + (long)(i0 + u * NT) * E);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = i0 + u * NT;
            if (i >= nfull) break;
            float o[E];
#pragma unroll
            for (int e = 0; e < E; ++e) o[e] = fast_exp2((q[u].get(e) - m) * c2) * cz;
            if (i == tp) {
#pragma unroll
                for (int e = 0; e < E; ++e) o[e] += e == te ? c : 0.f;
            }
            Piece<T>::store(d + (long)i * E, o);
        }
    }
    if (threadIdx.x < rem) {
        const float p = fast_exp2((Piece<T>::one(x + nfull * E + threadIdx.x) - m) * c2);
        Piece<T>::put(d + nfull * E + threadIdx.x, p * cz + (tp == nfull && te == (int)threadIdx.x ? c : 0.f));
    }
}

__device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

// out[0] = scale * sum v: one workgroup, a fixed order, in 64 bits (a loss is a sum of terms of both signs).
constexpr int SUM_NT = 1024;
__global__ __launch_bounds__(SUM_NT) void sum64_kernel(const double* __restrict__ v, long n, double scale,
                                                       float* __restrict__ out) {
    __shared__ double red[SUM_NT / 64];
    double s = 0.0;
    for (long i = threadIdx.x; i < n; i += SUM_NT) s += v[i];
    s = wave_sum64(s);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        double t = 0.0;
        for (int i = 0; i < SUM_NT / 64; ++i) t += red[i];
        out[0] = (float)(t * scale);
    }
}

// One workgroup per pair (p chosen, P + p rejected): the sentences' log-probabilities, the margin, the loss, and the
// gradient every row of the two sentences takes into its logits.
constexpr int PAIR_NT = 128;
__global__ __launch_bounds__(PAIR_NT) void pair_kernel(const double* __restrict__ lp64, const float* __restrict__ weight,
                                                       const float* __restrict__ ref, int P, int T, double beta,
                                                       double smooth, float* __restrict__ seq_logp,
                                                       float* __restrict__ margin, double* __restrict__ pair_loss,
                                                       float* __restrict__ coef) {
    __shared__ double S[2];
    const int p = blockIdx.x, side = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const long seq = (long)side * P + p;
    double s = 0.0;
    for (int t = lane; t < T; t += 64) s += lp64[seq * T + t];
    s = wave_sum64(s);
    if (lane == 0) {
        S[side] = s - (double)ref[seq];
        seq_logp[seq] = (float)s;
    }
    __syncthreads();
    const double mg = beta * (S[0] - S[1]);
    // log sig(m) = min(m, 0) - log1p(exp(-|m|)); sig(-m) = exp(-|m|) or 1 over 1 + exp(-|m|)
    const double ex = exp(-fabs(mg)), l1 = log1p(ex);
    const double pos = mg >= 0.0 ? 1.0 / (1.0 + ex) : ex / (1.0 + ex);
    const double neg = mg >= 0.0 ? ex / (1.0 + ex) : 1.0 / (1.0 + ex);
    const double up = -(beta / (double)P) * ((1.0 - smooth) * neg - smooth * pos);
    if (threadIdx.x == 0) {
        margin[p] = (float)mg;
        pair_loss[p] = -((1.0 - smooth) * (fmin(mg, 0.0) - l1) + smooth * (fmin(-mg, 0.0) - l1));
    }
    if (coef)
        for (int t = lane; t < T; t += 64)
            coef[seq * T + t] = (float)((side ? -up : up) * (double)weight[seq * T + t]);
}

template <typename T, int NT, int NV>
int launch_row(hipStream_t s, const RowArgs& a, int64_t M) {
    hipLaunchKernelGGL((row_kernel<T, NT, NV>), dim3((unsigned)M), dim3(NT), 0, s, a);
    CGN_LAUNCH_CHECK();
    return CGN_OK;
}

template <typename T>
int launch_grad(hipStream_t s, const GradArgs& g, int64_t M) {
    hipLaunchKernelGGL((row_grad_kernel<T, 512>), dim3((unsigned)M), dim3(512), 0, s, g);
    CGN_LAUNCH_CHECK();
    return CGN_OK;
}

// Row statistics and scalars of M rows; with a.dlogits the gradient too, where a workgroup's registers hold the row
// (*done says whether they did).
template <typename T>
int launch_rows(hipStream_t s, RowArgs a, int64_t M, bool* done) {
    const int n = cgn_cdiv(a.V, Piece<T>::E);
    *done = true;
    if (n <= 256 * 1) return launch_row<T, 256, 1>(s, a, M);
    if (n <= 256 * 2) return launch_row<T, 256, 2>(s, a, M);
    if (n <= 256 * 4) return launch_row<T, 256, 4>(s, a, M);
    if (n <= 256 * 8) return launch_row<T, 256, 8>(s, a, M);
    if (n <= 512 * 8) return launch_row<T, 512, 8>(s, a, M);
    if (n <= 512 * 12) return launch_row<T, 512, 12>(s, a, M);
    if (n <= 512 * 16) return launch_row<T, 512, 16>(s, a, M);
    if (n <= 1024 * 12) return launch_row<T, 1024, 12>(s, a, M);
    if (n <= 1024 * 16) return launch_row<T, 1024, 16>(s, a, M);
    *done = false;
    hipLaunchKernelGGL((row_stream_kernel<T, 1024>), dim3((unsigned)M), dim3(1024), 0, s, a);
    CGN_LAUNCH_CHECK();
    return CGN_OK;
}

int run_rows(hipStream_t s, const RowArgs& a, int64_t M, bool bf16, bool* done) {
    return bf16 ? launch_rows<Bf16>(s, a, M, done) : launch_rows<float>(s, a, M, done);
}

int run_grad(hipStream_t s, const GradArgs& g, int64_t M, bool bf16) {
    return bf16 ? launch_grad<Bf16>(s, g, M) : launch_grad<float>(s, g, M);
}

int run_sum(hipStream_t s, const double* v, int64_t n, double scale, float* out) {
    hipLaunchKernelGGL(sum64_kernel, dim3(1), dim3(SUM_NT), 0, s, v, (long)n, scale, out);
    CGN_LAUNCH_CHECK();
    return CGN_OK;
}

bool base_ok(const cgn_token_rows* r) {
    return r && r->M >= 0 && r->M <= 0x7fffffff && r->V > 0 && r->ld >= r->V &&
           (r->dyn_inv_tau || r->inv_tau > 0.f) && (r->M == 0 || (r->logits && r->target));
}

RowArgs row_args(const cgn_token_rows* r) {
    RowArgs a = {};
    a.logits = r->logits;
    a.ld = r->ld;
    a.target = r->target;
    a.weight = r->weight;
    a.V = r->V;
    a.inv_tau = r->inv_tau;
    a.dyn_inv_tau = r->dyn_inv_tau;
    return a;
}

int row_gradient(hipStream_t s, const cgn_token_rows* r, const float* stats, const float* coef, const float* scale,
                 void* dlogits, int64_t ldd) {
    GradArgs g = {r->logits, r->ld, r->target, r->weight, r->V, r->inv_tau, r->dyn_inv_tau, stats, coef, scale, dlogits,
                  ldd};
    return run_grad(s, g, r->M, r->bf16 != 0);
}

}  // namespace

extern "C" int cgn_token_logp(void* stream, const cgn_token_rows* r, float* logp, float* stats) {
    CGN_CHECK_ARG(base_ok(r));
    if (r->M == 0) return CGN_OK;
    CGN_CHECK_ARG(logp);
    RowArgs a = row_args(r);
    a.logp = logp;
    a.stats = stats;
    bool done;
    return run_rows((hipStream_t)stream, a, r->M, r->bf16 != 0, &done);
}

extern "C" int cgn_token_logp_bwd(void* stream, const cgn_token_rows* r, const float* stats, const float* coef,
                                  const float* scale, void* dlogits, int64_t ldd) {
    CGN_CHECK_ARG(base_ok(r) && ldd >= r->V);
    if (r->M == 0) return CGN_OK;
    CGN_CHECK_ARG(stats && coef && dlogits);
    return row_gradient((hipStream_t)stream, r, stats, coef, scale, dlogits, ldd);
}

extern "C" int cgn_policy_loss(void* stream, const cgn_token_rows* r, const float* advantage, const float* old_logp,
                               const float* ref_logp, float clip_lo, float clip_hi, float kl_coef, float* loss,
                               float* logp, float* stats, float* coef, void* dlogits, int64_t ldd, void* workspace,
                               int64_t workspace_bytes) {
    CGN_CHECK_ARG(base_ok(r) && loss && clip_lo >= 0.f && clip_hi >= 0.f && (!dlogits || ldd >= r->V));
    CGN_CHECK_ARG(r->M == 0 || (advantage && logp && workspace && (uintptr_t)workspace % 8 == 0));
    if (r->M * 24 + 16 > workspace_bytes) return CGN_ERR_WORKSPACE;
    hipStream_t s = (hipStream_t)stream;
    double* row_loss = (double*)workspace;
    if (dlogits) {  // (a row too long for the registers takes its gradient from these)
        stats = stats ? stats : (float*)(row_loss + r->M);
        coef = coef ? coef : (float*)(row_loss + 2 * r->M);
    }
    if (r->M > 0) {
        RowArgs a = row_args(r);
        a.advantage = advantage;
        a.old_logp = old_logp;
        a.ref_logp = ref_logp;
        a.clip_lo = clip_lo;
        a.clip_hi = clip_hi;
        a.kl_coef = kl_coef;
        a.logp = logp;
        a.stats = stats;
        a.coef = coef;
        a.row_loss = row_loss;
        a.dlogits = dlogits;
        a.ldd = ldd;
        bool done;
        int rc = run_rows(s, a, r->M, r->bf16 != 0, &done);
        if (rc == CGN_OK && dlogits && !done) rc = row_gradient(s, r, stats, coef, nullptr, dlogits, ldd);
        if (rc != CGN_OK) return rc;
    }
    return run_sum(s, row_loss, r->M, 1.0, loss);
}

extern "C" int cgn_preference_loss(void* stream, const cgn_token_rows* r, int32_t T, const float* ref_logp, double beta,
                                   double label_smoothing, float* loss, float* margin, float* seq_logp, float* stats,
                                   float* coef, void* dlogits, int64_t ldd, void* workspace, int64_t workspace_bytes) {
    CGN_CHECK_ARG(base_ok(r) && T > 0 && r->M > 0 && r->M % (2 * (int64_t)T) == 0 && r->weight);
    CGN_CHECK_ARG(beta > 0.0 && label_smoothing >= 0.0 && label_smoothing < 0.5);
    CGN_CHECK_ARG(ref_logp && loss && margin && seq_logp && (!dlogits || ldd >= r->V));
    CGN_CHECK_ARG(workspace && (uintptr_t)workspace % 8 == 0);
    const int P = (int)(r->M / (2 * (int64_t)T));
    if (r->M * 24 + 16 > workspace_bytes) return CGN_ERR_WORKSPACE;
    hipStream_t s = (hipStream_t)stream;
    double *lp64 = (double*)workspace, *pair_loss = lp64 + r->M;  // (P <= M / 2)
    if (dlogits) {
        stats = stats ? stats : (float*)(lp64 + r->M + (r->M + 1) / 2);
        coef = coef ? coef : (float*)(lp64 + r->M + (r->M + 1) / 2) + 2 * r->M;
    }
    RowArgs a = row_args(r);
    a.lp64 = lp64;
    a.stats = stats;
    bool done;
    int rc = run_rows(s, a, r->M, r->bf16 != 0, &done);
    if (rc != CGN_OK) return rc;
    hipLaunchKernelGGL(pair_kernel, dim3(P), dim3(PAIR_NT), 0, s, lp64, r->weight, ref_logp, P, T, beta, label_smoothing,
                       seq_logp, margin, pair_loss, coef);
    CGN_LAUNCH_CHECK();
    if (dlogits) rc = row_gradient(s, r, stats, coef, nullptr, dlogits, ldd);
    return rc != CGN_OK ? rc : run_sum(s, pair_loss, P, 1.0 / P, loss);
}
