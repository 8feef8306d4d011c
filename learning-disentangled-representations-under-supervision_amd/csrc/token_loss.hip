// Losses over sampled tokens, from the [M, V] logits of the vocabulary projection (hip/ops.py token_logp, policy_loss,
// preference_loss). With s = inv_tau, row maximum m and total z = sum exp(s (x - m)):
//   lp = s (x_t - m) - log z,   d(sum c_i lp_i) / dx_iv = c_i s (1[v = t_i] - exp(s (x_iv - m_i)) / z_i)
// m and z are kept apart (not as m s + log z): lp and the probabilities then carry no rounding of a sum that is large
// against them. HBM-bound: two to five flops and one v_exp_f32 per element. One workgroup holds a row in registers, so
// a loss whose row gradient needs nothing but the row (the policy loss) reads the logits once and writes the gradient
// once. Rows of weight zero (the padding of a batch) are not read: their log-probability and gradient are zeros.
// Loss and gradient of 10496 x 50000 bf16 rows: 414 us with all of them live (5.1 TB/s, what a copy reaches), 313 us with
// half of them padding; log-probabilities alone 5.3 to 5.7 TB/s; the gradient pass from saved statistics 5.4 to 6.0 TB/s.
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
    bool stream_in, stream_out;  // logits / dlogits are past the caches' size (rows.h)
};

__device__ __forceinline__ float fast_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

template <typename T>
__device__ __forceinline__ float piece_max(const Piece<T>& q, float m) {
#pragma unroll
    for (int e = 0; e < Piece<T>::E; e += 2) m = fmaxf(fmaxf(q.get(e), q.get(e + 1)), m);
    return m;
}
// An infinite total (an infinite logit): the row's results are NaN, as log_softmax has them.
__device__ __forceinline__ float total(float z) { return z < INFINITY ? z : NAN; }

// Everything of a row that is one number, in the hands of one thread: loaded before the row itself, so that the dependent
// loads (target, then the target's logit) pass beside the row's; then, with the row's maximum and total, first the factor
// that the workgroup waits for, in fp32, and at the end, behind the gradient's stores, what is written out, in 64 bits: a
// loss is a sum of terms of both signs, where the roundings of logf and expf would show.
struct RowScalars {
    float xt, A, old_logp, ref_logp;

    template <typename T>
    __device__ __forceinline__ void load(const RowArgs& a, long row) {
        const int64_t t = a.target[row];
        A = a.advantage ? a.advantage[row] : 0.f;
        old_logp = a.old_logp ? a.old_logp[row] : 0.f;
        ref_logp = a.ref_logp ? a.ref_logp[row] : 0.f;
        // (an out-of-range target gives NaN, never an out-of-bounds read)
        xt = t >= 0 && t < a.V ? Piece<T>::one((const T*)a.logits + row * a.ld + t) : NAN;
    }

    // The ratio to the policy that sampled the token. Without one it is 1, but for a token without a log-probability (a
    // target outside the vocabulary, a NaN logit): its loss and its gradient are NaN. (-inf has one: a ratio of 1.)
    static __device__ __forceinline__ double ratio_1(double lp) { return lp == lp ? 1.0 : lp; }

    // d loss / d lp. expm1: k is small where the two policies agree.
    __device__ __forceinline__ float slope(const RowArgs& a, float w, float inv_tau, float m, float z) const {
        const double lp = ((double)xt - (double)m) * (double)inv_tau - (double)logf(z);
        const float ratio = a.old_logp ? expf((float)(lp - (double)old_logp)) : (float)ratio_1(lp);
        const bool cut = (A > 0.f && ratio > 1.f + a.clip_hi) || (A < 0.f && ratio < 1.f - a.clip_lo);
        float g = cut ? 0.f : -ratio * A;
        if (a.ref_logp) g -= a.kl_coef * expm1f((float)((double)ref_logp - lp));
        return g * w;
    }

    __device__ __forceinline__ void write(const RowArgs& a, long row, float w, float inv_tau, float m, float z,
                                          float g) const {
        const double lp = ((double)xt - (double)m) * (double)inv_tau - log((double)z);
        if (a.logp) a.logp[row] = (float)lp;
        if (a.lp64) a.lp64[row] = lp * (double)w;
        if (a.stats) {
            a.stats[2 * row] = m;
            a.stats[2 * row + 1] = z;
        }
        if (!a.advantage) return;
        if (a.coef) a.coef[row] = g;
        const double ratio = a.old_logp ? exp(lp - (double)old_logp) : ratio_1(lp);
        const double lo = 1.0 - (double)a.clip_lo, hi = 1.0 + (double)a.clip_hi;
        // the smaller of ratio A and clip(ratio) A
        const double kept = A > 0.f ? (ratio > hi ? hi : ratio) : (ratio < lo ? lo : ratio);
        double loss = -kept * (double)A;
        if (a.ref_logp) {
            const double k = (double)ref_logp - lp, e = expm1(k);
            loss += (double)a.kl_coef * (e == INFINITY ? e : e - k);
        }
        a.row_loss[row] = loss * (double)w;
    }
};

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

template <typename T>
__device__ __forceinline__ void put_piece(T* p, const float (&o)[Piece<T>::E], bool stream) {
    if (stream)
        Piece<T>::store_stream(p, o);
    else
        Piece<T>::store(p, o);
}

// A row cut at the 128-byte lines of its buffer: `head` elements up to the first line, nfull whole 16-byte pieces from
// there on, the rest behind them. The head's and the rest's elements (at most 70) go one to a thread. The accesses of a wave
// are then whole lines: on rows that start 32 bytes into a line a copy of this shape loses a tenth without it.
template <typename T>
struct Cut {
    static constexpr int E = Piece<T>::E;
    int head, nfull, edge;
    __device__ __forceinline__ Cut(const T* row, int V) {
        head = (int)((128 - ((uintptr_t)row & 127)) & 127) / (int)sizeof(T);
        head = head < V ? head : V;
        nfull = (V - head) / E;
        edge = V - nfull * E;
    }
    __device__ __forceinline__ long piece(int i) const { return (long)i * E + head; }
    __device__ __forceinline__ int edge_col(int t) const { return t < head ? t : nfull * E + t; }
};

template <typename T, int NT>
__device__ __forceinline__ void zero_row(T* d, int V, bool stream) {
    const Cut<T> cut(d, V);
    float o[Piece<T>::E];
#pragma unroll
    for (int e = 0; e < Piece<T>::E; ++e) o[e] = 0.f;
    for (int i = threadIdx.x; i < cut.nfull; i += NT) put_piece<T>(d + cut.piece(i), o, stream);
    if ((int)threadIdx.x < cut.edge) Piece<T>::put(d + cut.edge_col(threadIdx.x), 0.f);
}

// Pieces threadIdx.x, threadIdx.x + NT, ... of a row; what lies past its last piece reads as -inf.
template <typename T, int NT, int NV>
__device__ __forceinline__ void load_all(Piece<T> (&q)[NV], const T* x, const Cut<T>& cut, bool stream) {
#pragma unroll
    for (int j = 0; j < NV; ++j) q[j].fill(-INFINITY);
    if (stream) {
#pragma unroll
        for (int j = 0; j < NV; ++j)
            if ((int)threadIdx.x + j * NT < cut.nfull) q[j].load_stream(x + cut.piece(threadIdx.x + j * NT));
    } else {
#pragma unroll
        for (int j = 0; j < NV; ++j)
            if ((int)threadIdx.x + j * NT < cut.nfull) q[j].load(x + cut.piece(threadIdx.x + j * NT));
    }
}

// One workgroup per row, the row in registers: NV 16-byte pieces per thread and one single element of its ragged ends.
// Rows of more than 1024 pieces take 1024 threads, two rows per CU: 10496 x 50000 bf16 413 us all live, 314 us half padding;
// with 512 threads and three rows per CU 398 and 328 us (a padded batch is the ordinary one), 256 and 640 in between.
template <typename T, int NT, int NV>
__global__ __launch_bounds__(NT) void row_kernel(const RowArgs a) {
    constexpr int E = Piece<T>::E, NW = NT / 64;
    __shared__ float red_m[NW], red_z[NW];
    __shared__ float coef_s;
    const long row = blockIdx.x;
    const float w = a.weight ? a.weight[row] : 1.f;
    T* d = a.dlogits ? (T*)a.dlogits + row * a.ldd : nullptr;
    if (w == 0.f) {
        if (d) zero_row<T, NT>(d, a.V, a.stream_out);
        if (threadIdx.x == 0) masked_scalars(a, row);
        return;
    }
    const float inv_tau = a.dyn_inv_tau ? a.dyn_inv_tau[0] : a.inv_tau;
    const T* x = (const T*)a.logits + row * a.ld;
    const Cut<T> cut(x, a.V);
    const bool has_edge = (int)threadIdx.x < cut.edge;
    const int ec = cut.edge_col(threadIdx.x);
    RowScalars rs;
    if (threadIdx.x == 0) rs.load<T>(a, row);
    Piece<T> q[NV];
    load_all<T, NT, NV>(q, x, cut, a.stream_in);
    const float xe = has_edge ? Piece<T>::one(x + ec) : -INFINITY;
    float m = xe;
#pragma unroll
    for (int j = 0; j < NV; ++j) m = piece_max(q[j], m);
    m = wave_max(m);
    if ((threadIdx.x & 63) == 0) red_m[threadIdx.x >> 6] = m;
    __syncthreads();
    m = red_m[0];
#pragma unroll
    for (int i = 1; i < NW; ++i) m = fmaxf(m, red_m[i]);
    keep_packed<T, NV>(q);
    const float c2 = inv_tau * LOG2E;
    const float pe = fast_exp2((xe - m) * c2);
    float part[E];
#pragma unroll
    for (int e = 0; e < E; ++e) part[e] = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int e = 0; e < E; ++e) part[e] += fast_exp2((q[j].get(e) - m) * c2);
    float z = pe;
#pragma unroll
    for (int e = 0; e < E; ++e) z += part[e];
    z = wave_sum(z);
    if ((threadIdx.x & 63) == 0) red_z[threadIdx.x >> 6] = z;
    __syncthreads();
    z = 0.f;
#pragma unroll
    for (int i = 0; i < NW; ++i) z += red_z[i];
    z = total(z);
    float g = 0.f;
    if (threadIdx.x == 0 && a.advantage) g = rs.slope(a, w, inv_tau, m, z);
    if (!d) {
        if (threadIdx.x == 0) rs.write(a, row, w, inv_tau, m, z, g);
        return;
    }
    if (threadIdx.x == 0) coef_s = g;
    __syncthreads();
    keep_packed<T, NV>(q);
    const float c = coef_s * inv_tau, cz = -c / z;
    const int64_t t64 = a.target[row];
    const int t = t64 >= 0 && t64 < a.V ? (int)t64 : -1;
    const int tp = t < cut.head ? -1 : (t - cut.head) / E, te = t - cut.head - tp * E;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int i = threadIdx.x + j * NT;
        if (i < cut.nfull) {
            float o[E];
#pragma unroll
            for (int e = 0; e < E; ++e) o[e] = fast_exp2((q[j].get(e) - m) * c2) * cz;
            if (i == tp) {
#pragma unroll
                for (int e = 0; e < E; ++e) o[e] += e == te ? c : 0.f;
            }
            put_piece<T>(d + cut.piece(i), o, a.stream_out);
        }
    }
    if (has_edge) Piece<T>::put(d + ec, pe * cz + (ec == t ? c : 0.f));
    if (threadIdx.x == 0) rs.write(a, row, w, inv_tau, m, z, g);
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
    const Cut<T> cut(x, a.V);
    constexpr int U = 4;  // pieces in flight
    float m = -INFINITY, z = 0.f;
    for (int i0 = threadIdx.x; i0 < cut.nfull; i0 += U * NT) {
        Piece<T> q[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (i0 + u * NT < cut.nfull)
                q[u].load(x + cut.piece(i0 + u * NT));
            else
                q[u].fill(-INFINITY);
        }
        float mx = m;
#pragma unroll
        for (int u = 0; u < U; ++u) mx = piece_max(q[u], mx);
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
    const float xe = (int)threadIdx.x < cut.edge ? Piece<T>::one(x + cut.edge_col(threadIdx.x)) : -INFINITY;
    const float mb = block_max<NT>(fmaxf(m, xe), red);
    const float mine = m == -INFINITY && z == 0.f ? 0.f : z * fast_exp2((m - mb) * c2);
    z = total(block_sum<NT>(mine + fast_exp2((xe - mb) * c2), red));
    if (threadIdx.x == 0) {
        RowScalars rs;
        rs.load<T>(a, row);
        rs.write(a, row, w, inv_tau, mb, z, a.advantage ? rs.slope(a, w, inv_tau, mb, z) : 0.f);
    }
}

__device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

// out[0] = scale * sum v by one workgroup of NT threads: a fixed order, in 64 bits (a loss is a sum of terms of both signs).
template <int NT>
__device__ __forceinline__ void sum64(const double* __restrict__ v, long n, double scale, float* __restrict__ out) {
    __shared__ double red[NT / 64];
    double s = 0.0;
    for (long i0 = threadIdx.x; i0 < n; i0 += 8 * NT) {
        double q[8];  // loads in flight
#pragma unroll
        for (int u = 0; u < 8; ++u) q[u] = i0 + u * NT < n ? v[i0 + u * NT] : 0.0;
#pragma unroll
        for (int u = 0; u < 8; ++u) s += q[u];
    }
    s = wave_sum64(s);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        double t = 0.0;
#pragma unroll
        for (int i = 0; i < NT / 64; ++i) t += red[i];
        out[0] = (float)(t * scale);
    }
}

constexpr int ROWS_SUM_NT = 1024, GRAD_NT = 256;
template <int NT>
__global__ __launch_bounds__(NT) void sum64_kernel(const double* __restrict__ v, long n, double scale,
                                                   float* __restrict__ out) {
    sum64<NT>(v, n, scale, out);
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
    bool stream_out;
    int chunks;  // workgroups per row
    const double* pair_loss;  // nullable: one workgroup more, the first, forms the mean of these
    int pairs;
    float* loss;
};

// grid: row by row, `chunks` workgroups each, of U pieces per thread and no loop. Many short workgroups stream better than
// few long ones: they keep the addresses in flight together. The preference loss has its mean formed here
// as well, one launch less (32 pairs of 21 x 20001 fp32: 50.0 -> 48.5 us; 64 of 41 x 50000 bf16: 203 -> 201).
template <typename T, int NT, int U>
__global__ __launch_bounds__(NT) void row_grad_kernel(const GradArgs a) {
    constexpr int E = Piece<T>::E;
    const unsigned more = a.pair_loss ? 1 : 0, b = blockIdx.x - more;
    if (blockIdx.x < more) {
        sum64<NT>(a.pair_loss, a.pairs, 1.0 / a.pairs, a.loss);
        return;
    }
    const int chunk = b % a.chunks;
    // backwards: the statistics' pass has left the last rows in the cache
    const long row = (gridDim.x - more) / a.chunks - 1 - b / a.chunks;
    T* d = (T*)a.dlogits + row * a.ldd;
    const Cut<T> cut(d, a.V);
    const int i0 = chunk * (NT * U) + threadIdx.x;
    const bool has_edge = chunk == 0 && (int)threadIdx.x < cut.edge;
    if (a.weight && a.weight[row] == 0.f) {
        float o[E];
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] = 0.f;
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (i0 + u * NT < cut.nfull) put_piece<T>(d + cut.piece(i0 + u * NT), o, a.stream_out);
        if (has_edge) Piece<T>::put(d + cut.edge_col(threadIdx.x), 0.f);
        return;
    }
    const T* x = (const T*)a.logits + row * a.ld;
    Piece<T> q[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
        if (i0 + u * NT < cut.nfull) q[u].load(x + cut.piece(i0 + u * NT));
    const int ec = cut.edge_col(threadIdx.x);
    const float xe = has_edge ? Piece<T>::one(x + ec) : 0.f;
    const float inv_tau = a.dyn_inv_tau ? a.dyn_inv_tau[0] : a.inv_tau;
    const float c2 = inv_tau * LOG2E, m = a.stats[2 * row], z = a.stats[2 * row + 1];
    const int64_t t64 = a.target[row];
    const int t = t64 >= 0 && t64 < a.V ? (int)t64 : -1;
    const float c = t < 0 ? NAN : a.coef[row] * (a.scale ? a.scale[0] : 1.f) * inv_tau, cz = -c / z;
    const int tp = t < cut.head ? -1 : (t - cut.head) / E, te = t - cut.head - tp * E;
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int i = i0 + u * NT;
        if (i < cut.nfull) {
            float o[E];
#pragma unroll
            for (int e = 0; e < E; ++e) o[e] = fast_exp2((q[u].get(e) - m) * c2) * cz;
            if (i == tp) {
#pragma unroll
                for (int e = 0; e < E; ++e) o[e] += e == te ? c : 0.f;
            }
            put_piece<T>(d + cut.piece(i), o, a.stream_out);
        }
    }
    if (has_edge) Piece<T>::put(d + ec, fast_exp2((xe - m) * c2) * cz + (ec == t ? c : 0.f));
}

// Two waves per pair (p chosen, P + p rejected): the sentences' log-probabilities, the margin, the loss, and the gradient
// every row of the two sentences takes into its logits. A few pairs share a workgroup, which then sums the loss as well (one
// launch less: 2 us of 26 for a single pair); more pairs take a workgroup each (64 pairs of 41 tokens in one: 20 us longer).
constexpr int PAIR_W = 8, PAIR_NT = 128 * PAIR_W;
__global__ __launch_bounds__(PAIR_NT) void pair_kernel(const double* __restrict__ lp64, const float* __restrict__ weight,
                                                       const float* __restrict__ ref, int p0, int P, int T, double beta,
                                                       double smooth, float* __restrict__ seq_logp,
                                                       float* __restrict__ margin, double* __restrict__ pair_loss,
                                                       float* __restrict__ coef, float* __restrict__ loss) {
    __shared__ double S[PAIR_W][2], sum[PAIR_W];
    const int slot = threadIdx.x >> 7, side = threadIdx.x >> 6 & 1, lane = threadIdx.x & 63;
    const int p = p0 + blockIdx.x * (blockDim.x >> 7) + slot;  // (the grids cover the pairs exactly)
    const long seq = (long)side * P + p;
    double s = 0.0;
    for (int t = lane; t < T; t += 64) s += lp64[seq * T + t];
    s = wave_sum64(s);
    if (lane == 0) {
        S[slot][side] = s - (double)ref[seq];
        seq_logp[seq] = (float)s;
    }
    __syncthreads();
    const double mg = beta * (S[slot][0] - S[slot][1]);
    // log sig(m) = min(m, 0) - log1p(exp(-|m|)); sig(-m) = exp(-|m|) or 1 over 1 + exp(-|m|)
    const double ex = exp(-fabs(mg)), l1 = log1p(ex);
    const double pos = mg >= 0.0 ? 1.0 / (1.0 + ex) : ex / (1.0 + ex);
    const double neg = mg >= 0.0 ? ex / (1.0 + ex) : 1.0 / (1.0 + ex);
    const double up = -(beta / (double)P) * ((1.0 - smooth) * neg - smooth * pos);
    if ((threadIdx.x & 127) == 0) {
        double ls = (1.0 - smooth) * (fmin(mg, 0.0) - l1);
        // left out without smoothing: log sig(-m) is -inf where the model cannot produce the rejected sentence, and such a
        // pair has a loss of 0
        if (smooth > 0.0) ls += smooth * (fmin(-mg, 0.0) - l1);
        margin[p] = (float)mg;
        pair_loss[p] = sum[slot] = mg != mg ? mg : -ls;  // (fmin drops a NaN margin; the loss keeps it)
    }
    if (coef)
        for (int t = lane; t < T; t += 64) coef[seq * T + t] = (float)((side ? -up : up) * (double)weight[seq * T + t]);
    if (!loss) return;  // summed elsewhere: this is not the only workgroup
    __syncthreads();
    if (threadIdx.x == 0) {
        double t = 0.0;
        for (int i = 0; i < P; ++i) t += sum[i];
        loss[0] = (float)(t / (double)P);
    }
}

// The rows from r0 on.
template <typename T>
RowArgs rows_from(RowArgs a, int64_t r0) {
    a.logits = (const T*)a.logits + r0 * a.ld;
    a.target += r0;
    if (a.weight) a.weight += r0;
    if (a.logp) a.logp += r0;
    if (a.lp64) a.lp64 += r0;
    if (a.stats) a.stats += 2 * r0;
    if (a.advantage) a.advantage += r0;
    if (a.old_logp) a.old_logp += r0;
    if (a.ref_logp) a.ref_logp += r0;
    if (a.row_loss) a.row_loss += r0;
    if (a.coef) a.coef += r0;
    if (a.dlogits) a.dlogits = (T*)a.dlogits + r0 * a.ldd;
    return a;
}

constexpr int64_t GRID_THREADS = 1LL << 31;  // threads of one launch (the hardware counts them in 32 bits)

template <typename T, int NT, int NV>
int launch_row(hipStream_t s, const RowArgs& a, int64_t M) {
    for (int64_t r = 0; r < M; r += GRID_THREADS / NT) {
        const int64_t n = M - r < GRID_THREADS / NT ? M - r : GRID_THREADS / NT;
        hipLaunchKernelGGL((row_kernel<T, NT, NV>), dim3((unsigned)n), dim3(NT), 0, s, rows_from<T>(a, r));
        CGN_LAUNCH_CHECK();
    }
    return CGN_OK;
}

template <typename T>
int launch_grad(hipStream_t s, GradArgs g, int64_t M) {
    constexpr int NT = GRAD_NT, U = 2;
    g.chunks = cgn_cdiv(g.V, (long)Piece<T>::E * NT * U);
    // whole rows per launch, as many as a grid holds
    const int64_t most = (GRID_THREADS / NT - 1) / g.chunks;
    for (int64_t r = M; r > 0; r -= most) {
        const int64_t n = r < most ? r : most, r0 = r - n;
        GradArgs b = g;
        b.logits = (const T*)g.logits + r0 * g.ld;
        b.dlogits = (T*)g.dlogits + r0 * g.ldd;
        b.target += r0;
        if (b.weight) b.weight += r0;
        b.stats += 2 * r0;
        b.coef += r0;
        const int64_t blocks = n * g.chunks + (g.pair_loss ? 1 : 0);
        hipLaunchKernelGGL((row_grad_kernel<T, NT, U>), dim3((unsigned)blocks), dim3(NT), 0, s, b);
        CGN_LAUNCH_CHECK();
        g.pair_loss = nullptr;
    }
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
    if (n <= 1024 * 2) return launch_row<T, 1024, 2>(s, a, M);
    if (n <= 1024 * 3) return launch_row<T, 1024, 3>(s, a, M);
    if (n <= 1024 * 4) return launch_row<T, 1024, 4>(s, a, M);
    if (n <= 1024 * 5) return launch_row<T, 1024, 5>(s, a, M);
    if (n <= 1024 * 7) return launch_row<T, 1024, 7>(s, a, M);
    if (n <= 1024 * 10) return launch_row<T, 1024, 10>(s, a, M);
    if (n <= 1024 * 13) return launch_row<T, 1024, 13>(s, a, M);
    if (n <= 1024 * 16) return launch_row<T, 1024, 16>(s, a, M);
    *done = false;
    for (int64_t r = 0; r < M; r += GRID_THREADS / 1024) {
        const int64_t m = M - r < GRID_THREADS / 1024 ? M - r : GRID_THREADS / 1024;
        hipLaunchKernelGGL((row_stream_kernel<T, 1024>), dim3((unsigned)m), dim3(1024), 0, s, rows_from<T>(a, r));
        CGN_LAUNCH_CHECK();
    }
    return CGN_OK;
}

int run_rows(hipStream_t s, const RowArgs& a, int64_t M, bool bf16, bool* done) {
    return bf16 ? launch_rows<Bf16>(s, a, M, done) : launch_rows<float>(s, a, M, done);
}

int run_grad(hipStream_t s, const GradArgs& g, int64_t M, bool bf16) {
    return bf16 ? launch_grad<Bf16>(s, g, M) : launch_grad<float>(s, g, M);
}

template <int NT>
int run_sum(hipStream_t s, const double* v, int64_t n, double scale, float* out) {
    hipLaunchKernelGGL(sum64_kernel<NT>, dim3(1), dim3(NT), 0, s, v, (long)n, scale, out);
    CGN_LAUNCH_CHECK();
    return CGN_OK;
}

bool base_ok(const cgn_token_rows* r) {
    return r && r->M >= 0 && r->M <= 0x7fffffff && r->V > 0 && r->ld >= r->V &&
           (r->dyn_inv_tau || r->inv_tau > 0.f) && (r->M == 0 || (r->logits && r->target)) &&
           (uintptr_t)r->logits % (r->bf16 ? 2 : 4) == 0;
}

// (element-aligned: what the row kernels' accesses take)
bool dest_ok(const cgn_token_rows* r, const void* d, int64_t ldd) {
    return ldd >= r->V && (uintptr_t)d % (r->bf16 ? 2 : 4) == 0;
}

bool streams(const cgn_token_rows* r) { return r->M * r->V * (r->bf16 ? 2 : 4) >= STREAM_BYTES; }

RowArgs row_args(const cgn_token_rows* r) {
    RowArgs a = {};
    a.logits = r->logits;
    a.ld = r->ld;
    a.target = r->target;
    a.weight = r->weight;
    a.V = r->V;
    a.inv_tau = r->inv_tau;
    a.dyn_inv_tau = r->dyn_inv_tau;
    return a;  // (logits that a second pass will read stay in the caches)
}

int row_gradient(hipStream_t s, const cgn_token_rows* r, const float* stats, const float* coef, const float* scale,
                 void* dlogits, int64_t ldd, const double* pair_loss = nullptr, int pairs = 0, float* loss = nullptr) {
    GradArgs g = {r->logits, r->ld, r->target, r->weight, r->V, r->inv_tau, r->dyn_inv_tau, stats, coef, scale, dlogits,
                  ldd, streams(r), 0, pair_loss, pairs, loss};
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
    CGN_CHECK_ARG(base_ok(r) && dest_ok(r, dlogits, ldd));
    if (r->M == 0) return CGN_OK;
    CGN_CHECK_ARG(stats && coef && dlogits);
    return row_gradient((hipStream_t)stream, r, stats, coef, scale, dlogits, ldd);
}

extern "C" int cgn_policy_loss(void* stream, const cgn_token_rows* r, const float* advantage, const float* old_logp,
                               const float* ref_logp, float clip_lo, float clip_hi, float kl_coef, float* loss,
                               float* logp, float* stats, float* coef, void* dlogits, int64_t ldd, void* workspace,
                               int64_t workspace_bytes) {
    CGN_CHECK_ARG(base_ok(r) && loss && clip_lo >= 0.f && clip_hi >= 0.f && (!dlogits || dest_ok(r, dlogits, ldd)));
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
        a.stream_in = a.stream_out = dlogits && streams(r);
        bool done;
        int rc = run_rows(s, a, r->M, r->bf16 != 0, &done);
        if (rc == CGN_OK && dlogits && !done) rc = row_gradient(s, r, stats, coef, nullptr, dlogits, ldd);
        if (rc != CGN_OK) return rc;
    }
    return run_sum<ROWS_SUM_NT>(s, row_loss, r->M, 1.0, loss);
}

extern "C" int cgn_preference_loss(void* stream, const cgn_token_rows* r, int32_t T, const float* ref_logp, double beta,
                                   double label_smoothing, float* loss, float* margin, float* seq_logp, float* stats,
                                   float* coef, void* dlogits, int64_t ldd, void* workspace, int64_t workspace_bytes) {
    CGN_CHECK_ARG(base_ok(r) && T > 0 && r->M > 0 && r->M % (2 * (int64_t)T) == 0 && r->weight);
    CGN_CHECK_ARG(beta > 0.0 && label_smoothing >= 0.0 && label_smoothing < 0.5);
    CGN_CHECK_ARG(ref_logp && loss && margin && seq_logp && (!dlogits || dest_ok(r, dlogits, ldd)));
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
    const bool few = P <= PAIR_W;
    for (int64_t p0 = 0; p0 < P; p0 += GRID_THREADS / 128) {
        const int64_t n = P - p0 < GRID_THREADS / 128 ? P - p0 : GRID_THREADS / 128;
        hipLaunchKernelGGL(pair_kernel, dim3(few ? 1 : (unsigned)n), dim3(few ? 128 * P : 128), 0, s, lp64, r->weight,
                           ref_logp, (int)p0, P, T, beta, label_smoothing, seq_logp, margin, pair_loss, coef,
                           few ? loss : nullptr);
        CGN_LAUNCH_CHECK();
    }
    if (dlogits) return row_gradient(s, r, stats, coef, nullptr, dlogits, ldd, few ? nullptr : pair_loss, P, loss);
    // (with as many threads as sum it in the gradient's launch: the same order, the same bits)
    return few ? CGN_OK : run_sum<GRAD_NT>(s, pair_loss, P, 1.0 / P, loss);
}
