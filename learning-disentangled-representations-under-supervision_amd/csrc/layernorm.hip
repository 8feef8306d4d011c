// Layer norm over the last axis of [R, C] rows, forward and backward (hip/ops.py layer_norm_fwd / layer_norm_bwd).
//   mu = mean(x), var = mean((x - mu)^2), r = 1 / sqrt(var + eps), xh = (x - mu) r, y = xh w + b
//   g = dy w,  dx = r (g - mean(g) - xh mean(g xh)),  dw = sum over rows dy xh,  db = sum over rows dy
// HBM-bound (8 to 22 flops per element): every row is read once into registers and stays there for all its sums. A group
// of G lanes owns a row; each lane holds NV 16-byte pieces of it. 83968 x 1024 bf16: forward 65 us (5.3 TB/s), backward
// 98 to 101 us (5.1 to 5.3 TB/s); fp32 rows of 300 to 4096 elements run at 4.7 to 5.6 TB/s, bf16 rows of odd width at 4.2 to
// 4.8 forward and 3.4 to 3.8 backward: a row's pieces start at its first element, so a wave's accesses there begin inside a
// 128-byte line (token_loss.hip cuts its rows at the lines).
#include "rows.h"

namespace {

using namespace cgn_rows;

// Sums over the row's group: inside the wave with shuffles, over a whole workgroup through LDS. Calls in a row alternate
// between two buffers `red`, so that one barrier each is enough: whoever writes a buffer again has passed the barrier of the
// call in between, behind which nobody reads it any more.
template <int NT, int G, int K>
__device__ __forceinline__ void row_sums(float (&s)[K], float* red) {
    static_assert(G <= 64 || G == NT, "a group is part of a wave or the whole workgroup");
#pragma unroll
    for (int k = 0; k < K; ++k) s[k] = group_sum<(G < 64 ? G : 64)>(s[k]);
    if constexpr (G > 64) {
        if ((threadIdx.x & 63) == 0) {
#pragma unroll
            for (int k = 0; k < K; ++k) red[(threadIdx.x >> 6) * K + k] = s[k];
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < K; ++k) {
            s[k] = 0.f;
#pragma unroll
            for (int w = 0; w < G / 64; ++w) s[k] += red[w * K + k];
        }
    }
}

// A row as its group holds it: lane l has the pieces l, l + G, ... of the C / E whole ones, and lane l < C % E the single
// element behind them. What a lane does not have reads as zero.
template <typename T, int NV, int G>
struct Row {
    Piece<T> q[NV];
    float t;
    __device__ __forceinline__ void load(const T* row, int lane, int nfull, int rem, bool stream) {
        constexpr int E = Piece<T>::E;
#pragma unroll
        for (int j = 0; j < NV; ++j) q[j].fill(0.f);
        if (stream) {
#pragma unroll
            for (int j = 0; j < NV; ++j)
                if (lane + j * G < nfull) q[j].load_stream(row + (long)(lane + j * G) * E);
        } else {
#pragma unroll
            for (int j = 0; j < NV; ++j)
                if (lane + j * G < nfull) q[j].load(row + (long)(lane + j * G) * E);
        }
        t = lane < rem ? Piece<T>::one(row + nfull * E + lane) : 0.f;
    }
};

// The group's share of a parameter vector (null: `none` everywhere), laid out like a Row.
template <int NV, int E, int G>
struct Param {
    float v[NV][E], t;
    __device__ __forceinline__ void load(const float* w, float none, int lane, int nfull, int rem) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int i = lane + j * G;
#pragma unroll
            for (int e = 0; e < E; ++e) v[j][e] = none;
            if (w && i < nfull) {
#pragma unroll
                for (int h = 0; h < E / 4; ++h) {
                    Piece<float> p;
                    p.load(w + (long)i * E + 4 * h);
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[j][4 * h + e] = p.get(e);
                }
            }
        }
        t = w && lane < rem ? w[nfull * E + lane] : none;
    }
};

// One row per group. Two sums are taken: the mean, then (both at once) the sums of d = x - mean and d^2; the first of them
// is what the mean's own rounding left over, so rows whose mean is large against their spread keep fp32 accuracy.
template <typename T, int NT, int G, int NV>
__global__ __launch_bounds__(NT) void layer_norm_fwd_kernel(const T* x, long ldx, long R, int C,
                                                            const float* __restrict__ w, const float* __restrict__ b,
                                                            float eps, T* y, long ldy, float* __restrict__ mean,
                                                            float* __restrict__ rstd, bool stream) {
    constexpr int E = Piece<T>::E;
    __shared__ float red[2][NT / 64 * 2];
    const int lane = threadIdx.x % G;
    const int nfull = C / E, rem = C % E;
    const float inv_c = 1.f / (float)C;
    Param<NV, E, G> pw, pb;
    pw.load(w, 1.f, lane, nfull, rem);
    pb.load(b, 0.f, lane, nfull, rem);
    for (long r = (long)blockIdx.x * (NT / G) + threadIdx.x / G; r < R; r += (long)gridDim.x * (NT / G)) {
        Row<T, NV, G> row;
        row.load(x + r * ldx, lane, nfull, rem, stream);
        float s1[1] = {row.t};
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int e = 0; e < E; ++e) s1[0] += row.q[j].get(e);
        row_sums<NT, G, 1>(s1, red[0]);
        const float mu = s1[0] * inv_c;
        float s2[2] = {0.f, 0.f};
#pragma unroll
        for (int j = 0; j < NV; ++j)
            if (lane + j * G < nfull) {
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const float d = row.q[j].get(e) - mu;
                    s2[0] += d;
                    s2[1] += d * d;
                }
            }
        if (lane < rem) {
            const float d = row.t - mu;
            s2[0] += d;
            s2[1] += d * d;
        }
        row_sums<NT, G, 2>(s2, red[1]);
        const float off = s2[0] * inv_c;
        const float v = s2[1] * inv_c - off * off;
        const float rs = 1.f / sqrtf((v < 0.f ? 0.f : v) + eps);  // (a NaN stays one)
        if (lane == 0) {
            mean[r] = mu + off;
            rstd[r] = rs;
        }
        T* yr = y + r * ldy;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int i = lane + j * G;
            if (i < nfull) {
                float o[E];
#pragma unroll
                for (int e = 0; e < E; ++e) o[e] = ((row.q[j].get(e) - mu) - off) * rs * pw.v[j][e] + pb.v[j][e];
                if (stream)
                    Piece<T>::store_stream(yr + (long)i * E, o);
                else
                    Piece<T>::store(yr + (long)i * E, o);
            }
        }
        if (lane < rem) Piece<T>::put(yr + nfull * E + lane, ((row.t - mu) - off) * rs * pw.t + pb.t);
    }
}

// Backward. Every group walks rows r, r + step, ...; its columns' shares of dw and db stay in registers and leave the
// workgroup once, as one [2][C] row of `part` per workgroup (fixed order: no atomics, the same bits every run). The next
// row's loads are in flight beside a row's sums: few waves fit beside the sums (83968 x 1024 bf16 at 8 waves per CU 117 us,
// at 12 101 us; fp32 rows of 1024 are as fast at 8, 54 us).
// dx may be dy's or x's own buffer: a row is in registers before anything of it is written.
template <typename T, int NT, int G, int NV>
__global__ __launch_bounds__(NT) void layer_norm_bwd_kernel(const T* dy, long lddy, const T* x, long ldx, long R, int C,
                                                            const float* __restrict__ w, const float* __restrict__ mean,
                                                            const float* __restrict__ rstd, T* dx, long lddx,
                                                            float* __restrict__ part, float* dw, float* db, float beta,
                                                            bool stream) {
    constexpr int E = Piece<T>::E;
    constexpr int GROUPS = NT / G;
    __shared__ float red[2][NT / 64 * 3];
    int turn = 0;
    const int lane = threadIdx.x % G, grp = threadIdx.x / G;
    const int nfull = C / E, rem = C % E;
    const float inv_c = 1.f / (float)C;
    Param<NV, E, G> pw;
    pw.load(w, 1.f, lane, nfull, rem);
    float aw[NV][E], ab[NV][E], awt = 0.f, abt = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int e = 0; e < E; ++e) aw[j][e] = ab[j][e] = 0.f;
    long r = (long)blockIdx.x * GROUPS + grp;
    const long step = (long)gridDim.x * GROUPS;
    Row<T, NV, G> nx, nd;
    float nmu = 0.f, nrs = 0.f;
    if (r < R) {
        nx.load(x + r * ldx, lane, nfull, rem, stream);
        nd.load(dy + r * lddy, lane, nfull, rem, stream);
        nmu = mean[r], nrs = rstd[r];
    }
    for (; r < R; r += step) {
        Row<T, NV, G> qx = nx, qd = nd;
        const float mu = nmu, rs = nrs;
        if (r + step < R) {  // in flight beside this row's sums
            nx.load(x + (r + step) * ldx, lane, nfull, rem, stream);
            nd.load(dy + (r + step) * lddy, lane, nfull, rem, stream);
            nmu = mean[r + step], nrs = rstd[r + step];
        }
        // xh = x r - mu r up to a constant of the row, the rounding of mu and of mu r: the mean of xh, which is that
        // constant, is summed with g and g xh and taken out below
        const float nb = -mu * rs;
        float s[3] = {0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < NV; ++j)
            if (lane + j * G < nfull) {
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const float xh = fmaf(qx.q[j].get(e), rs, nb), g = qd.q[j].get(e) * pw.v[j][e];
                    s[0] += xh;
                    s[1] += g;
                    s[2] += g * xh;
                }
            }
        const float xht = lane < rem ? fmaf(qx.t, rs, nb) : 0.f, gt = qd.t * pw.t;
        s[0] += xht;
        s[1] += gt;
        s[2] += gt * xht;
        row_sums<NT, G, 3>(s, red[turn]);
        turn ^= 1;
        keep_packed<T, NV>(qx.q);
        keep_packed<T, NV>(qd.q);
        const float off = s[0] * inv_c, mg = s[1] * inv_c, mgx = s[2] * inv_c - mg * off;
        // dx = r g - (r mgx) (xh - off) - r mg
        const float cx = -rs * mgx, c0 = -rs * mg;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int i = lane + j * G;
            if (i < nfull) {
                float o[E];
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const float d = qd.q[j].get(e);
                    const float xh = fmaf(qx.q[j].get(e), rs, nb) - off;
                    aw[j][e] += d * xh;
                    ab[j][e] += d;
                    o[e] = fmaf(d * pw.v[j][e], rs, fmaf(xh, cx, c0));
                }
                if (dx && stream)
                    Piece<T>::store_stream(dx + r * lddx + (long)i * E, o);
                else if (dx)
                    Piece<T>::store(dx + r * lddx + (long)i * E, o);
            }
        }
        if (lane < rem) {
            awt += qd.t * (xht - off);
            abt += qd.t;
            if (dx) Piece<T>::put(dx + r * lddx + nfull * E + lane, fmaf(gt, rs, fmaf(xht - off, cx, c0)));
        }
    }
    if (!part && !dw && !db) return;
    // the workgroup's groups summed in a fixed order, one piece of every lane at a time through LDS
    const auto put = [&](int k, int c, float v) {
        if (part) {
            part[((long)blockIdx.x * 2 + k) * C + c] = v;
        } else if (float* o = k ? db : dw) {  // the only workgroup: nothing is left to be reduced
            o[c] = beta != 0.f ? v + beta * o[c] : v;
        }
    };
    __shared__ float rows[GROUPS][GROUPS > 1 ? G * E : 1];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
#pragma unroll
        for (int j = 0; j <= NV; ++j) {
            const int width = j < NV ? E : 1;            // (the last round: the single elements)
            const int col0 = j < NV ? j * G * E : nfull * E;
            const int cend = j < NV ? nfull * E : C;
            if constexpr (GROUPS == 1) {
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    if (e >= width) break;
                    const int c = col0 + lane * width + e;
                    const float v = j < NV ? (k ? ab[j < NV ? j : 0][e] : aw[j < NV ? j : 0][e]) : (k ? abt : awt);
                    if (c < cend) put(k, c, v);
                }
            } else {
                __syncthreads();
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    if (e >= width) break;
                    rows[grp][lane * width + e] =
                        j < NV ? (k ? ab[j < NV ? j : 0][e] : aw[j < NV ? j : 0][e]) : (k ? abt : awt);
                }
                __syncthreads();
                for (int c = threadIdx.x; c < G * width; c += NT) {
                    float t = 0.f;
#pragma unroll
                    for (int q = 0; q < GROUPS; ++q) t += rows[q][c];
                    if (col0 + c < cend) put(k, col0 + c, t);
                }
            }
        }
    }
}

// dw[c] = beta dw[c] + sum over the workgroups' rows of part, in a fixed order; db likewise. Summed in 64 bits, which costs
// no time behind these loads and halves the error (1280 x 825 fp32: 1.3e-7 -> 7e-8; 40000 x 600: 1.8e-7 -> 1.0e-7).
constexpr int LNF_NT = 1024;
__global__ __launch_bounds__(LNF_NT) void layer_norm_params_kernel(const float* __restrict__ part, int nb, int C,
                                                                   float beta, float* __restrict__ dw,
                                                                   float* __restrict__ db) {
    __shared__ double red[LNF_NT / 64][64];
    const int lane = threadIdx.x & 63, seg = threadIdx.x >> 6;
    const int c = blockIdx.x * 64 + lane;
    double t = 0.0;
    if (c < 2 * C) {
#pragma unroll 8
        for (int i = seg; i < nb; i += LNF_NT / 64) t += (double)part[(long)i * 2 * C + c];
    }
    red[seg][lane] = t;
    __syncthreads();
    if (seg == 0 && c < 2 * C) {
        double v = 0.0;
#pragma unroll
        for (int k = 0; k < LNF_NT / 64; ++k) v += red[k][lane];
        float* o = c < C ? dw : db;
        if (!o) return;
        o += c < C ? c : c - C;
        *o = (float)(beta != 0.f ? v + (double)beta * (double)*o : v);
    }
}

constexpr int LN_MAX_C = 8192;    // widest row that the groups below hold in registers
constexpr int LN_ALONE = 4;       // a backward pass of that many workgroups' rows is left to one
constexpr int LN_FWD_NB = 8192;   // workgroups of a forward pass at most: each with many rows behind one read of w and b

template <typename T, int NT, int G, int NV>
int launch_fwd(hipStream_t s, const void* x, int64_t ldx, int64_t R, int C, const float* w, const float* b, float eps,
               void* y, int64_t ldy, float* mean, float* rstd) {
    int64_t nb = (R + NT / G - 1) / (NT / G);
    if (nb > LN_FWD_NB) nb = LN_FWD_NB;
    hipLaunchKernelGGL((layer_norm_fwd_kernel<T, NT, G, NV>), dim3((unsigned)nb), dim3(NT), 0, s, (const T*)x, (long)ldx,
                       (long)R, C, w, b, eps, (T*)y, (long)ldy, mean, rstd,
                       R * C * (int64_t)sizeof(T) >= STREAM_BYTES);
    CGN_LAUNCH_CHECK();
    return CGN_OK;
}

// Workgroups of a backward pass. WAVES: waves per CU that the grid is made for; as many workgroups walk the rows, and
// leave a row of `part` each (more would only lengthen the reduction behind them). A variant of up to 128 registers has
// room for 16 waves, up to 168 for 12. Those that do not go by it: fp32 rows of up to 256 elements (78 to 80 registers,
// room for 24, get 16), of 513 to 1024 (157 registers, room for 12, get 8: as fast) and of 1025 to 2048 (112, room for
// 16, get 12), bf16 rows of 1025 to 2048 (103, room for 16, get 12); and fp32 rows of 2049 to 4096, whose 130 registers
// leave room for one workgroup of 8 waves where the grid is made for two, which makes two rounds of it. From LN_ALONE
// workgroups' rows on a group starts with one row only: at 1280 x 825 fp32 `part` then is half the size of x, and the
// two launches take 7.3 and 4.2 us. A few rows take one workgroup and one launch, with no reduction: at 10 x 800 fp32
// (three workgroups' rows) a call from Python takes 14 us instead of 18, in a graph 6.7 instead of 6.4; at 32 x 800
// (eight) it would be 12.4 instead of 6.5 in a graph.
template <int NT, int G, int WAVES>
int64_t bwd_blocks(int64_t R) {
    const int64_t per = NT / G, nb = (R + per - 1) / per, most = 256 * WAVES * 64 / NT;
    return nb <= LN_ALONE ? (nb > 0) : nb > most ? most : nb;
}

template <typename T, int NT, int G, int NV, int WAVES>
int launch_bwd(hipStream_t s, const void* dy, int64_t lddy, const void* x, int64_t ldx, int64_t R, int C, const float* w,
               const float* mean, const float* rstd, void* dx, int64_t lddx, float* dw, float* db, float beta,
               float* part, int64_t part_bytes, int64_t* need) {
    const int64_t nb = bwd_blocks<NT, G, WAVES>(R);
    const bool params = dw || db, alone = nb == 1;
    if (need) {
        *need = alone ? 0 : nb * 2 * C * 4;
        return CGN_OK;
    }
    if (params && !alone && nb * 2 * C * 4 > part_bytes) return CGN_ERR_WORKSPACE;
    // the two are written by threads that do not know of each other
    if (dw && db && (uintptr_t)dw < (uintptr_t)(db + C) && (uintptr_t)db < (uintptr_t)(dw + C)) return CGN_ERR_INVALID_ARG;
    if (nb > 0) {
        hipLaunchKernelGGL((layer_norm_bwd_kernel<T, NT, G, NV>), dim3((unsigned)nb), dim3(NT), 0, s, (const T*)dy,
                           (long)lddy, (const T*)x, (long)ldx, (long)R, C, w, mean, rstd, (T*)dx, (long)lddx,
                           params && !alone ? part : nullptr, dw, db, beta, R * C * (int64_t)sizeof(T) >= STREAM_BYTES);
        CGN_LAUNCH_CHECK();
    }
    if (params && !alone) {
        hipLaunchKernelGGL(layer_norm_params_kernel, dim3(cgn_cdiv(2L * C, 64)), dim3(LNF_NT), 0, s, part, (int)nb, C, beta,
                           dw, db);
        CGN_LAUNCH_CHECK();
    }
    return CGN_OK;
}

// The narrowest group whose lanes hold the row in a few pieces: narrow rows share a wave, wide ones take a workgroup.
template <typename T>
int norm_fwd(hipStream_t s, const void* x, int64_t ldx, int64_t R, int C, const float* w, const float* b, float eps,
             void* y, int64_t ldy, float* mean, float* rstd) {
    const int n = cgn_cdiv(C, Piece<T>::E);
#define LN_FWD(NT, G, NV) return launch_fwd<T, NT, G, NV>(s, x, ldx, R, C, w, b, eps, y, ldy, mean, rstd)
    if (n <= 8) LN_FWD(256, 8, 1);
    if (n <= 16) LN_FWD(256, 16, 1);
    if (n <= 32) LN_FWD(256, 32, 1);
    if (n <= 64) LN_FWD(256, 64, 1);
    if (n <= 128) LN_FWD(256, 64, 2);
    if constexpr (Piece<T>::E == 4) {
        if (n <= 256) LN_FWD(256, 64, 4);
    } else {
        if (n <= 256) LN_FWD(256, 256, 1);
    }
    if (n <= 512) LN_FWD(256, 256, 2);
    if constexpr (Piece<T>::E == 4) {
        if (n <= 1024) LN_FWD(256, 256, 4);
        LN_FWD(1024, 1024, 2);
    } else {
        LN_FWD(1024, 1024, 1);
    }
#undef LN_FWD
}

// A lane's share of a row is 4 to 16 elements: with gradient, weight, the two sums and the next row's loads 78 to 157
// registers. The widest fp32 rows (4097 to 8192 elements, 1024 threads) are held to 128 and spill 12 bytes a lane.
template <typename T>
int norm_bwd(hipStream_t s, const void* dy, int64_t lddy, const void* x, int64_t ldx, int64_t R, int C, const float* w,
             const float* mean, const float* rstd, void* dx, int64_t lddx, float* dw, float* db, float beta, float* part,
             int64_t part_bytes, int64_t* need) {
    const int n = cgn_cdiv(C, Piece<T>::E);
#define LN_BWD(NT, G, NV, WAVES)                                                                                       \
    return launch_bwd<T, NT, G, NV, WAVES>(s, dy, lddy, x, ldx, R, C, w, mean, rstd, dx, lddx, dw, db, beta, part,     \
                                           part_bytes, need)
    if (n <= 8) LN_BWD(512, 8, 1, 16);
    if (n <= 16) LN_BWD(512, 16, 1, 16);
    if (n <= 32) LN_BWD(512, 32, 1, 16);
    if (n <= 64) LN_BWD(512, 64, 1, 16);
    if constexpr (Piece<T>::E == 4) {
        if (n <= 128) LN_BWD(512, 64, 2, 16);
        if (n <= 256) LN_BWD(256, 64, 4, 8);
        if (n <= 512) LN_BWD(256, 256, 2, 12);
        if (n <= 1024) LN_BWD(512, 512, 2, 16);
        LN_BWD(1024, 1024, 2, 16);
    } else {
        if (n <= 128) LN_BWD(256, 64, 2, 12);
        if (n <= 256) LN_BWD(256, 256, 1, 12);
        if (n <= 512) LN_BWD(512, 512, 1, 16);
        LN_BWD(1024, 1024, 1, 16);
    }
#undef LN_BWD
}

}  // namespace

extern "C" int cgn_layer_norm_fwd(void* stream, const void* x, int64_t ldx, int64_t R, int32_t C, int32_t bf16,
                                  const float* weight, const float* bias, float eps, void* y, int64_t ldy, float* mean,
                                  float* rstd) {
    CGN_CHECK_ARG(R >= 0 && C > 0 && C <= LN_MAX_C && ldx >= C && ldy >= C && eps >= 0.f);
    if (R == 0) return CGN_OK;
    CGN_CHECK_ARG(x && y && mean && rstd && ((uintptr_t)x | (uintptr_t)y) % (bf16 ? 2 : 4) == 0);
    hipStream_t s = (hipStream_t)stream;
    return bf16 ? norm_fwd<Bf16>(s, x, ldx, R, C, weight, bias, eps, y, ldy, mean, rstd)
                : norm_fwd<float>(s, x, ldx, R, C, weight, bias, eps, y, ldy, mean, rstd);
}

extern "C" int cgn_layer_norm_bwd_workspace(int64_t R, int32_t C, int32_t bf16, int64_t* bytes) {
    CGN_CHECK_ARG(R >= 0 && C > 0 && C <= LN_MAX_C && bytes);
    return bf16 ? norm_bwd<Bf16>(nullptr, nullptr, C, nullptr, C, R, C, nullptr, nullptr, nullptr, nullptr, C, nullptr,
                                 nullptr, 0.f, nullptr, 0, bytes)
                : norm_bwd<float>(nullptr, nullptr, C, nullptr, C, R, C, nullptr, nullptr, nullptr, nullptr, C, nullptr,
                                  nullptr, 0.f, nullptr, 0, bytes);
}

extern "C" int cgn_layer_norm_bwd(void* stream, const void* dy, int64_t lddy, const void* x, int64_t ldx, int64_t R,
                                  int32_t C, int32_t bf16, const float* weight, const float* mean, const float* rstd,
                                  void* dx, int64_t lddx, float* dweight, float* dbias, float beta, float* workspace,
                                  int64_t workspace_bytes) {
    CGN_CHECK_ARG(R >= 0 && C > 0 && C <= LN_MAX_C && lddy >= C && ldx >= C && (!dx || lddx >= C));
    CGN_CHECK_ARG(R == 0 || (dy && x && mean && rstd));
    CGN_CHECK_ARG(((uintptr_t)dy | (uintptr_t)x | (uintptr_t)dx) % (bf16 ? 2 : 4) == 0);
    CGN_CHECK_ARG((!dweight && !dbias) || workspace || workspace_bytes == 0);
    hipStream_t s = (hipStream_t)stream;
    return bf16 ? norm_bwd<Bf16>(s, dy, lddy, x, ldx, R, C, weight, mean, rstd, dx, lddx, dweight, dbias, beta, workspace,
                                 workspace_bytes, nullptr)
                : norm_bwd<float>(s, dy, lddy, x, ldx, R, C, weight, mean, rstd, dx, lddx, dweight, dbias, beta,
                                  workspace, workspace_bytes, nullptr);
}
