// Layer norm, dropout and the two in one pass (dropout + residual + layer norm), forward and
// backward, for gfx950.  All are bound by HBM traffic: up to 8192 columns every array is read or written once.
//
//   mean = sum_c x / C, rstd = 1 / sqrt(sum_c (x - mean)^2 / C + eps)      per row of C columns
//   xhat = (x - mean) * rstd, y = gamma * xhat + beta
//   gx = rstd * (g - sum_c(g) / C - xhat * sum_c(g * xhat) / C), g = gy * gamma
//   ggamma = sum_rows gy * xhat, gbeta = sum_rows gy
//   dropout: y = x * keep / (share kept) (+ residual), keep from random.h
//
// A row is held in registers between its statistics and its result: one wavefront per row up to
// 1024 columns, one workgroup of four up to 8192; beyond that a workgroup walks the row once per
// statistic and once for the result, and in the backward pass once more for the weights (2048 x 16384: 85 us forward, 167
// backward, at a copy's rate for one walk 43 and 65; 64 rows of 2^20 columns are 64 workgroups: 672 and 1112).  The variance is the mean
// of the squared distances from the mean, not a difference of two sums, so rows far from zero
// keep their digits.  A lane owns the same columns in every row it meets: gamma and beta are
// loaded once, and the weights' gradients are summed over a workgroup's rows in registers, left
// as one partial row per workgroup, and added by a second kernel in a fixed order (no atomics:
// same input, same bits).
#include "random.h"
#include <algorithm>

namespace cgt_amd {

struct __attribute__((packed, aligned(4))) float4a {      // 16 bytes at any 4-byte aligned address
    float v[4];
};

constexpr int kNormThreads = 256;
constexpr int kWideThreads = 1024;

// Columns [c0, c0 + N) of a row, zero outside [0, cols).
template <int N>
__device__ __forceinline__ void load_cols(const float* __restrict__ row, int c0, int cols, float (&v)[N]) {
    if (c0 + N <= cols) {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const float4a q = *reinterpret_cast<const float4a*>(row + c0 + i);
#pragma unroll
            for (int k = 0; k < 4; ++k) v[i + k] = q.v[k];
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = c0 + i < cols ? row[c0 + i] : 0.0f;
    }
}
// `stream`: the rows are 16-byte aligned and not read again soon.
template <int N>
__device__ __forceinline__ void store_cols(float* __restrict__ row, int c0, int cols, const float (&v)[N], bool stream = false) {
    if (stream && c0 + N <= cols) {
#pragma unroll
        for (int i = 0; i < N; i += 4) stream_store4(row + c0 + i, v[i], v[i + 1], v[i + 2], v[i + 3]);
    } else if (c0 + N <= cols) {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            float4a q;
#pragma unroll
            for (int k = 0; k < 4; ++k) q.v[k] = v[i + k];
            *reinterpret_cast<float4a*>(row + c0 + i) = q;
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (c0 + i < cols) row[c0 + i] = v[i];
    }
}

// keep / (share kept) of eight consecutive elements that start at flat index e0.  They lie in one
// group of the generator when e0 is a multiple of 8 and in two otherwise.
__device__ __forceinline__ void keep_factors(const RngState& rng, const DropoutRate& rate, unsigned long long e0, float (&f)[8]) {
    unsigned w[4];
    random_group(rng, e0 >> 3, w);
    const int shift = (int)(e0 & 7);
    if (shift) {
        unsigned u[4];
        random_group(rng, (e0 >> 3) + 1, u);
        unsigned all[8] = {w[0], w[1], w[2], w[3], u[0], u[1], u[2], u[3]};
        // all >>= 16 * shift bits
        if (shift & 4)
#pragma unroll
            for (int i = 0; i < 6; ++i) all[i] = all[i + 2];
        if (shift & 2)
#pragma unroll
            for (int i = 0; i < 5; ++i) all[i] = all[i + 1];
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = (shift & 1) ? (all[i] >> 16) | (all[i + 1] << 16) : all[i];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = random16(w, i) >= rate.threshold ? rate.scale : 0.0f;
}

// Half of a group for each of two neighbouring units of four elements (u even: the first half): the even lane of a
// pair brings the group of one run of units, the odd lane that of the next; `run` says whose is wanted.
__device__ __forceinline__ void pair_words(const unsigned (&w)[4], int run, unsigned (&mine)[2]) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const int low = run ? __builtin_amdgcn_mov_dpp((int)w[k], 0xF5, 0xf, 0xf, true) : __builtin_amdgcn_mov_dpp((int)w[k], 0xA0, 0xf, 0xf, true);
        const int high = run ? __builtin_amdgcn_mov_dpp((int)w[k + 2], 0xF5, 0xf, 0xf, true) : __builtin_amdgcn_mov_dpp((int)w[k + 2], 0xA0, 0xf, 0xf, true);
        mine[k] = (unsigned)((threadIdx.x & 1) ? high : low);
    }
}
__device__ __forceinline__ float keep4(const unsigned (&mine)[2], int i, const DropoutRate& rate) {
    return ((i & 1) ? mine[i >> 1] >> 16 : mine[i >> 1] & 0xffffu) >= rate.threshold ? rate.scale : 0.0f;
}
// keep / (share kept) of a row's pieces.  N = 8: a piece is eight columns, wherever its groups begin.  N = 4: rows of a
// multiple of 8 columns, where a pair of lanes has a group together.
template <int TPR, int CH, int N>
__device__ __forceinline__ void row_factors(const RngState& rng, const DropoutRate& rate, long at, int cols, float (&f)[CH][N]) {
    const int lane = threadIdx.x % TPR;
    if constexpr (N == 8) {
#pragma unroll
        for (int c = 0; c < CH; ++c)
            if ((lane + c * TPR) * N < cols) keep_factors(rng, rate, (unsigned long long)(at + (lane + c * TPR) * N), f[c]);
    } else {
#pragma unroll
        for (int c = 0; c < CH; c += 2) {
            const int pieces = CH - c >= 2 ? 2 : 1;
            unsigned w[4], mine[2];
            const int piece = pieces == 2 ? c + (lane & 1) : c;
            random_group(rng, ((unsigned long long)at >> 3) + ((lane + piece * TPR) >> 1), w);
#pragma unroll
            for (int run = 0; run < pieces; ++run) {
                if (pieces == 2) {
                    pair_words(w, run, mine);
                } else {
                    mine[0] = (lane & 1) ? w[2] : w[0];
                    mine[1] = (lane & 1) ? w[3] : w[1];
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) f[c + run][i] = keep4(mine, i, rate);
            }
        }
    }
}

// Sum over the THREADS lanes that share a row; every lane gets it.  `red` holds one pair per
// wavefront; a caller alternates between two of them so that one barrier per call is enough.
template <int THREADS>
__device__ __forceinline__ float2 row_sum(float a, float b, float2* red) {
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) {
        a += __shfl_xor(a, d);
        b += __shfl_xor(b, d);
    }
    if (THREADS > kWave) {
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = make_float2(a, b);
        __syncthreads();
        a = b = 0.0f;
#pragma unroll
        for (int i = 0; i < THREADS / kWave; ++i) {
            a += red[i].x;
            b += red[i].y;
        }
    }
    return make_float2(a, b);
}

struct NormFwd {
    const float *x, *residual, *gamma, *beta;
    float *y, *h, *mean, *rstd;      // mean, rstd may be null
    const long long* rng;
    DropoutRate rate;
    unsigned channel;
    long rows;
    int cols;
    float eps;
    bool stream;
};

// FUSED: h = residual + dropout(x) is formed, stored and normalised; DROP: with a mask (p > 0).
template <int TPR, int CH, int N, bool FUSED, bool DROP>
__global__ __launch_bounds__(kNormThreads) void norm_fwd_kernel(NormFwd a) {
    constexpr int RPB = kNormThreads / TPR;
    __shared__ float2 red[2][kNormThreads / kWave];
    const int lane = threadIdx.x % TPR;
    const float inv = 1.0f / (float)a.cols;
    float gamma[CH][N], beta[CH][N];
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        load_cols<N>(a.gamma, (lane + c * TPR) * N, a.cols, gamma[c]);
        load_cols<N>(a.beta, (lane + c * TPR) * N, a.cols, beta[c]);
    }
    RngState rng = {};
    if (DROP) rng = load_rng(a.rng, a.channel);
    for (long row = (long)blockIdx.x * RPB + threadIdx.x / TPR; row < a.rows; row += (long)gridDim.x * RPB) {
        const long at = row * a.cols;
        float v[CH][N];
        float sum = 0.0f;
#pragma unroll
        for (int c = 0; c < CH; ++c) load_cols<N>(a.x + at, (lane + c * TPR) * N, a.cols, v[c]);
        if (FUSED) {
            float r[CH][N];
#pragma unroll
            for (int c = 0; c < CH; ++c) load_cols<N>(a.residual + at, (lane + c * TPR) * N, a.cols, r[c]);
            float f[CH][N];
            if constexpr (DROP) row_factors<TPR, CH, N>(rng, a.rate, at, a.cols, f);
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                const int c0 = (lane + c * TPR) * N;
                if (DROP && c0 < a.cols)
#pragma unroll
                    for (int i = 0; i < N; ++i) v[c][i] = f[c][i] > 0.0f ? v[c][i] * f[c][i] : 0.0f;
#pragma unroll
                for (int i = 0; i < N; ++i) v[c][i] += r[c][i];
                store_cols<N>(a.h + at, c0, a.cols, v[c], a.stream);
            }
        }
#pragma unroll
        for (int c = 0; c < CH; ++c)
#pragma unroll
            for (int i = 0; i < N; ++i) sum += v[c][i];
        const float mean = row_sum<TPR>(sum, 0.0f, red[0]).x * inv;
        float sq = 0.0f;
#pragma unroll
        for (int c = 0; c < CH; ++c)
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float d = v[c][i] - mean;
                v[c][i] = d;
                if ((lane + c * TPR) * N + i < a.cols) sq += d * d;
            }
        const float rstd = 1.0f / sqrtf(row_sum<TPR>(sq, 0.0f, red[1]).x * inv + a.eps);
#pragma unroll
        for (int c = 0; c < CH; ++c) {
#pragma unroll
            for (int i = 0; i < N; ++i) v[c][i] = v[c][i] * rstd * gamma[c][i] + beta[c][i];
            store_cols<N>(a.y + at, (lane + c * TPR) * N, a.cols, v[c], a.stream);
        }
        if (lane == 0) {
            if (a.mean) a.mean[row] = mean;
            if (a.rstd) a.rstd[row] = rstd;
        }
    }
}

// Rows longer than the registers hold.  A thread meets the same columns in every walk, so what it
// reads back from h is what it wrote.
template <bool FUSED, bool DROP>
__global__ __launch_bounds__(kWideThreads) void norm_fwd_wide_kernel(NormFwd a) {
    __shared__ float2 red[2][kWideThreads / kWave];
    const float inv = 1.0f / (float)a.cols;
    RngState rng = {};
    if (DROP) rng = load_rng(a.rng, a.channel);
    for (long row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const long at = row * a.cols;
        const float* src = FUSED ? a.h + at : a.x + at;
        float sum = 0.0f;
        for (int c0 = threadIdx.x * 8; c0 < a.cols; c0 += kWideThreads * 8) {
            float v[8];
            load_cols<8>(a.x + at, c0, a.cols, v);
            if (FUSED) {
                float r[8];
                load_cols<8>(a.residual + at, c0, a.cols, r);
                if (DROP) {
                    float f[8];
                    keep_factors(rng, a.rate, (unsigned long long)(at + c0), f);
#pragma unroll
                    for (int i = 0; i < 8; ++i) v[i] = f[i] > 0.0f ? v[i] * f[i] : 0.0f;
                }
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] += r[i];
                store_cols<8>(a.h + at, c0, a.cols, v);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) sum += v[i];
        }
        const float mean = row_sum<kWideThreads>(sum, 0.0f, red[0]).x * inv;
        float sq = 0.0f;
        for (int c0 = threadIdx.x * 8; c0 < a.cols; c0 += kWideThreads * 8) {
            float v[8];
            load_cols<8>(src, c0, a.cols, v);
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (c0 + i < a.cols) sq += (v[i] - mean) * (v[i] - mean);
        }
        const float rstd = 1.0f / sqrtf(row_sum<kWideThreads>(sq, 0.0f, red[1]).x * inv + a.eps);
        for (int c0 = threadIdx.x * 8; c0 < a.cols; c0 += kWideThreads * 8) {
            float v[8], g[8], b[8];
            load_cols<8>(src, c0, a.cols, v);
            load_cols<8>(a.gamma, c0, a.cols, g);
            load_cols<8>(a.beta, c0, a.cols, b);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = (v[i] - mean) * rstd * g[i] + b[i];
            store_cols<8>(a.y + at, c0, a.cols, v);
        }
        if (threadIdx.x == 0) {
            if (a.mean) a.mean[row] = mean;
            if (a.rstd) a.rstd[row] = rstd;
        }
    }
}

struct NormBwd {
    const float *x, *gamma, *mean, *rstd, *gy, *gh;      // gh: cotangent of x itself, or null
    float *gx, *gdrop;                                   // gdrop: gradient through the dropout (DROP only)
    float* partial;                                      // [workgroups][2][cols]: sums of gy * xhat, of gy
    const long long* rng;
    DropoutRate rate;
    unsigned channel;
    long rows;
    int cols;
    bool stream;
};

template <int TPR, int CH, int N, bool ADD, bool DROP>
__global__ __launch_bounds__(kNormThreads) void norm_bwd_kernel(NormBwd a) {
    constexpr int RPB = kNormThreads / TPR;
    __shared__ float2 red[2][kNormThreads / kWave];
    __shared__ float join[TPR == kWave ? 3 * kWave * CH * N : 1];
    const int lane = threadIdx.x % TPR, sub = threadIdx.x / TPR;
    const float inv = 1.0f / (float)a.cols;
    float gamma[CH][N], sum_gx[CH][N], sum_g[CH][N];
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        load_cols<N>(a.gamma, (lane + c * TPR) * N, a.cols, gamma[c]);
#pragma unroll
        for (int i = 0; i < N; ++i) sum_gx[c][i] = sum_g[c][i] = 0.0f;
    }
    RngState rng = {};
    if (DROP) rng = load_rng(a.rng, a.channel);
    int turn = 0;
    for (long row = (long)blockIdx.x * RPB + sub; row < a.rows; row += (long)gridDim.x * RPB, turn ^= 1) {
        const long at = row * a.cols;
        float x[CH][N], g[CH][N], add[CH][N];
#pragma unroll
        for (int c = 0; c < CH; ++c) load_cols<N>(a.x + at, (lane + c * TPR) * N, a.cols, x[c]);
#pragma unroll
        for (int c = 0; c < CH; ++c) load_cols<N>(a.gy + at, (lane + c * TPR) * N, a.cols, g[c]);
        if (ADD)
#pragma unroll
            for (int c = 0; c < CH; ++c) load_cols<N>(a.gh + at, (lane + c * TPR) * N, a.cols, add[c]);
        const float mean = a.mean[row], rstd = a.rstd[row];
        float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
        for (int c = 0; c < CH; ++c)
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float xhat = (x[c][i] - mean) * rstd, gy = g[c][i];
                sum_gx[c][i] += gy * xhat;       // columns beyond the row: gy and gamma are 0, and nothing of them is stored
                sum_g[c][i] += gy;
                const float gg = gy * gamma[c][i];
                x[c][i] = xhat;
                g[c][i] = gg;
                if ((lane + c * TPR) * N + i < a.cols) {
                    s1 += gg;
                    s2 += gg * xhat;
                }
            }
        const float2 s = row_sum<TPR>(s1, s2, red[turn]);
        const float m1 = s.x * inv, m2 = s.y * inv;
        float f[CH][N];
        if constexpr (DROP) row_factors<TPR, CH, N>(rng, a.rate, at, a.cols, f);
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int c0 = (lane + c * TPR) * N;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                g[c][i] = rstd * (g[c][i] - m1 - x[c][i] * m2);
                if (ADD) g[c][i] += add[c][i];
            }
            store_cols<N>(a.gx + at, c0, a.cols, g[c], a.stream);
            if constexpr (DROP) {
                if (c0 < a.cols) {
#pragma unroll
                    for (int i = 0; i < N; ++i) g[c][i] = f[c][i] > 0.0f ? g[c][i] * f[c][i] : 0.0f;
                    store_cols<N>(a.gdrop + at, c0, a.cols, g[c], a.stream);
                }
            }
        }
    }
    float* out = a.partial + (long)blockIdx.x * 2 * a.cols;
    if constexpr (TPR == kWave) {       // the four wavefronts own the same columns: added in order
#pragma unroll
        for (int which = 0; which < 2; ++which) {
            __syncthreads();
            if (sub > 0)
#pragma unroll
                for (int c = 0; c < CH; ++c)
#pragma unroll
                    for (int i = 0; i < N; ++i)
                        join[((sub - 1) * CH * N + c * N + i) * kWave + lane] = which ? sum_g[c][i] : sum_gx[c][i];
            __syncthreads();
            if (sub == 0)
#pragma unroll
                for (int c = 0; c < CH; ++c) {
#pragma unroll
                    for (int i = 0; i < N; ++i)
#pragma unroll
                        for (int o = 0; o < 3; ++o) {
                            const float v = join[(o * CH * N + c * N + i) * kWave + lane];
                            if (which) sum_g[c][i] += v;
                            else sum_gx[c][i] += v;
                        }
                    store_cols<N>(out + which * a.cols, (lane + c * TPR) * N, a.cols, which ? sum_g[c] : sum_gx[c]);
                }
        }
    } else {
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            store_cols<N>(out, (lane + c * TPR) * N, a.cols, sum_gx[c]);
            store_cols<N>(out + a.cols, (lane + c * TPR) * N, a.cols, sum_g[c]);
        }
    }
}

template <bool ADD, bool DROP>
__global__ __launch_bounds__(kWideThreads) void norm_bwd_wide_kernel(NormBwd a) {
    __shared__ float2 red[2][kWideThreads / kWave];
    const float inv = 1.0f / (float)a.cols;
    RngState rng = {};
    if (DROP) rng = load_rng(a.rng, a.channel);
    int turn = 0;
    for (long row = blockIdx.x; row < a.rows; row += gridDim.x, turn ^= 1) {
        const long at = row * a.cols;
        const float mean = a.mean[row], rstd = a.rstd[row];
        float s1 = 0.0f, s2 = 0.0f;
        for (int c0 = threadIdx.x * 8; c0 < a.cols; c0 += kWideThreads * 8) {
            float x[8], g[8], w[8];
            load_cols<8>(a.x + at, c0, a.cols, x);
            load_cols<8>(a.gy + at, c0, a.cols, g);
            load_cols<8>(a.gamma, c0, a.cols, w);
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (c0 + i < a.cols) {
                    const float gg = g[i] * w[i];
                    s1 += gg;
                    s2 += gg * ((x[i] - mean) * rstd);
                }
        }
        const float2 s = row_sum<kWideThreads>(s1, s2, red[turn]);
        const float m1 = s.x * inv, m2 = s.y * inv;
        for (int c0 = threadIdx.x * 8; c0 < a.cols; c0 += kWideThreads * 8) {
            float x[8], g[8], w[8];
            load_cols<8>(a.x + at, c0, a.cols, x);
            load_cols<8>(a.gy + at, c0, a.cols, g);
            load_cols<8>(a.gamma, c0, a.cols, w);
#pragma unroll
            for (int i = 0; i < 8; ++i) g[i] = rstd * (g[i] * w[i] - m1 - (x[i] - mean) * rstd * m2);
            if (ADD) {
                float add[8];
                load_cols<8>(a.gh + at, c0, a.cols, add);
#pragma unroll
                for (int i = 0; i < 8; ++i) g[i] += add[i];
            }
            store_cols<8>(a.gx + at, c0, a.cols, g);
            if (DROP) {
                float f[8];
                keep_factors(rng, a.rate, (unsigned long long)(at + c0), f);
#pragma unroll
                for (int i = 0; i < 8; ++i) g[i] = f[i] > 0.0f ? g[i] * f[i] : 0.0f;
                store_cols<8>(a.gdrop + at, c0, a.cols, g);
            }
        }
    }
}

// Partial sums of the weights' gradients for wide rows: workgroup (strip of 64 columns, part of the rows).
__global__ __launch_bounds__(kNormThreads) void norm_bwd_wide_weights_kernel(NormBwd a, long rows_per) {
    __shared__ float2 join[kNormThreads];
    const int c = blockIdx.x * 64 + (threadIdx.x & 63);
    const long first = blockIdx.y * rows_per, last = first + rows_per < a.rows ? first + rows_per : a.rows;
    float s1 = 0.0f, s2 = 0.0f;
    if (c < a.cols)
        for (long row = first + (threadIdx.x >> 6); row < last; row += kNormThreads / 64) {
            const float g = a.gy[row * a.cols + c];
            s1 += g * ((a.x[row * a.cols + c] - a.mean[row]) * a.rstd[row]);
            s2 += g;
        }
    join[threadIdx.x] = make_float2(s1, s2);
    __syncthreads();
    if (threadIdx.x < 64 && c < a.cols) {
        for (int o = 1; o < kNormThreads / 64; ++o) {
            s1 += join[threadIdx.x + o * 64].x;
            s2 += join[threadIdx.x + o * 64].y;
        }
        float* out = a.partial + (long)blockIdx.y * 2 * a.cols;
        out[c] = s1;
        out[a.cols + c] = s2;
    }
}

// ggamma, gbeta = the partial rows added up: 32 columns per workgroup and trip, 32 groups of rows.  (A grid holds less than
// 2^32 threads, that is 2^26 columns: wider rows take several trips.)
constexpr long kWeightsGrid = 1L << 20;
__global__ __launch_bounds__(1024) void norm_weights_kernel(const float* __restrict__ partial, int parts, int cols,
                                                            float* __restrict__ ggamma, float* __restrict__ gbeta) {
    __shared__ float join[32][33];
    const int g = threadIdx.x >> 5;
    const long pitch = 2L * cols;
    for (long c0 = blockIdx.x * 32L; c0 < pitch; c0 += gridDim.x * 32L) {
        const long c = c0 + (threadIdx.x & 31);      // in [0, 2 * cols)
        float s = 0.0f;
        if (c < pitch) {
#pragma unroll 8
            for (int p = g; p < parts; p += 32) s += partial[p * pitch + c];
        }
        join[g][threadIdx.x & 31] = s;
        __syncthreads();
        if (g == 0 && c < pitch) {
            for (int o = 1; o < 32; ++o) s += join[o][threadIdx.x];
            if (c < cols) ggamma[c] = s;
            else gbeta[c - cols] = s;
        }
        __syncthreads();
    }
}

// y = dropout(x) (+ residual).  The first `whole` workgroups take PIECES x 2048 elements each of 16-byte aligned arrays
// in accesses of 64 neighbouring 16-byte units a wavefront.  Unit u of such a run is half of group u / 2, so a pair of
// lanes shares each group it meets: the even lane forms those of one run, the odd lane those of the
// next, and they exchange halves.  The other workgroups take what is left (everything, where an array is not aligned) a
// group per thread.  33.5 M elements: 42.6 us (6.3 TB/s, the rate of a copy), 54.5 with a group per thread throughout.
template <bool RES, int PIECES>
__global__ __launch_bounds__(256) void dropout_kernel(const float* __restrict__ xs, const float* __restrict__ rs, float* __restrict__ ys,
                                                      const long long* __restrict__ state, DropoutRate rate, unsigned channel, long whole, long n) {
    const RngState rng = load_rng(state, channel);
    if ((long)blockIdx.x >= whole) {
        const long g = whole * (PIECES * 256) + ((long)blockIdx.x - whole) * 256 + threadIdx.x;
        if (8 * g >= n) return;
        const int left = n - 8 * g < 8 ? (int)(n - 8 * g) : 8;
        float v[8], r[8], f[8];
        load_cols<8>(xs + 8 * g, 0, left, v);
        if (RES) load_cols<8>(rs + 8 * g, 0, left, r);
        keep_factors(rng, rate, 8ull * g, f);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            v[i] = f[i] > 0.0f ? v[i] * f[i] : 0.0f;
            if (RES) v[i] += r[i];
        }
        store_cols<8>(ys + 8 * g, 0, left, v);
        return;
    }
    const v4f *x = reinterpret_cast<const v4f*>(xs), *residual = reinterpret_cast<const v4f*>(rs);
    v4f* y = reinterpret_cast<v4f*>(ys);
    const int lane = threadIdx.x & 63;
    const long unit0 = ((long)blockIdx.x * 4 + (threadIdx.x >> 6)) * (128 * PIECES) + lane;
    v4f v[2 * PIECES], r[2 * PIECES];
#pragma unroll
    for (int p = 0; p < 2 * PIECES; ++p) v[p] = __builtin_nontemporal_load(x + unit0 + 64 * p);
    if (RES)
#pragma unroll
        for (int p = 0; p < 2 * PIECES; ++p) r[p] = __builtin_nontemporal_load(residual + unit0 + 64 * p);
#pragma unroll
    for (int p = 0; p < PIECES; ++p) {
        unsigned w[4];
        random_group(rng, (unsigned long long)(unit0 - lane + 128 * p + 64 * (lane & 1) + (lane & ~1)) >> 1, w);
#pragma unroll
        for (int run = 0; run < 2; ++run) {      // the group's words from the lane of the pair that formed it
            unsigned mine[2];
            pair_words(w, run, mine);
            v4f q = v[2 * p + run];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                q[i] = keep4(mine, i, rate) > 0.0f ? q[i] * rate.scale : 0.0f;
                if (RES) q[i] += r[2 * p + run][i];
            }
            __builtin_nontemporal_store(q, y + unit0 + 64 * (2 * p + run));
        }
    }
}

// ---------------------------------------------------------------- launchers

// Whether the results of a pass are stored past the caches: aligned rows, 4 MiB of them or more.  Both sides (stored
// past / through the caches, rows of 1024, buffers in turn): forward 1024 rows 4.3 / 5.1 us, 2048 rows 5.2 / 7.0, 16384
// rows 25.8 / 27.0; backward 9.1 / 10.2, 12.0 / 13.6, 40.9 / 41.8.  512 rows and fewer are alike (3.8 / 3.9 us).  A
// second norm that reads the first one's result at once: 2048 rows 10.6 / 12.5 us for both, 8192 rows 29.2 / 29.5,
// 16384 rows 51.5 / 47.9 (64 MiB that the last-level cache would have kept).
constexpr long kStreamFloats = 1L << 20;
static bool stream_results(long rows, long cols, const void* p, const void* q) {
    return cols % 4 == 0 && (reinterpret_cast<uintptr_t>(p) | reinterpret_cast<uintptr_t>(q)) % 16 == 0 && rows * cols >= kStreamFloats;
}

template <bool FUSED, bool DROP, int N>
static int launch_norm_fwd(NormFwd a, hipStream_t st) {
    a.stream = stream_results(a.rows, a.cols, a.y, a.h);
    auto blocks = [&](int rpb) { return dim3((unsigned)std::min(cdiv(a.rows, rpb), 4L * kNumCU * 2)); };
    const int pieces = (int)cdiv(a.cols, N);
    if (pieces <= 64) norm_fwd_kernel<64, 1, N, FUSED, DROP><<<blocks(4), kNormThreads, 0, st>>>(a);
    else if (pieces <= 128) norm_fwd_kernel<64, 2, N, FUSED, DROP><<<blocks(4), kNormThreads, 0, st>>>(a);
    else if (N == 4 && pieces <= 256) norm_fwd_kernel<64, 16 / N, N, FUSED, DROP><<<blocks(4), kNormThreads, 0, st>>>(a);
    else if (pieces <= 4096 / N) norm_fwd_kernel<256, 16 / N, N, FUSED, DROP><<<blocks(1), kNormThreads, 0, st>>>(a);
    else if (pieces <= 8192 / N) norm_fwd_kernel<256, 32 / N, N, FUSED, DROP><<<blocks(1), kNormThreads, 0, st>>>(a);
    else norm_fwd_wide_kernel<FUSED, DROP><<<dim3((unsigned)std::min(a.rows, 2L * kNumCU)), kWideThreads, 0, st>>>(a);
    CGT_LAUNCH_CHECK("layer norm forward");
    return CGT_AMD_OK;
}

template <bool ADD, bool DROP, int N>
static int launch_norm_bwd(NormBwd a, float* ggamma, float* gbeta, void* stream) {
    const StreamTurn turn(stream);
    hipStream_t st = as_stream(stream);
    const int pieces = (int)cdiv(a.cols, N);
    const bool wave_rows = a.cols <= 1024, wide = a.cols > 8192;
    long parts = wide ? std::min(cdiv(a.rows, 64), 64L) : std::min(cdiv(a.rows, wave_rows ? 4 : 1), 2L * kNumCU);
    const long rows_per = wide ? cdiv(a.rows, parts) : 0;
    if (wide) parts = cdiv(a.rows, rows_per);
    a.stream = stream_results(a.rows, a.cols, a.gx, a.gdrop);
    a.partial = stream_workspace(stream, kWsNorm, (size_t)parts * 2 * a.cols * sizeof(float), "layer norm backward");
    if (!a.partial) return CGT_AMD_ERR_NOMEM;
    const dim3 grid((unsigned)parts);
    if (pieces <= 64) norm_bwd_kernel<64, 1, N, ADD, DROP><<<grid, kNormThreads, 0, st>>>(a);
    else if (pieces <= 128) norm_bwd_kernel<64, 2, N, ADD, DROP><<<grid, kNormThreads, 0, st>>>(a);
    else if (N == 4 && pieces <= 256) norm_bwd_kernel<64, 16 / N, N, ADD, DROP><<<grid, kNormThreads, 0, st>>>(a);
    else if (pieces <= 4096 / N) norm_bwd_kernel<256, 16 / N, N, ADD, DROP><<<grid, kNormThreads, 0, st>>>(a);
    else if (!wide) norm_bwd_kernel<256, 32 / N, N, ADD, DROP><<<grid, kNormThreads, 0, st>>>(a);
    else {
        norm_bwd_wide_kernel<ADD, DROP><<<dim3((unsigned)std::min(a.rows, 2L * kNumCU)), kWideThreads, 0, st>>>(a);
        CGT_LAUNCH_CHECK("layer norm backward");
        norm_bwd_wide_weights_kernel<<<dim3((unsigned)cdiv(a.cols, 64), (unsigned)parts), kNormThreads, 0, st>>>(a, rows_per);
    }
    CGT_LAUNCH_CHECK("layer norm backward");
    norm_weights_kernel<<<dim3((unsigned)std::min(cdiv(2L * a.cols, 32), kWeightsGrid)), 1024, 0, st>>>(a.partial, (int)parts, a.cols, ggamma, gbeta);
    CGT_LAUNCH_CHECK("layer norm weight gradient");
    return CGT_AMD_OK;
}

static int check_rows(const char* what, long rows, long cols) {
    CGT_ARG_CHECK(rows >= 0 && cols >= 0, "%s: negative extent (%ld rows, %ld columns)", what, rows, cols);
    CGT_ARG_CHECK(cols < (1L << 30), "%s: rows of %ld columns are too long (2^30 at most)", what, cols);
    CGT_ARG_CHECK(cols == 0 || rows < (1L << 60) / cols, "%s: the array is too large", what);
    return CGT_AMD_OK;
}

static int zero_weights(float* ggamma, float* gbeta, long cols, void* stream) {
    CGT_ARG_CHECK(ggamma && gbeta, "layer norm backward: null pointer");
    const int rc = cgt_amd_fill_u32(ggamma, 0u, cols, stream);
    return rc == CGT_AMD_OK ? cgt_amd_fill_u32(gbeta, 0u, cols, stream) : rc;
}

}  // namespace cgt_amd

using namespace cgt_amd;

CGT_API int cgt_amd_layer_norm_fwd_f32(const float* x, long rows, long cols, const float* gamma, const float* beta, double eps,
                                       float* y, float* mean, float* rstd, void* stream) {
    if (int rc = check_rows("layer norm", rows, cols)) return rc;
    CGT_ARG_CHECK(eps >= 0.0, "layer norm: eps must not be negative (got %g)", eps);
    CGT_ARG_CHECK(cols > 0 || rows == 0 || !(mean || rstd), "layer norm: rows of no columns have no statistics");
    if (rows == 0 || cols == 0) return CGT_AMD_OK;
    CGT_ARG_CHECK(x && gamma && beta && y, "layer norm: null pointer");
    NormFwd a = {};
    a.x = x, a.gamma = gamma, a.beta = beta, a.y = y, a.mean = mean, a.rstd = rstd;
    a.rows = rows, a.cols = (int)cols, a.eps = (float)eps;
    return launch_norm_fwd<false, false, 4>(a, as_stream(stream));
}

CGT_API int cgt_amd_layer_norm_bwd_f32(const float* x, const float* gamma, const float* mean, const float* rstd, const float* gy,
                                       long rows, long cols, float* gx, float* ggamma, float* gbeta, void* stream) {
    if (int rc = check_rows("layer norm backward", rows, cols)) return rc;
    if (cols == 0) return CGT_AMD_OK;
    if (rows == 0) return zero_weights(ggamma, gbeta, cols, stream);
    CGT_ARG_CHECK(x && gamma && mean && rstd && gy && gx && ggamma && gbeta, "layer norm backward: null pointer");
    NormBwd a = {};
    a.x = x, a.gamma = gamma, a.mean = mean, a.rstd = rstd, a.gy = gy, a.gx = gx;
    a.rows = rows, a.cols = (int)cols;
    return launch_norm_bwd<false, false, 4>(a, ggamma, gbeta, stream);
}

CGT_API int cgt_amd_dropout_f32(const float* x, const float* residual, long n, double p, const long long* rng, unsigned channel,
                                float* y, void* stream) {
    CGT_ARG_CHECK(n >= 0, "dropout: negative count");
    DropoutRate rate;
    if (!dropout_rate(p, "dropout", &rate)) return CGT_AMD_ERR_ARG;
    if (n == 0) return CGT_AMD_OK;
    CGT_ARG_CHECK(x && y && rng, "dropout: null pointer");
    hipStream_t st = as_stream(stream);
    const uintptr_t all = reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(residual) | reinterpret_cast<uintptr_t>(y);
    constexpr int kPieces = 2;
    const long whole = all % 16 == 0 ? n / (2048 * kPieces) : 0, blocks = whole + cdiv(cdiv(n, 8) - whole * (256 * kPieces), 256);
    CGT_ARG_CHECK(blocks < (1L << 31), "dropout: too many elements");
    if (residual) dropout_kernel<true, kPieces><<<dim3((unsigned)blocks), 256, 0, st>>>(x, residual, y, rng, rate, channel, whole, n);
    else dropout_kernel<false, kPieces><<<dim3((unsigned)blocks), 256, 0, st>>>(x, nullptr, y, rng, rate, channel, whole, n);
    CGT_LAUNCH_CHECK("dropout");
    return CGT_AMD_OK;
}

CGT_API int cgt_amd_dropout_add_layer_norm_fwd_f32(const float* x, const float* residual, long rows, long cols, double p,
                                                   const long long* rng, unsigned channel, const float* gamma, const float* beta,
                                                   double eps, float* y, float* h, float* mean, float* rstd, void* stream) {
    if (int rc = check_rows("dropout + add + layer norm", rows, cols)) return rc;
    CGT_ARG_CHECK(eps >= 0.0, "dropout + add + layer norm: eps must not be negative (got %g)", eps);
    NormFwd a = {};
    if (!dropout_rate(p, "dropout + add + layer norm", &a.rate)) return CGT_AMD_ERR_ARG;
    CGT_ARG_CHECK(cols > 0 || rows == 0 || !(mean || rstd), "dropout + add + layer norm: rows of no columns have no statistics");
    if (rows == 0 || cols == 0) return CGT_AMD_OK;
    CGT_ARG_CHECK(x && residual && gamma && beta && y && h, "dropout + add + layer norm: null pointer");
    CGT_ARG_CHECK(rng || a.rate.threshold == 0, "dropout + add + layer norm: dropout needs the generator's state");
    a.x = x, a.residual = residual, a.gamma = gamma, a.beta = beta, a.y = y, a.h = h, a.mean = mean, a.rstd = rstd;
    a.rng = rng, a.channel = channel, a.rows = rows, a.cols = (int)cols, a.eps = (float)eps;
    if (a.rate.threshold == 0) return launch_norm_fwd<true, false, 4>(a, as_stream(stream));
    // four columns a lane and piece where a pair of lanes has a generator's group together (neighbouring lanes then read
    // neighbouring 16 bytes; 16384 x 1024: 47.5 us, eight columns a lane 51.8), eight where rows begin inside a group
    return a.cols % 8 == 0 ? launch_norm_fwd<true, true, 4>(a, as_stream(stream)) : launch_norm_fwd<true, true, 8>(a, as_stream(stream));
}

CGT_API int cgt_amd_dropout_add_layer_norm_bwd_f32(const float* h, const float* gamma, const float* mean, const float* rstd,
                                                   const float* gy, const float* gh, long rows, long cols, double p,
                                                   const long long* rng, unsigned channel, float* gx, float* gresidual,
                                                   float* ggamma, float* gbeta, void* stream) {
    if (int rc = check_rows("dropout + add + layer norm backward", rows, cols)) return rc;
    NormBwd a = {};
    if (!dropout_rate(p, "dropout + add + layer norm backward", &a.rate)) return CGT_AMD_ERR_ARG;
    if (cols == 0) return CGT_AMD_OK;
    if (rows == 0) return zero_weights(ggamma, gbeta, cols, stream);
    CGT_ARG_CHECK(h && gamma && mean && rstd && gy && gresidual && ggamma && gbeta, "dropout + add + layer norm backward: null pointer");
    CGT_ARG_CHECK(a.rate.threshold == 0 || (rng && gx), "dropout + add + layer norm backward: dropout needs the generator's state and gx");
    a.x = h, a.gamma = gamma, a.mean = mean, a.rstd = rstd, a.gy = gy, a.gh = gh, a.gx = gresidual, a.gdrop = gx;
    a.rng = rng, a.channel = channel, a.rows = rows, a.cols = (int)cols;
    if (a.rate.threshold == 0) {
        // without a mask the two gradients are one array; a caller that wants both gets a copy
        const int rc = gh ? launch_norm_bwd<true, false, 4>(a, ggamma, gbeta, stream) : launch_norm_bwd<false, false, 4>(a, ggamma, gbeta, stream);
        if (rc != CGT_AMD_OK || !gx || gx == gresidual) return rc;
        return cgt_amd_stream_copy(gx, gresidual, rows * cols * (long)sizeof(float), stream);
    }
    // (four or eight columns a lane as in the forward pass: 4095 x 768 17.4 us with four, 18.6 with eight)
    if (a.cols % 8 == 0) return gh ? launch_norm_bwd<true, true, 4>(a, ggamma, gbeta, stream) : launch_norm_bwd<false, true, 4>(a, ggamma, gbeta, stream);
    return gh ? launch_norm_bwd<true, true, 8>(a, ggamma, gbeta, stream) : launch_norm_bwd<false, true, 8>(a, ggamma, gbeta, stream);
}
