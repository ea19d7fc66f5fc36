// Attention with a learned relative position bias, forward and backward, for gfx950.
//
//   s_ij = scale * q_i . k_j + table[bucket(j - i - offset)][head]
//   p_ij = exp(s_ij - lse_i), lse_i = log sum_j exp(s_ij) over the keys query i may see
//   o_i = sum_j p_ij keep_ij v_j
//   gv_j = sum_i p_ij keep_ij go_i
//   ds_ij = p_ij (keep_ij go_i . v_j - go_i . o_i)
//   gq_i = scale sum_j ds_ij k_j,  gk_j = scale sum_i ds_ij q_i
//   gtable[c] = sum of ds_ij over batch, i and j with bucket(j - i - offset) = c
//
// The scores never leave the registers: a pass walks the keys (or the queries) in tiles of 32 and
// keeps a running maximum and sum of every row.  The backward pass forms the probabilities again
// from lse: one kernel per block of queries leaves gq and the table's gradient, one per block of
// keys gk and gv, so no sum is shared between workgroups and results do not depend on the order
// they run in.
//
// Matrix products run at float32 accuracy on the fp16 matrix cores: an operand, times a power of two, is cut into two
// fp16 terms, x = h + l (l is the rounded rest: 22 bits and the sign), and the products l h, h l, h h are accumulated in
// float32.  Three v_mfma_f32_32x32x16_f16 do in 3 x 32 cycles what eight v_mfma_f32_32x32x2_f32 do in 8 x 64, and the vector
// units work beside them (fp32 matrix instructions keep them busy).  Measured on products of 128 (64) normal values: error
// 1.1e-7 (1.0e-7) of the results' rms, 2.0e-7 (1.4e-7) with the fp32 instructions.  The powers of two:
//   a lane's own column has one, that brings its largest value to [2^14, 2^15);
//   a tile of 32 rows in LDS has one, or one a row where its rows differ by more than 2^8 (attn_scale_kernel).  So a row's
//     digits do not depend on the rows around it: values keep 22 bits down to 2^-9 of its largest and an absolute 2^-31 of
//     that below, at least;
//   what multiplies such a tile in the sums over keys or queries (p v, ds k, p go, ds q) takes over the rows' factors, so that
//     it is of the size of the terms that are added, and gets the power of two that its largest term needs: of the tile in
//     the backward pass, of the terms met so far in the forward pass, where the others are cut with an absolute error
//     of 2^-35 of the largest at most.
// Nothing is read behind the lengths.  A NaN or infinity in a row of q makes that row NaN, one in a row of k or v that the
// walk meets all of its head: a key that a causal mask hides has probability 0, and 0 * NaN is NaN.
//
// A wavefront owns 32 columns (queries in the forward and the first backward kernel, keys in the
// second) and forms the *transposed* score tile, rows = the other side: lane l then holds, for
// column l % 32, rows 8 g + 4 (l / 32) + t in register 4 g + t.  With the k positions of the next
// product's 16-wide step taken in the order (row 8 b + 4 half + t at position 8 half + 4 b + t)
// the score tile, cut into its terms, is that product's B operand as it stands, with no
// exchange between lanes; the other operand is laid out in that order when it is put into LDS.
#include "random.h"
#include <algorithm>
#include <cmath>
#include <type_traits>

namespace cgt_amd {

typedef float v16f __attribute__((ext_vector_type(16)));
struct __attribute__((packed, aligned(4))) float4p {      // 16 bytes at any 4-byte aligned address
    float x, y, z, w;
};

struct __attribute__((packed, aligned(4))) float2p {
    float x, y;
};

constexpr int kAttnThreads = 256;
constexpr int kAttnCols = 128;     // columns (queries or keys) per workgroup: 32 per wavefront
constexpr int kAttnRows = 32;      // rows of the tile that the four wavefronts share
constexpr int kMaxBuckets = 256;
constexpr int kMaxDistance = 1024;
constexpr float kLog2e = 1.4426950408889634f;

struct BucketRule {
    int buckets, bidirectional, max_distance, first, side;
    int edge[kMaxBuckets / 2 + 1];      // edge[e]: the smallest distance of logarithmic bucket e of a side, e >= 1
};

struct Attn {
    const float *q, *k, *v, *table;
    const int *q_lengths, *k_lengths, *q_offsets;
    const long long* rng;
    long q_b, q_h, q_t, k_b, k_h, k_t;      // strides in floats; o, go, gq as q, and v, gk, gv as k
    int B, H, Tq, Tk, D, causal, q_offset;
    float scale;
    DropoutRate rate;
    unsigned channel;
    BucketRule rule;
};

// Bucket of relative position `rel` (key minus query).
__host__ __device__ inline int bucket_of(const BucketRule& r, int rel) {
    const int n = r.bidirectional ? (rel < 0 ? -rel : rel) : (rel < 0 ? -rel : 0);
    int b = n;
    if (n >= r.first) {
        b = r.first;
        for (int e = 1; e < r.side - r.first; ++e) b += n >= r.edge[e] ? 1 : 0;
    }
    return b + (r.bidirectional && rel > 0 ? r.side : 0);
}

// ---- the bias in LDS: one value per relative position in [-reach, reach], reach = max_distance + 62.
// A wavefront's tile spans 63 relative positions around its origin (that of its first row and
// column).  An origin max_distance + 31 or more away makes the tile far: all of it is in the last
// bucket of a side.  Any other origin keeps every index inside the window.
__host__ __device__ inline int bias_reach(const BucketRule& r) { return r.max_distance + 62; }
__host__ __device__ inline int bias_window(const BucketRule& r) { return 2 * bias_reach(r) + 1; }
__device__ __forceinline__ bool far_tile(const BucketRule& r, int rel0) { return rel0 >= r.max_distance + 31 || rel0 <= -r.max_distance - 31; }
__device__ __forceinline__ float to_log2(float x);
__device__ __forceinline__ void fill_bias(const Attn& a, int head, float* win) {
    const int n = bias_window(a.rule), reach = bias_reach(a.rule);
    for (int s = threadIdx.x; s < n; s += kAttnThreads) win[s] = to_log2(a.table[(long)bucket_of(a.rule, s - reach) * a.H + head]);
}

// Four floats of a row of D at column c; zero beyond the row's end.
__device__ __forceinline__ float4 load4(const float* row, int c, int D) {
    if (c + 4 <= D) {
        const float4p v = *reinterpret_cast<const float4p*>(row + c);
        return make_float4(v.x, v.y, v.z, v.w);
    }
    return make_float4(c < D ? row[c] : 0.0f, c + 1 < D ? row[c + 1] : 0.0f, c + 2 < D ? row[c + 2] : 0.0f, 0.0f);
}
__device__ __forceinline__ void store4(float* row, int c, int D, float x, float y, float z, float w) {
    if (c + 4 <= D) {
        *reinterpret_cast<float4p*>(row + c) = {x, y, z, w};
    } else {
        if (c < D) row[c] = x;
        if (c + 1 < D) row[c + 1] = y;
        if (c + 2 < D) row[c + 2] = z;
    }
}

// Rows 8 g + 4 half .. + 3 of a 32-row result block, times f; zero where the column is none.
__device__ __forceinline__ void store_scaled(float* row, int c, int D, const v16f& v, int g, bool valid, float f) {
    store4(row, c, D, valid ? v[4 * g] * f : 0.0f, valid ? v[4 * g + 1] * f : 0.0f, valid ? v[4 * g + 2] * f : 0.0f, valid ? v[4 * g + 3] * f : 0.0f);
}

typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef float v2f __attribute__((ext_vector_type(2)));
typedef unsigned v4u32 __attribute__((ext_vector_type(4)));

// The power of two that brings `top` to [2^14, 2^15).  Capped at 2^126: values below 2^-112 lose digits.
__device__ __forceinline__ float power_scale(float top) {
    const unsigned e = __float_as_uint(top) >> 23 & 255u;
    return __uint_as_float(min(268u - e, 253u) << 23);
}
__device__ __forceinline__ float reciprocal_power(float s) { return __uint_as_float((254u << 23) - __float_as_uint(s)); }

// The two fp16 terms of two floats, each times a power of two, packed (first in the low half).
struct Terms {
    unsigned t[2];
};
__device__ __forceinline__ Terms split2(float x, float y, float sx, float sy) {
    const v2h h = {(_Float16)__builtin_fmaf(x, sx, 0.0f), (_Float16)__builtin_fmaf(y, sy, 0.0f)};
    const v2h l = {(_Float16)__builtin_fmaf(x, sx, -(float)h.x), (_Float16)__builtin_fmaf(y, sy, -(float)h.y)};
    return {{__builtin_bit_cast(unsigned, h), __builtin_bit_cast(unsigned, l)}};
}
__device__ __forceinline__ Terms split2(float x, float y) {
    const v2f v = {x, y};
    const v2h h = __builtin_convertvector(v, v2h);
    float one = 1.0f;
    asm("" : "+s"(one));      // a 1 that the compiler does not see: subtraction and rounding stay one instruction
    const v2h l = {(_Float16)__builtin_fmaf(x, one, -(float)h.x), (_Float16)__builtin_fmaf(y, one, -(float)h.y)};
    return {{__builtin_bit_cast(unsigned, h), __builtin_bit_cast(unsigned, l)}};
}
// An operand of one 16-wide step: 8 values of the lane, two terms.
struct Frag {
    v8h t[2];
};
__device__ __forceinline__ Frag split8(const float (&x)[8]) {
    v4u32 w[2];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const Terms t = split2(x[2 * i], x[2 * i + 1]);
        w[0][i] = t.t[0];
        w[1][i] = t.t[1];
    }
    return {{__builtin_bit_cast(v8h, w[0]), __builtin_bit_cast(v8h, w[1])}};
}
// acc += a * b
__device__ __forceinline__ v16f mul_step(v16f acc, const Frag& a, const Frag& b) {
    acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(a.t[1], b.t[0], acc, 0, 0, 0);
    acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(a.t[0], b.t[1], acc, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a.t[0], b.t[0], acc, 0, 0, 0);
}

// What a tile's rows are scaled by: one power of two, or 0 and one for each row where the rows are mixed (rare: see
// attn_scale_kernel).  Where they are not, a tile costs a scalar load.
struct ScaleArray {
    const float *tiles, *rows, *weights;      // a head's; weights of rows (null: 1) that go into what undoes the scales of a mixed tile
};
// One of a tile's, by the scalar unit (nothing in the same kernel writes there).
__device__ __forceinline__ float tile_scale(const float* tiles, int n) {
    return reinterpret_cast<const __attribute__((address_space(4))) float*>(reinterpret_cast<uintptr_t>(tiles))[__builtin_amdgcn_readfirstlane(n)];
}

// A tile of 32 rows of DP columns, shared by the workgroup.  A thread loads four neighbouring rows of
// DP / 32 columns (rows at or beyond `end` are zero and not read), scales them, cuts them into terms and
// writes them to LDS in one or both of two layouts, two planes (terms) each:
//   by rows:    [row][DP + 8]  the A operand whose rows are the tile's
//   by columns: [column][40]   the A operand whose rows are the tile's columns; the 32 rows in the
//                              order of the score tile's registers (see above)
// With these pitches the 16-byte reads of eight neighbouring rows start in different banks.
template <int DP>
struct Tile {
    static constexpr int E = DP / 32, kRowPitch = DP + 8, kColPitch = 40;
    static constexpr int kRowPlane = kAttnRows * kRowPitch, kColPlane = DP * kColPitch;      // in 16-bit values
    static constexpr int kRowBytes = 2 * kRowPlane * 2, kColBytes = 2 * kColPlane * 2;
    float v[4][E];

    // What does not change from tile to tile: the lane's offsets (bytes) from a tile's first row.
    struct Offsets {
        unsigned at[4];
        bool fit;
        __device__ __forceinline__ Offsets(long stride, int D) : fit(D == DP && stride < (1L << 24)) {
            const int c = (threadIdx.x & 31) * E, r0 = (threadIdx.x >> 5) * 4;
#pragma unroll
            for (int r = 0; r < 4; ++r) at[r] = (unsigned)((r0 + r) * (int)stride + c) * 4u;
        }
    };
    // Rows row0 .. row0 + 31, zero at or beyond `end` and in columns beyond a head's own (both are read from the last
    // row or column inside, so that all loads are issued together; `end` is positive).
    __device__ __forceinline__ void load(const Offsets& off, const float* base, long stride, int row0, int end, int D) {
        if (off.fit && row0 + kAttnRows <= end) {      // a whole tile: one wave-uniform origin
            const char* tile = reinterpret_cast<const char*>(base + row0 * stride);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                if constexpr (E == 4) {
                    const float4p q = *reinterpret_cast<const float4p*>(tile + off.at[r]);
                    v[r][0] = q.x, v[r][1] = q.y, v[r][2] = q.z, v[r][3] = q.w;
                } else if constexpr (E == 2) {
                    const float2p q = *reinterpret_cast<const float2p*>(tile + off.at[r]);
                    v[r][0] = q.x, v[r][1] = q.y;
                } else {
                    v[r][0] = *reinterpret_cast<const float*>(tile + off.at[r]);
                }
            }
        } else {
            const int c = (threadIdx.x & 31) * E, r0 = (threadIdx.x >> 5) * 4;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float* row = base + min(row0 + r0 + r, end - 1) * stride;
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const float x = row[min(c + e, D - 1)];
                    v[r][e] = row0 + r0 + r < end && c + e < D ? x : 0.0f;
                }
            }
        }
    }
    // `factors`: where a mixed tile (row0 its first row, `end` as in load) leaves the reciprocals of its rows' scales
    template <bool ROWS, bool COLS>
    __device__ __forceinline__ void store(unsigned short* rows, unsigned short* cols, float tile_scale, const ScaleArray& scales, float* factors, int row0, int end) const {
        if (__builtin_expect(tile_scale != 0.0f, 1)) {
            const float scale[4] = {tile_scale, tile_scale, tile_scale, tile_scale};
            store<ROWS, COLS>(rows, cols, scale);
        } else {
            float scale[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int row = min(row0 + (int)(threadIdx.x >> 5) * 4 + r, end - 1);
                scale[r] = scales.rows[row];
                if ((threadIdx.x & 31) == 0) factors[(threadIdx.x >> 5) * 4 + r] = reciprocal_power(scale[r]) * (scales.weights ? scales.weights[row] : 1.0f);
            }
            store<ROWS, COLS>(rows, cols, scale);
        }
    }
    template <bool ROWS, bool COLS>
    __device__ __forceinline__ void store(unsigned short* rows, unsigned short* cols, const float (&scale)[4]) const {
        const int c = (threadIdx.x & 31) * E, rb = threadIdx.x >> 5;
        const int pos = 16 * (rb >> 2) + 8 * (rb & 1) + 4 * ((rb >> 1) & 1);
        Terms t[E][2];
#pragma unroll
        for (int e = 0; e < E; ++e) {
            t[e][0] = split2(v[0][e], v[1][e], scale[0], scale[1]);
            t[e][1] = split2(v[2][e], v[3][e], scale[2], scale[3]);
        }
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            if (COLS) {
#pragma unroll
                for (int e = 0; e < E; ++e)
                    *reinterpret_cast<uint2*>(cols + n * kColPlane + (c + e) * kColPitch + pos) = make_uint2(t[e][0].t[n], t[e][1].t[n]);
            }
            if (ROWS) {
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    unsigned short* to = rows + n * kRowPlane + (4 * rb + r) * kRowPitch + c;
                    if constexpr (E == 1) {
                        *to = (unsigned short)(t[0][r >> 1].t[n] >> (16 * (r & 1)));
                    } else {
                        unsigned w[E / 2];
#pragma unroll
                        for (int e = 0; e < E; e += 2)      // the same half of two columns' words
                            w[e / 2] = __builtin_amdgcn_perm(t[e + 1][r >> 1].t[n], t[e][r >> 1].t[n], (r & 1) ? 0x07060302u : 0x05040100u);
                        if constexpr (E == 2) *reinterpret_cast<unsigned*>(to) = w[0];
                        else *reinterpret_cast<uint2*>(to) = make_uint2(w[0], w[1]);
                    }
                }
            }
        }
    }
};

// The lane's column as a B operand: d = 16 s + 8 half + 0..7 in step s.
template <int DP>
struct Column {
    Frag s[DP / 16];
    float v[DP / 2];
    __device__ __forceinline__ void load(const float* row, bool valid, int D) {
        const int half = (threadIdx.x & 63) >> 5;
#pragma unroll
        for (int i = 0; i < DP / 8; ++i) {
            const float4 x = valid ? load4(row, 16 * (i >> 1) + 8 * half + 4 * (i & 1), D) : make_float4(0, 0, 0, 0);
            v[4 * i] = x.x, v[4 * i + 1] = x.y, v[4 * i + 2] = x.z, v[4 * i + 3] = x.w;
        }
    }
    // largest magnitude of the whole column (both halves)
    __device__ __forceinline__ float top() const {
        float t = 0.0f;
#pragma unroll
        for (int i = 0; i < DP / 2; ++i) t = fmaxf(t, fabsf(v[i]));
        return fmaxf(t, __shfl_xor(t, 32));
    }
    // odd: the sign of the odd steps (see product_rows)
    __device__ __forceinline__ void split(float scale, float odd) {
#pragma unroll
        for (int i = 0; i < DP / 16; ++i) {
            const float f = i & 1 ? odd * scale : scale;
            const float x[8] = {v[8 * i] * f, v[8 * i + 1] * f, v[8 * i + 2] * f, v[8 * i + 3] * f,
                                v[8 * i + 4] * f, v[8 * i + 5] * f, v[8 * i + 6] * f, v[8 * i + 7] * f};
            s[i] = split8(x);
        }
    }
};

// The operands of each step are read from LDS before the matrix instructions of the step in front of it (the backward
// pass of 16 heads of 2047, 128 columns, one wavefront a SIMD: 661 -> 616 us; at 64 columns and below 1-2 %).
template <int STEPS>
__device__ __forceinline__ void reads_ahead() {
    __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
        if (i + 1 < STEPS) __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
        __builtin_amdgcn_sched_group_barrier(0x8, 3, 0);
    }
}
// sum_d tile[row][d] * column[d].  A matrix instruction aligns the products it adds and cuts their
// last bits, always downwards.  That shift is some 1e-8 of the result, nothing in itself, but it has the
// same sign everywhere, and the gradient of the bias sums millions of nearly cancelling ds: APART
// sums even and odd steps apart, the column's odd ones negated; in their difference the shifts cancel.
template <int DP, bool APART>
__device__ __forceinline__ v16f product_rows(const unsigned short* rows, const Column<DP>& col) {
    const int lane = threadIdx.x & 63;
    const unsigned short* at = rows + (lane & 31) * Tile<DP>::kRowPitch + 8 * (lane >> 5);
    v16f sum = {}, odd = {};
    const auto read = [&](int i) {
        Frag f;
#pragma unroll
        for (int n = 0; n < 2; ++n) f.t[n] = *reinterpret_cast<const v8h*>(at + n * Tile<DP>::kRowPlane + 16 * i);
        return f;
    };
    Frag next = read(0);
#pragma unroll
    for (int i = 0; i < DP / 16; ++i) {
        const Frag f = next;
        if (i + 1 < DP / 16) next = read(i + 1);
        if (APART && (i & 1)) odd = mul_step(odd, f, col.s[i]);
        else sum = mul_step(sum, f, col.s[i]);
    }
    reads_ahead<DP / 16>();
    return APART ? sum - odd : sum;
}
__device__ __forceinline__ int tile_row(int r) { return 8 * (r >> 2) + 4 * ((threadIdx.x & 63) >> 5) + (r & 3); }
// v of lane ^ 32
__device__ __forceinline__ float other_half(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float((threadIdx.x & 32) ? r[0] : r[1]);
}
// Scores are kept in powers of two (times log2 e): the exponential is then one instruction.
constexpr float kLn2 = 0.6931471805599453f, kLowest = -3.4028234663852886e38f;
__device__ __forceinline__ float pow2(float x) { return __builtin_amdgcn_exp2f(x); }      // below 2^-126 it is 0
// x log2 e; finite values stay finite at the lower end (a bias of the lowest float)
__device__ __forceinline__ float to_log2(float x) { return x < -1e38f && x >= kLowest ? fmaxf(x * kLog2e, kLowest) : x * kLog2e; }
// log sum exp from the reference of a row's exponentials (in powers of two) and their sum; the lowest float stays what it is
__device__ __forceinline__ float log_sum(float ref, float sum) { return ref == kLowest ? ref : ref * kLn2 + logf(sum); }
// What the backward pass takes from a row's scores, p = 2^(s - this).  Infinity, that is p = 0, for a row that saw nothing,
// and for one whose lse has no digits behind the point: next to 2^22 a rounding of it is a factor in p.  The lowest
// float is exact: p is 1 for every key there, and the row's weight (attn_scale_kernel) has their number.
__device__ __forceinline__ float row_reference(float lse) {
    return lse == kLowest ? lse : fabsf(lse) >= 0x1p22f ? INFINITY : lse * kLog2e;
}

// What undoes the scales of a tile's rows: one factor, or 32 in LDS where the rows are mixed.  A product of such a tile is
// multiplied row by row, by a branch around 16 multiplications that the other tiles do without.
struct TileRows {
    const float* at;
    float one;
    bool mixed;
    __device__ __forceinline__ TileRows(float tile_scale, const float* factors)
        : at(factors), one(tile_scale != 0.0f ? reciprocal_power(tile_scale) : 1.0f), mixed(__builtin_expect(tile_scale == 0.0f, 0)) {}
    __device__ __forceinline__ float exponent() const { return (float)__builtin_amdgcn_frexp_expf(one) - 1.0f; }      // of one
    // v, but for the factor `one`
    __device__ __forceinline__ void undo(v16f& v) const {
        if (__builtin_expect(mixed, 0)) {
            const float* f = at + 4 * ((threadIdx.x & 63) >> 5);
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const float4 x = *reinterpret_cast<const float4*>(f + 8 * g);
                v[4 * g] *= x.x, v[4 * g + 1] *= x.y, v[4 * g + 2] *= x.z, v[4 * g + 3] *= x.w;
            }
        }
    }
};
__device__ __forceinline__ float magnitude(const v16f& v) {
    float top = fabsf(v[0]);
#pragma unroll
    for (int r = 1; r < 16; ++r) top = fmaxf(top, fabsf(v[r]));
    return fmaxf(top, other_half(top));
}
// An operand of a tile by columns.
template <int DP>
__device__ __forceinline__ Frag read_cols(const unsigned short* cols, int block, int step) {
    const int lane = threadIdx.x & 63;
    const unsigned short* at = cols + (32 * block + (lane & 31)) * Tile<DP>::kColPitch + 8 * (lane >> 5) + 16 * step;
    return {{*reinterpret_cast<const v8h*>(at), *reinterpret_cast<const v8h*>(at + Tile<DP>::kColPlane)}};
}
// The lane's column of 32 rows as a B operand of two steps.
__device__ __forceinline__ void split16(Frag (&b)[2], const v16f& w) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const float v[8] = {w[8 * i], w[8 * i + 1], w[8 * i + 2], w[8 * i + 3], w[8 * i + 4], w[8 * i + 5], w[8 * i + 6], w[8 * i + 7]};
        b[i] = split8(v);
    }
}
// acc[d][column] += sum over a tile's rows of x[row][d] * w[row][column].  `cols` has x by columns, each row times its
// scale, `rows` the reciprocals, which go over to w.  A lane brings the largest of its column's terms to [2^14, 2^15)
// and adds what the tile gives to acc on the vector units, with the power of two undone: tiles do not share a scale,
// and acc is rounded where a matrix instruction would cut it.
template <int DP>
__device__ __forceinline__ void add_tile(v16f (&acc)[DP / 32], const unsigned short* cols, const TileRows& rows, v16f w) {
    rows.undo(w);
    const float scale = power_scale(magnitude(w)), back = reciprocal_power(scale) * rows.one;
    Frag b[2];
    split16(b, w * scale);
#pragma unroll
    for (int d = 0; d < DP / 32; ++d) {
        const v16f part = mul_step(mul_step(v16f{}, read_cols<DP>(cols, d, 0), b[0]), read_cols<DP>(cols, d, 1), b[1]);
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[d][r] = __builtin_fmaf(part[r], back, acc[d][r]);
        if (d & 1) __builtin_amdgcn_sched_barrier(0);
    }
}

// Forward: s * unscale + bias for a score tile of origin rel0, rows = keys.
template <bool BIAS>
__device__ __forceinline__ void scores(v16f& s, float unscale, const BucketRule& rule, const float* win, int rel0) {
    if (!BIAS) {
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] *= unscale;
    } else if (far_tile(rule, rel0)) {
        const float v = win[rel0 < 0 ? 0 : bias_window(rule) - 1];
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = __builtin_fmaf(s[r], unscale, v);
    } else {
        const float* at = win + bias_reach(rule) + rel0 + 4 * ((threadIdx.x & 63) >> 5) - (int)(threadIdx.x & 31);
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = __builtin_fmaf(s[r], unscale, at[8 * (r >> 2) + (r & 3)]);
    }
}
// Backward: the bias of a score tile of origin rel0 (sign 1: rows are keys, -1: queries), -inf where hide(r) says so if
// any element may be hidden.  It is read before the tile's products, which leaves no branch between them and what the
// vector units do with their results, so that both can run at once: 16 heads of 2047, 128 columns 620 -> 544 us, 64 columns
// 285 -> 266, 32 heads of 1000, 32 columns 128 -> 113.  (The forward pass loses by the registers it takes: 157 -> 159 us.)
// For the same reason the backward kernels do not skip a wavefront's hidden tiles: at 128 columns the compiler carried the
// running sums between the two register files around that branch (728 us with it, 667 without).
// 64 columns with dropout read it after the products: 2 wavefronts a SIMD leave no registers for both the bias and the
// generator (8 x 8 heads of 512, padded: 127 us before, 118 after).
constexpr bool shifts_early(int DP, bool DROP) { return !(DROP && DP == 64); }
template <bool BIAS, class Hide>
__device__ __forceinline__ v16f shifts(const BucketRule& rule, const float* win, int rel0, int sign, bool edge, Hide hide) {
    v16f b = {};
    if (BIAS) {
        if (far_tile(rule, rel0)) {
            b = win[rel0 < 0 ? 0 : bias_window(rule) - 1];
        } else {
            const float* at = win + bias_reach(rule) + rel0 + sign * (4 * ((threadIdx.x & 63) >> 5) - (int)(threadIdx.x & 31));
#pragma unroll
            for (int r = 0; r < 16; ++r) b[r] = at[sign * (8 * (r >> 2) + (r & 3))];
        }
    }
    if (edge) {
#pragma unroll
        for (int r = 0; r < 16; ++r) b[r] = hide(r) ? -INFINITY : b[r];
    }
    return b;
}
// Between LDS writes and reads of one wavefront, by different lanes.
__device__ __forceinline__ void wave_lds_fence() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}
constexpr int kSquare = 32 * 32;
__device__ __forceinline__ int square_at(int d, int row) { return d * 32 + (row ^ (d & 7) << 2); }

struct Where {
    int b, h, tile;
};
// Workgroups of one head follow each other on one XCD (ids go round the eight of them), so that its
// keys and values are read into one L2.  Under a causal mask the tiles of a head differ in work, and
// the ones that come last decide the time: there all heads' heaviest tiles come first (its last
// ones for blocks of queries, its first for blocks of keys).
enum TileOrder { kByHead, kHeavyLast, kHeavyFirst };      // where a head's heaviest tiles are
__device__ __forceinline__ Where where(const Attn& a, int tiles, TileOrder order) {
    const int heads = a.B * a.H, group = heads % kNumXCD == 0 ? kNumXCD : 1;
    const int slot = blockIdx.x / group, per = heads / group;
    const bool by_tile = a.causal && order != kByHead;
    int head = by_tile ? slot % per : slot / tiles, tile = by_tile ? slot / per : slot % tiles;
    head = head * group + blockIdx.x % group;
    if (by_tile && order == kHeavyLast) tile = tiles - 1 - tile;
    return {head / a.H, head % a.H, tile};
}
__device__ __forceinline__ int length_of(const int* lengths, int b, int T) {
    if (!lengths) return T;
    const int n = lengths[b];
    return n < 0 ? 0 : n > T ? T : n;
}

// Position of a sequence's first query among its keys.
constexpr int kMaxOffset = (1 << 29) - 1;
__device__ __forceinline__ int offset_of(const Attn& a, int b) {
    if (!a.q_offsets) return a.q_offset;
    return min(max(a.q_offsets[b], -kMaxOffset), kMaxOffset);
}

// Sum over aligned groups of N lanes (8, 16 or 32); every lane gets it.
template <int N>
__device__ __forceinline__ float group_sum(float x) {
    auto add = [](float v, auto ctrl) {
        return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), decltype(ctrl)::value, 0xf, 0xf, true));
    };
    x = add(x, std::integral_constant<int, 0xB1>());       // lane ^ 1
    x = add(x, std::integral_constant<int, 0x4E>());       // lane ^ 2
    x = add(x, std::integral_constant<int, 0x141>());      // mirrored within 8: the other quad
    if (N >= 16) x = add(x, std::integral_constant<int, 0x140>());      // mirrored within 16: the other eight
    if (N >= 32) x += __shfl_xor(x, 16);
    return x;
}

// Largest over aligned groups of N lanes (8, 16 or 32) of values that are not negative; every lane gets it.
template <int N>
__device__ __forceinline__ float group_max(float x) {
    auto top = [](float v, auto ctrl) {
        return fmaxf(v, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), decltype(ctrl)::value, 0xf, 0xf, true)));
    };
    x = top(x, std::integral_constant<int, 0xB1>());
    x = top(x, std::integral_constant<int, 0x4E>());
    x = top(x, std::integral_constant<int, 0x141>());
    if (N >= 16) x = top(x, std::integral_constant<int, 0x140>());
    if (N >= 32) x = fmaxf(x, __shfl_xor(x, 16));
    return x;
}

// ---- the rows' scales

// What the workgroups of a call have in common, worked out once: the powers of two that the products of the arrays staged
// through LDS are formed with, for each tile of 32 rows (within the length) and for each row; and the bias by relative
// position, [head of H][window], in the grid's last row.  A tile's scale brings its largest magnitude (values that are no
// numbers left out) to [2^14, 2^15), unless a row, not all zeros, is smaller by more than 2^8: there it is 0, and each row's brings
// its own.  So the 22 bits of a row reach down to 2^-9 of its largest value at least, whatever other rows hold.
//
// With go comes lse.  A row whose lse is the lowest float has nothing but keys of that bias, p is 1 for each of them in the
// backward kernels, and go and go . o get the reciprocal of their number as a weight (1 for all other rows).  Its tile
// counts as mixed.
struct ScaledArrays {
    const float* base[4];
    int keys[4];      // 1: laid out and limited as k, 0: as q
    const float* lse;      // of the fourth
};
// Where they are: of each array first the tiles', [head][tile], then the rows', [head][row].
struct Scales {
    const float *arrays, *window, *weights;      // weights of the rows of the fourth, [head][row]
    long start[4];
    int heads;
    __device__ __forceinline__ ScaleArray of(int array, int head, int T) const {
        const int tiles = (T + kAttnRows - 1) / kAttnRows;
        const float* at = arrays + start[array];
        return {at + (long)head * tiles, at + (long)heads * tiles + (long)head * T, array == 3 ? weights + (long)head * T : nullptr};
    }
};
// How many keys a query may see that are not switched off by a bias of -inf.
__device__ __forceinline__ int keys_in_sight(const Attn& a, int b, int h, int query) {
    const int q_offset = offset_of(a, b);
    int end = length_of(a.k_lengths, b, a.Tk), n = 0;
    if (a.causal) end = min(end, query + q_offset + 1);
    if (!a.table) return end;
    for (int j = 0; j < end; ++j) n += a.table[(long)bucket_of(a.rule, j - query - q_offset) * a.H + h] >= kLowest ? 1 : 0;
    return n;
}
// BACKWARD: with lse and weights.
template <int DP, bool BACKWARD>
__global__ __launch_bounds__(kAttnThreads) void attn_scale_kernel(Attn a, ScaledArrays arrays, Scales scales, int n_arrays, int runs) {
    constexpr int LANES = DP / 4, STEP = kAttnThreads / LANES, DEEP = 8;
    __shared__ float tops[kAttnThreads];
    const int n = blockIdx.y;
    if (n == n_arrays) {
        const int size = bias_window(a.rule);
        const long total = (long)size * a.H;
        for (long i = (long)blockIdx.x * kAttnThreads + threadIdx.x; i < total; i += (long)gridDim.x * kAttnThreads)
            const_cast<float*>(scales.window)[i] = to_log2(a.table[(long)bucket_of(a.rule, (int)(i % size) - bias_reach(a.rule)) * a.H + i / size]);
        return;
    }
    const int head = blockIdx.x / runs, at = blockIdx.x % runs, b = head / a.H, h = head % a.H, keys = arrays.keys[n];
    const int T = keys ? a.Tk : a.Tq, end = length_of(keys ? a.k_lengths : a.q_lengths, b, T);
    // a run is a multiple of the 256 rows that the workgroup has in hand at a time
    const long run = ((long)T + runs * kAttnThreads - 1) / (runs * kAttnThreads) * kAttnThreads;
    const int first = (int)min((long)end, at * run), last = (int)min((long)end, first + run), lane = threadIdx.x % LANES;
    const long stride = keys ? a.k_t : a.q_t;
    const float* base = arrays.base[n] + (keys ? b * a.k_b + h * a.k_h : b * a.q_b + h * a.q_h);
    const ScaleArray to = scales.of(n, head, T);
    for (int c0 = first; c0 < last; c0 += kAttnThreads) {
#pragma unroll
        for (int u0 = 0; u0 < kAttnThreads / STEP; u0 += DEEP) {
            const int r0 = c0 + u0 * STEP + threadIdx.x / LANES;
            float4 v[DEEP];
#pragma unroll
            for (int u = 0; u < DEEP; ++u) v[u] = load4(base + min(r0 + u * STEP, last - 1) * stride, 4 * lane, a.D);
#pragma unroll
            for (int u = 0; u < DEEP; ++u) {
                const float x[4] = {fabsf(v[u].x), fabsf(v[u].y), fabsf(v[u].z), fabsf(v[u].w)};
                float top = 0.0f;
#pragma unroll
                for (int e = 0; e < 4; ++e) top = fmaxf(top, x[e] <= -kLowest ? x[e] : 0.0f);
                top = group_max<LANES>(top);
                if (lane == 0) tops[r0 + u * STEP - c0] = r0 + u * STEP < last ? top : 0.0f;
            }
        }
        __syncthreads();
        const float top = tops[threadIdx.x], tile = group_max<kAttnRows>(top);
        const int row = c0 + threadIdx.x;
        const bool lowest = BACKWARD && n == 3 && row < last && arrays.lse[(long)head * T + row] == kLowest;
        const bool mixed = group_max<kAttnRows>(lowest || (top > 0.0f && top < 0x1p-8f * tile) ? 1.0f : 0.0f) > 0.0f;
        if (BACKWARD && n == 3 && row < last) const_cast<float*>(to.weights)[row] = lowest ? 1.0f / (float)max(1, keys_in_sight(a, b, h, row)) : 1.0f;
        if (row < last) {
            const_cast<float*>(to.rows)[row] = power_scale(top);
            if (threadIdx.x % kAttnRows == 0) const_cast<float*>(to.tiles)[row / kAttnRows] = mixed ? 0.0f : power_scale(tile);
        }
        __syncthreads();
    }
}
__device__ __forceinline__ void copy_bias(const Attn& a, const float* window, int head, float* win) {
    const int n = bias_window(a.rule);
    for (int s = threadIdx.x; s < n; s += kAttnThreads) win[s] = window[(long)head * n + s];
}
// Which of a tile's 16 elements of a lane are hidden; rows are keys, the column is a query.
__device__ __forceinline__ bool hidden(const Attn& a, int key, int query, int k_end, int q_offset) {
    return key >= k_end || (a.causal && key > query + q_offset);
}

// ---------------------------------------------------------------- forward

// o and lse of a block of 128 queries, or of a run of its keys.  8x16 heads of 1024, 64 columns, padded, 21.7 GFLOP of the
// formulas' products: 126 us (and 13 for the scales; one power of two a head, without regard to what its rows hold, took 117).
// The matrix cores are 0.30 busy beside 10.5 other vector instructions a matrix instruction, about half the time together: a
// tile's products and its softmax follow each other, with two barriers for each 32 keys, and three wavefronts a SIMD fill the
// gaps in part (two take the same time).  With dropout of 0.1 139 us; 166 where every tile's rows of v are mixed, 185 with
// those of k too.
template <int DP, bool BIAS, bool DROP>
__global__ __launch_bounds__(kAttnThreads, DP == 128 ? 2 : 3) void attn_fwd_kernel(Attn a, Scales scales, float* o, float* lse, float* part, float2* part_ml, int tiles, int splits) {
    extern __shared__ __align__(16) unsigned short lds[];
    unsigned short *kt = lds, *vt = kt + Tile<DP>::kRowBytes / 2;
    float* krows = reinterpret_cast<float*>(vt + Tile<DP>::kColBytes / 2);      // reciprocal scales of the tile's rows of k, of v
    float *vrows = krows + kAttnRows, *win = vrows + kAttnRows;
    const Where w = where(a, tiles * splits, kHeavyLast);
    const int split = w.tile % splits, q0 = w.tile / splits * kAttnCols;
    const int lane = threadIdx.x & 63, qw = q0 + (threadIdx.x >> 6) * 32, query = qw + (lane & 31);
    const int q_end = length_of(a.q_lengths, w.b, a.Tq), k_end = length_of(a.k_lengths, w.b, a.Tk), q_offset = offset_of(a, w.b);
    const float* kbase = a.k + w.b * a.k_b + w.h * a.k_h;
    const float* vbase = a.v + w.b * a.k_b + w.h * a.k_h;
    const long qrow = w.b * a.q_b + w.h * a.q_h + query * a.q_t;
    if (BIAS) copy_bias(a, scales.window, w.h, win);
    // keys this workgroup walks: to the last one its last query sees, cut into `splits` runs of whole tiles
    int last = k_end;
    if (a.causal) last = min(last, max(0, min(q0 + kAttnCols, q_end) + q_offset));
    if (q0 >= q_end) last = 0;
    const int run = (last + kAttnRows * splits - 1) / (kAttnRows * splits) * kAttnRows;
    const int first = split * run;
    last = min(last, first + run);

    const ScaleArray kscales = scales.of(0, w.b * a.H + w.h, a.Tk), vscales = scales.of(1, w.b * a.H + w.h, a.Tk);
    Column<DP> qcol;
    qcol.load(a.q + qrow, query < q_end, a.D);
    const float qscale = power_scale(qcol.top());
    qcol.split(qscale, 1.0f);
    const float unscale = a.scale * kLog2e * reciprocal_power(qscale);      // of a score, beside its key's
    RngState rng = {};
    unsigned long long group0 = 0;
    if (DROP) {
        rng = load_rng(a.rng, a.channel);
        group0 = ((unsigned long long)(w.b * a.H + w.h) * a.Tq + query) * ((a.Tk + 15) / 16) * 2 + (lane >> 5);
    }
    v16f acc[DP / 32] = {};
    float ref = -INFINITY, from = 0.0f, l = 0.0f;      // the exponentials are 2^(s - from); from = ref once a key was seen
    float e = -INFINITY, limit = INFINITY;             // acc is the sum of p v times 2^e, -inf while there was nothing to add
    const auto rescale = [&](float f) __attribute__((always_inline)) {
#pragma unroll
        for (int d = 0; d < DP / 32; ++d)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[d][r] *= f;
    };
    // Settles e for terms p v of this size: the first to [2^10, 2^11), lowered where one outgrows 2^15 (as seldom); returns
    // what acc has to be multiplied by.
    const auto settle = [&](float largest) __attribute__((always_inline)) {
        const bool unset = e == -INFINITY, change = unset ? largest > 0.0f : ldexpf(largest, (int)e) > 0x1p15f;
        const int to = (int)min(268u - (__float_as_uint(largest) >> 23 & 255u), 253u) - 131;
        const float f = !change ? 1.0f : unset ? 0.0f : ldexpf(1.0f, to - (int)e);
        e = change ? (float)to : e;
        return f;
    };
    const typename Tile<DP>::Offsets off(a.k_t, a.D);
    Tile<DP> kr, vr;
    float knext = 1.0f, vnext = 1.0f;      // the scales of the tiles on their way
    if (first < last) {
        kr.load(off, kbase, a.k_t, first, last, a.D);
        vr.load(off, vbase, a.k_t, first, last, a.D);
        knext = tile_scale(kscales.tiles, first / kAttnRows);
        vnext = tile_scale(vscales.tiles, first / kAttnRows);
    }
    for (int j0 = first; j0 < last; j0 += kAttnRows) {
        const float kscale = knext, vscale = vnext;
        __syncthreads();
        kr.template store<true, false>(kt, nullptr, kscale, kscales, krows, j0, last);
        vr.template store<false, true>(nullptr, vt, vscale, vscales, vrows, j0, last);
        __syncthreads();
        if (j0 + kAttnRows < last) {
            kr.load(off, kbase, a.k_t, j0 + kAttnRows, last, a.D);
            vr.load(off, vbase, a.k_t, j0 + kAttnRows, last, a.D);
            knext = tile_scale(kscales.tiles, j0 / kAttnRows + 1);
            vnext = tile_scale(vscales.tiles, j0 / kAttnRows + 1);
        }
        if (qw >= q_end || (a.causal && j0 > qw + 31 + q_offset)) continue;      // nothing here for this wavefront
        const int rel0 = j0 - qw - q_offset;
        v16f s = product_rows<DP, false>(kt, qcol);
        const TileRows key_rows(kscale, krows), value_rows(vscale, vrows);
        key_rows.undo(s);
        scores<BIAS>(s, unscale * key_rows.one, a.rule, win, rel0);
        if (j0 + kAttnRows > k_end || (a.causal && j0 + kAttnRows - 1 > qw + q_offset)) {
#pragma unroll
            for (int r = 0; r < 16; ++r)
                if (hidden(a, j0 + tile_row(r), query, k_end, q_offset)) s[r] = -INFINITY;
        }
        float top = s[0];
#pragma unroll
        for (int r = 1; r < 16; ++r) top = fmaxf(top, s[r]);
        top = fmaxf(top, other_half(top));
        // What keeps the exponentials and the terms p v in range changes seldom, and one test finds that it must: the reference, a
        // whole number, follows the running maximum where that is 2^7 above it; the terms' scale is lowered where one outgrows
        // it.  In a tile with one factor the scale goes into the exponent and comes out of the sum (lift), unless the sum would
        // lose by it or the difference of the two is not exact: such tiles, and mixed ones, are scaled apart.
        const float one = value_rows.exponent();
        float lift = e + one;
        bool apart = false;
        if (value_rows.mixed || __any((top > ref + 7.0f) | (top + one > limit) | !(fabsf(lift) <= 40.0f))) {
            const float to = top > ref + 7.0f ? ceilf(top) : ref;
            float f = to == -INFINITY ? 0.0f : pow2(ref - to);
            ref = to;
            from = ref == -INFINITY ? 0.0f : ref;
            l *= f;
            if (!value_rows.mixed) f *= settle(pow2(top - from) * value_rows.one);
            rescale(f);
            lift = e == -INFINITY ? 0.0f : e + one;
            apart = value_rows.mixed || __any((fabsf(lift) > 40.0f) | (fabsf(from) >= 0x1p20f));
            if (apart) lift = 0.0f;
            limit = fabsf(from) < 0x1p20f ? from + 15.0f - e : -INFINITY;
        }
        const float lifted = from - lift;
        float part_l[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            s[r] = pow2(s[r] - lifted);
            part_l[r & 3] += s[r];
        }
        l += ldexpf((part_l[0] + part_l[1]) + (part_l[2] + part_l[3]), -(int)lift);
        asm volatile("" : "+v"(l));      // summed here: the branch below would otherwise take a copy of all terms along
        if (DROP) {
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                unsigned u[4];
                random_group(rng, group0 + 2ull * (j0 / 16 + b), u);
#pragma unroll
                for (int i = 0; i < 8; ++i) s[8 * b + i] = random16(u, i) >= a.rate.threshold ? s[8 * b + i] : 0.0f;      // scaled at the end
            }
        }
        if (__builtin_expect(apart, 0)) {
            value_rows.undo(s);
            rescale(settle(magnitude(s) * value_rows.one));
            if (fabsf(from) < 0x1p20f) limit = from + 15.0f - e;
#pragma unroll
            for (int r = 0; r < 16; ++r) s[r] = ldexpf(s[r] * value_rows.one, (int)e);
        }
        Frag b[2];
        split16(b, s);
        Frag next = read_cols<DP>(vt, 0, 0);
#pragma unroll
        for (int i = 0; i < DP / 16; ++i) {
            const Frag x = next;
            if (i + 1 < DP / 16) next = read_cols<DP>(vt, (i + 1) % (DP / 32), (i + 1) / (DP / 32));
            acc[i % (DP / 32)] = mul_step(acc[i % (DP / 32)], x, b[i / (DP / 32)]);
        }
        reads_ahead<DP / 16>();
    }
    if (query >= a.Tq) return;
    l += other_half(l);
    const float back = e == -INFINITY ? 1.0f : ldexpf(1.0f, -(int)e);
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[d][r] = acc[d][r] * back * (DROP ? a.rate.scale : 1.0f);
    const int half4 = 4 * (lane >> 5);
    const long stat = ((long)w.b * a.H + w.h) * a.Tq + query;
    if (splits > 1) {
        const long row = (long)split * a.B * a.H * a.Tq + stat;
#pragma unroll
        for (int d = 0; d < DP / 32; ++d)
#pragma unroll
            for (int g = 0; g < 4; ++g)
                store4(part + row * a.D, 32 * d + 8 * g + half4, a.D, acc[d][4 * g], acc[d][4 * g + 1], acc[d][4 * g + 2], acc[d][4 * g + 3]);
        if (half4 == 0) part_ml[row] = make_float2(ref, l);
        return;
    }
    const bool saw = query < q_end && l != 0.0f;      // a row that saw no key is zero, whatever the values hold
    const float inv = 1.0f / l;
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
        for (int g = 0; g < 4; ++g) store_scaled(o + qrow, 32 * d + 8 * g + half4, a.D, acc[d], g, saw, inv);
    if (half4 == 0) lse[stat] = saw ? log_sum(ref, l) : -INFINITY;
}

// o and lse from the pieces of a split key axis.  DP / 4 lanes take a row's columns, TEAMS such groups a row: team t
// sums pieces t, t + TEAMS, ... in order, then the teams' sums are added in order through LDS.  One team a row while
// there are few pieces, the workgroup's 256 threads a row where one team would walk many, each a trip to memory.  Both
// sides, of the whole call (64 columns): one token, 16 heads, 8192 keys in 64 pieces 41 us with one team, 19 with 16;
// 4 x 128 queries, 32 pieces 35 / 31; 8 heads of 4096 queries in 3 pieces 148 / 174, of 1024 in 4 pieces 35 / 42.
constexpr int kJoinTeams = 6;      // pieces from which a row gets the workgroup
template <int DP, int TEAMS>
__global__ __launch_bounds__(kAttnThreads) void attn_join_kernel(Attn a, float* o, float* lse, const float* part, const float2* part_ml, int splits) {
    constexpr int LANES = DP / 4, ROWS = kAttnThreads / (LANES * TEAMS);
    __shared__ float4 sums[TEAMS > 1 ? TEAMS : 1][LANES];
    __shared__ float weights[TEAMS];
    const long rows = (long)a.B * a.H * a.Tq, row = (long)blockIdx.x * ROWS + threadIdx.x / (LANES * TEAMS);
    if (row >= rows) return;      // (TEAMS > 1: a row a workgroup, so all of it or none)
    const int team = threadIdx.x / LANES % TEAMS, c = threadIdx.x % LANES * 4, head = (int)(row / a.Tq), query = (int)(row - (long)head * a.Tq);
    const int b = head / a.H, h = head % a.H;
    const bool valid = query < length_of(a.q_lengths, b, a.Tq);
    float m = -INFINITY, l = 0.0f;
    if constexpr (TEAMS > 1) {
        for (int s = threadIdx.x & 63; s < splits; s += kWave) m = fmaxf(m, part_ml[s * rows + row].x);
#pragma unroll
        for (int d = 1; d < kWave; d <<= 1) m = fmaxf(m, __shfl_xor(m, d));
    } else {
        for (int s = 0; s < splits; ++s) m = fmaxf(m, part_ml[s * rows + row].x);
    }
    const float ref = m == -INFINITY ? 0.0f : m;
    float4 acc = make_float4(0, 0, 0, 0);
#pragma unroll 4
    for (int s = team; s < splits; s += TEAMS) {
        const float2 ml = part_ml[s * rows + row];
        const float f = pow2(ml.x - ref);
        const float4 v = load4(part + (s * rows + row) * a.D, c, a.D);
        l += ml.y * f;
        acc = make_float4(acc.x + v.x * f, acc.y + v.y * f, acc.z + v.z * f, acc.w + v.w * f);
    }
    if constexpr (TEAMS > 1) {
        sums[team][threadIdx.x % LANES] = acc;
        if (c == 0) weights[team] = l;
        __syncthreads();
        if (team) return;
        acc = make_float4(0, 0, 0, 0);
        l = 0.0f;
#pragma unroll
        for (int t = 0; t < TEAMS; ++t) {
            const float4 v = sums[t][threadIdx.x % LANES];
            l += weights[t];
            acc = make_float4(acc.x + v.x, acc.y + v.y, acc.z + v.z, acc.w + v.w);
        }
    }
    const bool saw = valid && l != 0.0f;
    const float inv = 1.0f / l;
    store4(o + b * a.q_b + h * a.q_h + query * a.q_t, c, a.D, saw ? acc.x * inv : 0.0f, saw ? acc.y * inv : 0.0f, saw ? acc.z * inv : 0.0f,
           saw ? acc.w * inv : 0.0f);
    if (c == 0) lse[row] = saw ? log_sum(m, l) : -INFINITY;
}

// ---------------------------------------------------------------- forward: a few queries against many keys

// One workgroup per head and run of keys; up to NQ queries share what is read.  DP / 4 lanes hold a
// key's columns, so a wavefront's load covers 256 / DP neighbouring keys, and kTokenUnroll of those
// are in flight at once.  Every group of lanes keeps a running maximum, sum and result of its own
// keys; they are joined at the end, first in the wavefront, then through LDS, then (splits > 1) by
// attn_join_kernel.  No matrix instructions: up to four rows the time is that of reading k and v (one
// token of 16 sequences of 16 heads against 8192 keys, 64 columns, 1.07 GB: 188 us, 5.7 TB/s; four tokens
// 203 us), with eight the vector units bound it (268 us).
constexpr int kTokenUnroll = 4;
template <int DP, int NQ, bool BIAS>
__global__ __launch_bounds__(kAttnThreads) void attn_token_kernel(Attn a, float* o, float* lse, float* part, float2* part_ml, int splits) {
    constexpr int LANES = DP / 4, GROUPS = kWave / LANES, STEP = GROUPS * kTokenUnroll;      // keys per wavefront and trip
    extern __shared__ float win[];
    __shared__ float4 join_o[NQ][4][LANES];
    __shared__ float2 join_ml[NQ][4];
    const Where w = where(a, splits, kByHead);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane % LANES * 4, group = lane / LANES, split = w.tile;
    const int q_end = length_of(a.q_lengths, w.b, a.Tq), k_end = length_of(a.k_lengths, w.b, a.Tk), q_offset = offset_of(a, w.b);
    int last = k_end;
    if (a.causal) last = min(last, max(0, a.Tq + q_offset));
    if (q_end == 0) last = 0;
    const int run = (last + 4 * STEP * splits - 1) / (4 * STEP * splits) * 4 * STEP;
    const int first = split * run;
    last = min(last, first + run);
    if (BIAS && first < last) fill_bias(a, w.h, win);
    const int reach = BIAS ? bias_reach(a.rule) : 0;
    __syncthreads();
    const float* kbase = a.k + w.b * a.k_b + w.h * a.k_h;
    const float* vbase = a.v + w.b * a.k_b + w.h * a.k_h;
    const float qs = a.scale * kLog2e;
    float4 q[NQ], acc[NQ];
    float m[NQ], l[NQ];
#pragma unroll
    for (int i = 0; i < NQ; ++i) {
        q[i] = i < q_end ? load4(a.q + w.b * a.q_b + w.h * a.q_h + i * a.q_t, c, a.D) : make_float4(0, 0, 0, 0);
        q[i] = make_float4(q[i].x * qs, q[i].y * qs, q[i].z * qs, q[i].w * qs);
        acc[i] = make_float4(0, 0, 0, 0);
        m[i] = -INFINITY;
        l[i] = 0.0f;
    }
    for (int j0 = first + wave * STEP; j0 < last; j0 += 4 * STEP) {
        float4 kv[kTokenUnroll], vv[kTokenUnroll];
#pragma unroll
        for (int u = 0; u < kTokenUnroll; ++u) {
            const int j = j0 + u * GROUPS + group;
            kv[u] = j < last ? load4(kbase + j * a.k_t, c, a.D) : make_float4(0, 0, 0, 0);
        }
#pragma unroll
        for (int u = 0; u < kTokenUnroll; ++u) {
            const int j = j0 + u * GROUPS + group;
            vv[u] = j < last ? load4(vbase + j * a.k_t, c, a.D) : make_float4(0, 0, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < NQ; ++i) {
            float s[kTokenUnroll], top = m[i];
#pragma unroll
            for (int u = 0; u < kTokenUnroll; ++u) {
                const int j = j0 + u * GROUPS + group;
                s[u] = group_sum<LANES>(kv[u].x * q[i].x + kv[u].y * q[i].y + (kv[u].z * q[i].z + kv[u].w * q[i].w));
                if (BIAS) s[u] += win[reach + max(-reach, min(reach, j - i - q_offset))];
                if (j >= last || (a.causal && j > i + q_offset)) s[u] = -INFINITY;
                top = fmaxf(top, s[u]);
            }
            const float ref = top == -INFINITY ? 0.0f : top, f = pow2(m[i] - ref);
            m[i] = top;
            l[i] *= f;
            acc[i] = make_float4(acc[i].x * f, acc[i].y * f, acc[i].z * f, acc[i].w * f);
#pragma unroll
            for (int u = 0; u < kTokenUnroll; ++u) {
                const float p = pow2(s[u] - ref);
                l[i] += p;
                acc[i] = make_float4(acc[i].x + p * vv[u].x, acc[i].y + p * vv[u].y, acc[i].z + p * vv[u].z, acc[i].w + p * vv[u].w);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < NQ; ++i) {
        float top = m[i];
#pragma unroll
        for (int d = LANES; d < kWave; d <<= 1) top = fmaxf(top, __shfl_xor(top, d));
        const float f = pow2(m[i] - (top == -INFINITY ? 0.0f : top));
        l[i] *= f;
        acc[i] = make_float4(acc[i].x * f, acc[i].y * f, acc[i].z * f, acc[i].w * f);
#pragma unroll
        for (int d = LANES; d < kWave; d <<= 1) {
            l[i] += __shfl_xor(l[i], d);
            acc[i].x += __shfl_xor(acc[i].x, d);
            acc[i].y += __shfl_xor(acc[i].y, d);
            acc[i].z += __shfl_xor(acc[i].z, d);
            acc[i].w += __shfl_xor(acc[i].w, d);
        }
        if (group == 0) join_o[i][wave][lane] = acc[i];
        if (lane == 0) join_ml[i][wave] = make_float2(top, l[i]);
    }
    __syncthreads();
    for (int t = threadIdx.x; t < NQ * LANES; t += kAttnThreads) {
        const int i = t / LANES, col = t % LANES;
        if (i >= a.Tq) continue;
        float top = -INFINITY, sum = 0.0f;
        for (int o4 = 0; o4 < 4; ++o4) top = fmaxf(top, join_ml[i][o4].x);
        const float ref = top == -INFINITY ? 0.0f : top;
        float4 r = make_float4(0, 0, 0, 0);
        for (int o4 = 0; o4 < 4; ++o4) {
            const float f = pow2(join_ml[i][o4].x - ref);
            const float4 v = join_o[i][o4][col];
            sum += join_ml[i][o4].y * f;
            r = make_float4(r.x + v.x * f, r.y + v.y * f, r.z + v.z * f, r.w + v.w * f);
        }
        const long stat = ((long)w.b * a.H + w.h) * a.Tq + i;
        if (splits > 1) {
            const long row = (long)split * a.B * a.H * a.Tq + stat;
            store4(part + row * a.D, col * 4, a.D, r.x, r.y, r.z, r.w);
            if (col == 0) part_ml[row] = make_float2(top, sum);
        } else {
            const bool saw = i < q_end && sum != 0.0f;
            const float inv = 1.0f / sum;
            store4(o + w.b * a.q_b + w.h * a.q_h + i * a.q_t, col * 4, a.D, saw ? r.x * inv : 0.0f, saw ? r.y * inv : 0.0f, saw ? r.z * inv : 0.0f,
                   saw ? r.w * inv : 0.0f);
            if (col == 0) lse[stat] = saw ? log_sum(top, sum) : -INFINITY;
        }
    }
}

// ---------------------------------------------------------------- backward: queries

// gq, the row products go . o (for the other kernel) and one partial row of the table's gradient.  Bound by the vector
// instructions beside the matrix cores (10.5 a matrix instruction at 128 columns, 20 at 64 with dropout) and, at 128 columns, by one
// wavefront a SIMD: its operands q and go (128 registers), gq (64) and the tiles on their way take more than half of the registers.
// At 64 columns 4 registers (dropout; 14 without) go through scratch memory.  8x8 heads of 512, 64 columns, dropout, padded: 52 us; 2x8
// heads of 2047, 128 columns, causal: 187 us, the matrix cores 0.20 busy.
template <int DP, bool BIAS, bool DROP>
__global__ __launch_bounds__(kAttnThreads, DP == 128 ? 1 : 2) void attn_bwd_q_kernel(Attn a, Scales scales, const float* o, const float* lse, const float* go, float* gq,
    float* part, float* delta, float* part_table, int tiles, int splits) {
    extern __shared__ __align__(16) unsigned short lds[];
    unsigned short *kt = lds, *kc = kt + Tile<DP>::kRowBytes / 2, *vt = kc + Tile<DP>::kColBytes / 2;
    float* krows = reinterpret_cast<float*>(vt + Tile<DP>::kRowBytes / 2);      // reciprocal scales of the tile's rows of k, of v
    float *vrows = krows + kAttnRows, *square = vrows + kAttnRows;              // square: [wavefront][32][32]
    float* win = square + (BIAS ? 4 * kSquare : 0);
    const int window = BIAS ? bias_window(a.rule) : 0;
    float* diag = win + window;      // [wavefront][window]: sums of ds by relative position
    const Where w = where(a, tiles * splits, kHeavyLast);
    const int split = w.tile % splits, q0 = w.tile / splits * kAttnCols, lane = threadIdx.x & 63, wave = threadIdx.x >> 6, qw = q0 + wave * 32, query = qw + (lane & 31);
    const int q_end = length_of(a.q_lengths, w.b, a.Tq), k_end = length_of(a.k_lengths, w.b, a.Tk), q_offset = offset_of(a, w.b);
    const float* kbase = a.k + w.b * a.k_b + w.h * a.k_h;
    const float* vbase = a.v + w.b * a.k_b + w.h * a.k_h;
    const long qrow = w.b * a.q_b + w.h * a.q_h + query * a.q_t;
    if (BIAS) {
        copy_bias(a, scales.window, w.h, win);
        for (int s = threadIdx.x; s < 4 * window; s += kAttnThreads) diag[s] = 0.0f;
        __syncthreads();      // a workgroup without a key meets no other barrier before its wavefronts add to their sums
    }
    int last = k_end;
    if (a.causal) last = min(last, max(0, min(q0 + kAttnCols, q_end) + q_offset));
    if (q0 >= q_end) last = 0;
    const int run = (last + kAttnRows * splits - 1) / (kAttnRows * splits) * kAttnRows, first = split * run;
    last = min(last, first + run);
    const bool valid = query < q_end;
    const long stat = ((long)w.b * a.H + w.h) * a.Tq + query;
    float dl = 0.0f;
    if (valid) {
        const float *orow = o + qrow, *grow = go + qrow;
        for (int c = 4 * (lane >> 5); c < a.D; c += 8) {
            const float4 x = load4(orow, c, a.D), y = load4(grow, c, a.D);
            dl += (x.x * y.x + x.y * y.y) + (x.z * y.z + x.w * y.w);
        }
    }
    dl += other_half(dl);
    const ScaleArray kscales = scales.of(0, w.b * a.H + w.h, a.Tk), vscales = scales.of(1, w.b * a.H + w.h, a.Tk);
    Column<DP> qcol, gcol;
    qcol.load(a.q + qrow, valid, a.D);
    const float qscale = power_scale(qcol.top());
    qcol.split(qscale, 1.0f);
    gcol.load(go + qrow, valid, a.D);
    const float gscale = power_scale(gcol.top());
    gcol.split(gscale, -1.0f);
    const float unscale = a.scale * kLog2e * reciprocal_power(qscale);
    float dscale = reciprocal_power(gscale) * (DROP ? a.rate.scale : 1.0f);
    const float weight = valid ? scales.weights[stat] : 1.0f;
    dl *= weight;
    dscale *= weight;
    if (query < a.Tq && lane < 32 && split == 0) delta[stat] = dl;
    const float row_lse = valid ? row_reference(lse[stat]) : INFINITY;
    RngState rng = {};
    unsigned long long group0 = 0;
    if (DROP) {
        rng = load_rng(a.rng, a.channel);
        group0 = (unsigned long long)stat * ((a.Tk + 15) / 16) * 2 + (lane >> 5);
    }
    float far_before = 0.0f, far_after = 0.0f;
    v16f acc[DP / 32] = {};
    const typename Tile<DP>::Offsets off(a.k_t, a.D);
    Tile<DP> kr, vr;
    float knext = 1.0f, vnext = 1.0f;      // the scales of the tiles on their way
    if (first < last) {
        kr.load(off, kbase, a.k_t, first, last, a.D);
        vr.load(off, vbase, a.k_t, first, last, a.D);
        knext = tile_scale(kscales.tiles, first / kAttnRows);
        vnext = tile_scale(vscales.tiles, first / kAttnRows);
    }
    for (int j0 = first; j0 < last; j0 += kAttnRows) {
        const float kscale = knext, vscale = vnext;
        __syncthreads();
        kr.template store<true, true>(kt, kc, kscale, kscales, krows, j0, last);
        vr.template store<true, false>(vt, nullptr, vscale, vscales, vrows, j0, last);
        __syncthreads();
        if (j0 + kAttnRows < last) {
            kr.load(off, kbase, a.k_t, j0 + kAttnRows, last, a.D);
            vr.load(off, vbase, a.k_t, j0 + kAttnRows, last, a.D);
            knext = tile_scale(kscales.tiles, j0 / kAttnRows + 1);
            vnext = tile_scale(vscales.tiles, j0 / kAttnRows + 1);
        }
        const int rel0 = j0 - qw - q_offset;
        const bool edge = j0 + kAttnRows > k_end || (a.causal && j0 + kAttnRows - 1 > qw + q_offset);
        const auto tile_shifts = [&] {
            return shifts<BIAS>(a.rule, win, rel0, 1, edge, [&](int r) { return hidden(a, j0 + tile_row(r), query, k_end, q_offset); });
        };
        v16f shift;
        if constexpr (shifts_early(DP, DROP)) shift = tile_shifts();
        v16f s = product_rows<DP, false>(kt, qcol);
        v16f dp = product_rows<DP, true>(vt, gcol);
        const TileRows key_rows(kscale, krows), value_rows(vscale, vrows);
        key_rows.undo(s);
        value_rows.undo(dp);
        const float score_scale = unscale * key_rows.one, dp_scale = dscale * value_rows.one;
        if constexpr (!shifts_early(DP, DROP)) shift = tile_shifts();
        if (DROP) {
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                unsigned u[4];
                random_group(rng, group0 + 2ull * (j0 / 16 + b), u);
#pragma unroll
                for (int e = 0; e < 8; ++e) dp[8 * b + e] = random16(u, e) >= a.rate.threshold ? dp[8 * b + e] : 0.0f;
            }
        }
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const float p = pow2(__builtin_fmaf(s[r], score_scale, shift[r]) - row_lse);      // (0 for queries behind the last)
            s[r] = p * __builtin_fmaf(dp[r], dp_scale, -dl);
        }
        if (BIAS) {
            if (far_tile(a.rule, rel0)) {      // one bucket has the whole tile
                float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int r = 0; r < 16; ++r) sum[r & 3] += s[r];
                (rel0 < 0 ? far_before : far_after) += (sum[0] + sum[1]) + (sum[2] + sum[3]);
            } else {
                // Sums along the tile's 63 diagonals: element (row, column) goes to row (row - column) mod 32 of a
                // 32 x 32 square (its 16-byte units permuted by row), where lane l finds half of diagonals l and l - 32.  (Atomic additions in LDS
                // take about 180 cycles an instruction: 2900 for this tile, all wavefronts together.)
                float* sq = square + wave * kSquare;
                wave_lds_fence();
#pragma unroll
                for (int r = 0; r < 16; ++r) sq[square_at((tile_row(r) - lane) & 31, tile_row(r))] = s[r];
                wave_lds_fence();
                const int d = lane & 31, row0 = 16 * (lane >> 5);
                float same = 0.0f, less = 0.0f;       // diagonals d and d - 32
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float4 v = *reinterpret_cast<const float4*>(sq + square_at(d, row0 + 4 * i));
                    const float e[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                    for (int t = 0; t < 4; ++t) {
                        same += row0 + 4 * i + t >= d ? e[t] : 0.0f;
                        less += row0 + 4 * i + t >= d ? 0.0f : e[t];
                    }
                }
                same += other_half(same);
                less += other_half(less);
                // the wavefront's own sums by relative position: lanes 0-31 add the upper diagonals, 32-63 the lower
                float* mine = diag + wave * window + bias_reach(a.rule) + rel0 + d - (lane < 32 ? 0 : 32);
                if (lane != 32) *mine += lane < 32 ? same : less;      // (there is no diagonal -32)
            }
        }
        add_tile<DP>(acc, kc, key_rows, s);
    }
    if (query < a.Tq) {
        float* out = splits > 1 ? part + ((long)split * a.B * a.H * a.Tq + stat) * a.D : gq + qrow;
#pragma unroll
        for (int d = 0; d < DP / 32; ++d)
#pragma unroll
            for (int g = 0; g < 4; ++g)
                store_scaled(out, 32 * d + 8 * g + 4 * (lane >> 5), a.D, acc[d], g, valid, a.scale);
    }
    if (BIAS) {
        // by bucket: the window's sums of the four wavefronts and the far tiles' in the window's ends
#pragma unroll
        for (int d = 32; d > 0; d >>= 1) {
            far_before += __shfl_xor(far_before, d);
            far_after += __shfl_xor(far_after, d);
        }
        if (lane == 0) {
            diag[wave * window] += far_before;
            diag[wave * window + window - 1] += far_after;
        }
        __syncthreads();
        const int reach = bias_reach(a.rule);
        int* bucket = reinterpret_cast<int*>(square);
        for (int s = threadIdx.x; s < window; s += kAttnThreads) {
            win[s] = (diag[s] + diag[window + s]) + (diag[2 * window + s] + diag[3 * window + s]);
            bucket[s] = bucket_of(a.rule, s - reach);
        }
        __syncthreads();
        // 8 neighbouring lanes share a bucket's sum (buckets <= 256: eight rounds of 32 at most)
        for (int c = threadIdx.x >> 3; c < a.rule.buckets; c += kAttnThreads / 8) {
            float sum = 0.0f;
            for (int s = threadIdx.x & 7; s < window; s += 8) sum += bucket[s] == c ? win[s] : 0.0f;
            sum = group_sum<8>(sum);
            if ((threadIdx.x & 7) == 0)
                part_table[(((long)w.b * tiles * splits + w.tile) * a.H + w.h) * a.rule.buckets + c] = sum;
        }
    }
}

// gtable[c][h] = the partial rows of head h added up in order.
__global__ __launch_bounds__(kAttnThreads) void attn_table_kernel(const float* part, int parts, int H, int buckets, float* gtable) {
    __shared__ float join[kAttnThreads];
    const int at = blockIdx.x * 16 + (threadIdx.x & 15), n = H * buckets, group = threadIdx.x >> 4;
    float s = 0.0f;
    if (at < n)
        for (int p = group; p < parts; p += 16) s += part[(long)p * n + at];
    join[threadIdx.x] = s;
    __syncthreads();
    if (group == 0 && at < n) {
        for (int g = 1; g < 16; ++g) s += join[g * 16 + threadIdx.x];
        gtable[(at % buckets) * H + at / buckets] = s;
    }
}

// ---------------------------------------------------------------- backward: keys

// gk and gv of a block of 128 keys.  Both sums stay in registers (128 of them at 128 columns) beside the columns of k and v
// (another 128), hence one wavefront a SIMD there.  2x8 heads of 2047, 128 columns, causal: 221 us, the matrix cores 0.23 busy,
// with 10 vector instructions a matrix instruction, a third of them moves between the two register files; 8x8 heads of 512, 64
// columns, dropout, padded: 49 us, with 16 registers through scratch memory (11 without dropout).
template <int DP, bool BIAS, bool DROP>
__global__ __launch_bounds__(kAttnThreads, DP == 128 ? 1 : 2) void attn_bwd_kv_kernel(Attn a, Scales scales, const float* lse, const float* delta, const float* go, float* gk,
    float* gv, float* part, int tiles, int splits) {
    extern __shared__ __align__(16) unsigned short lds[];
    unsigned short *qt = lds, *gt = qt + Tile<DP>::kRowBytes / 2, *qc = gt + Tile<DP>::kRowBytes / 2, *gc = qc + Tile<DP>::kColBytes / 2;
    float* stats = reinterpret_cast<float*>(gc + Tile<DP>::kColBytes / 2);
    float *qrows = stats + 2 * kAttnRows, *grows = qrows + kAttnRows;         // reciprocal scales of the tile's rows of q, of go
    unsigned* bits = reinterpret_cast<unsigned*>(grows + kAttnRows);          // [wavefront][half][query]: 16 keep bits each
    float* win = grows + kAttnRows + (DROP ? kAttnThreads : 0);
    const Where w = where(a, tiles * splits, kHeavyFirst);
    const int split = w.tile % splits, k0 = w.tile / splits * kAttnCols, lane = threadIdx.x & 63, kw = k0 + (threadIdx.x >> 6) * 32, key = kw + (lane & 31);
    const int q_end = length_of(a.q_lengths, w.b, a.Tq), k_end = length_of(a.k_lengths, w.b, a.Tk), q_offset = offset_of(a, w.b);
    const float* qbase = a.q + w.b * a.q_b + w.h * a.q_h;
    const float* gbase = go + w.b * a.q_b + w.h * a.q_h;
    const long krow = w.b * a.k_b + w.h * a.k_h + key * a.k_t;
    if (BIAS) copy_bias(a, scales.window, w.h, win);
    // queries this workgroup walks: from the first that sees its first key
    int first = 0, last = q_end;
    if (a.causal) first = max(0, k0 - q_offset) / kAttnRows * kAttnRows;
    if (k0 >= k_end) last = 0;
    const int run = (max(0, last - first) + kAttnRows * splits - 1) / (kAttnRows * splits) * kAttnRows;
    first += split * run;
    last = min(last, first + run);
    const bool valid = key < k_end;
    Column<DP> kcol, vcol;
    kcol.load(a.k + krow, valid, a.D);
    const float kscale = power_scale(kcol.top());
    kcol.split(kscale, 1.0f);
    vcol.load(a.v + krow, valid, a.D);
    const float vscale = power_scale(vcol.top());
    vcol.split(vscale, -1.0f);
    const float unscale = a.scale * kLog2e * reciprocal_power(kscale), dscale = reciprocal_power(vscale) * (DROP ? a.rate.scale : 1.0f);
    const long stat0 = ((long)w.b * a.H + w.h) * a.Tq;
    RngState rng = {};
    if (DROP) rng = load_rng(a.rng, a.channel);
    const int bit = 8 * ((lane & 31) >> 4) + 4 * ((lane & 31) >> 3 & 1) + (lane & 3);      // of the lane's key in `kept`, by query
    const unsigned* kept = bits + (threadIdx.x >> 6) * kWave + 32 * (lane >> 2 & 1);
    v16f acck[DP / 32] = {}, accv[DP / 32] = {};
    const typename Tile<DP>::Offsets off(a.q_t, a.D);
    const ScaleArray qscales = scales.of(2, w.b * a.H + w.h, a.Tq), gscales = scales.of(3, w.b * a.H + w.h, a.Tq);
    Tile<DP> qr, gr;
    float qnext = 1.0f, gnext = 1.0f;
    if (first < last) {
        qr.load(off, qbase, a.q_t, first, last, a.D);
        gr.load(off, gbase, a.q_t, first, last, a.D);
        qnext = tile_scale(qscales.tiles, first / kAttnRows);
        gnext = tile_scale(gscales.tiles, first / kAttnRows);
    }
    for (int i0 = first; i0 < last; i0 += kAttnRows) {
        const float qscale = qnext, gscale = gnext;
        __syncthreads();
        qr.template store<true, true>(qt, qc, qscale, qscales, qrows, i0, last);
        gr.template store<true, true>(gt, gc, gscale, gscales, grows, i0, last);
        if (threadIdx.x < kAttnRows) {
            const int i = i0 + threadIdx.x;
            stats[threadIdx.x] = row_reference(i < last ? lse[stat0 + i] : INFINITY);
            stats[kAttnRows + threadIdx.x] = i < last ? delta[stat0 + i] : 0.0f;
        }
        __syncthreads();
        if (i0 + kAttnRows < last) {
            qr.load(off, qbase, a.q_t, i0 + kAttnRows, last, a.D);
            gr.load(off, gbase, a.q_t, i0 + kAttnRows, last, a.D);
            qnext = tile_scale(qscales.tiles, i0 / kAttnRows + 1);
            gnext = tile_scale(gscales.tiles, i0 / kAttnRows + 1);
        }
        const int rel0 = kw - i0 - q_offset;
        if (DROP) {
            // The generator's groups run along the keys of a query.  Lane l forms the numbers of query l % 32 and
            // its half's 16 keys of this tile, bit 8 b + e for number e of 16-key block b, and leaves the bits in LDS,
            // where the lane that owns one of these keys finds all its queries.
            unsigned* mine = bits + (threadIdx.x >> 6) * kWave;
            unsigned mask = 0;
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                unsigned u[4];
                random_group(rng, ((unsigned long long)(stat0 + i0 + (lane & 31)) * ((a.Tk + 15) / 16) + kw / 16 + b) * 2 + (lane >> 5), u);
#pragma unroll
                for (int e = 0; e < 8; ++e) mask |= random16(u, e) >= a.rate.threshold ? 1u << (8 * b + e) : 0u;
            }
            wave_lds_fence();
            mine[lane] = mask;
            wave_lds_fence();
        }
        const bool edge = kw + 32 > k_end || (a.causal && kw + 31 > i0 + q_offset);
        const auto tile_shifts = [&] {
            return shifts<BIAS>(a.rule, win, rel0, -1, edge, [&](int r) { return hidden(a, key, i0 + tile_row(r), k_end, q_offset); });
        };
        v16f shift;
        if constexpr (shifts_early(DP, DROP)) shift = tile_shifts();
        v16f s = product_rows<DP, false>(qt, kcol);
        v16f dp = product_rows<DP, true>(gt, vcol);
        const TileRows query_rows(qscale, qrows), go_rows(gscale, grows);
        query_rows.undo(s);
        go_rows.undo(dp);
        const float score_scale = unscale * query_rows.one, dp_scale = dscale * go_rows.one;
        if constexpr (!shifts_early(DP, DROP)) shift = tile_shifts();
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const int row = tile_row(r);
            const float p = pow2(__builtin_fmaf(s[r], score_scale, shift[r]) - stats[row]);      // rows beyond the queries: 0 by their lse
            const bool keep = !DROP || (kept[row] >> bit & 1u);
            s[r] = keep ? p : 0.0f;
            dp[r] = p * __builtin_fmaf(keep ? dp[r] : 0.0f, dp_scale, -stats[kAttnRows + row]);
        }
        add_tile<DP>(accv, gc, go_rows, s);
        add_tile<DP>(acck, qc, query_rows, dp);
    }
    if (key >= a.Tk) return;
    // partial sums: [split][array][head][key][D]
    const long heads = (long)a.B * a.H, at = (2L * split * heads + w.b * a.H + w.h) * a.Tk + key;
    float *out_k = splits > 1 ? part + at * a.D : gk + krow, *out_v = splits > 1 ? part + (at + heads * a.Tk) * a.D : gv + krow;
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int c = 32 * d + 8 * g + 4 * (lane >> 5);
            store_scaled(out_k, c, a.D, acck[d], g, valid, a.scale);
            store_scaled(out_v, c, a.D, accv[d], g, valid, DROP ? a.rate.scale : 1.0f);
        }
}

// Adds up the partial gradients of a split axis, in order: part is [split][arrays][head][row][D]; a group of
// DP / 4 lanes takes a row.
template <int DP>
__global__ __launch_bounds__(kAttnThreads) void attn_sum_kernel(Attn a, const float* part, float* out0, float* out1, int T, int splits, long s_b, long s_h, long s_t) {
    constexpr int LANES = DP / 4;
    const long rows = (long)a.B * a.H * T, row = (long)blockIdx.x * (kAttnThreads / LANES) + threadIdx.x / LANES, step = rows * a.D * gridDim.y;
    const int c = threadIdx.x % LANES * 4;
    if (row >= rows) return;
    const float* p = part + (blockIdx.y * rows + row) * a.D;
    float4 s = load4(p, c, a.D);
    for (int k = 1; k < splits; ++k) {
        const float4 v = load4(p + k * step, c, a.D);
        s = make_float4(s.x + v.x, s.y + v.y, s.z + v.z, s.w + v.w);
    }
    const int head = (int)(row / T), t = (int)(row - (long)head * T);
    store4((blockIdx.y ? out1 : out0) + head / a.H * s_b + head % a.H * s_h + t * s_t, c, a.D, s.x, s.y, s.z, s.w);
}

// ---------------------------------------------------------------- launchers

// Calls f(head width rounded up), and f(that, bias, dropout), with types for arguments.
template <class F>
static int attn_width(const Attn& a, F f) {
    if (a.D <= 32) return f(std::integral_constant<int, 32>());
    if (a.D <= 64) return f(std::integral_constant<int, 64>());
    return f(std::integral_constant<int, 128>());
}
template <class F>
static int attn_dispatch(const Attn& a, F f) {
    return attn_width(a, [&](auto width) {
        const bool bias = a.table != nullptr, drop = a.rate.threshold != 0;
        if (bias) return drop ? f(width, std::true_type(), std::true_type()) : f(width, std::true_type(), std::false_type());
        return drop ? f(width, std::false_type(), std::true_type()) : f(width, std::false_type(), std::false_type());
    });
}
template <class... P, class... A>
static int attn_launch(const char* name, void (*kernel)(P...), long grid, int grid_y, int threads, size_t lds_bytes, hipStream_t st, A... args) {
    if (lds_bytes > 65536)
        CGT_HIP_TRY(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds_bytes));
    kernel<<<dim3((unsigned)grid, (unsigned)grid_y), threads, lds_bytes, st>>>(args...);
    CGT_LAUNCH_CHECK(name);
    return CGT_AMD_OK;
}

static size_t scale_floats(long heads, long T) { return (size_t)heads * (cdiv(T, kAttnRows) + T); }
// Fills `scales` (of n arrays of Tk or Tq rows), the weights (if there is lse) and the bias window behind them, all at `ws`.
static int launch_scales(const Attn& a, const ScaledArrays& arrays, int n_arrays, int runs, float* ws, Scales* scales, hipStream_t st) {
    const long heads = (long)a.B * a.H;
    long at = 0;
    for (int n = 0; n < n_arrays; ++n) {
        scales->start[n] = at;
        at += (long)scale_floats(heads, arrays.keys[n] ? a.Tk : a.Tq);
    }
    scales->arrays = ws, scales->weights = ws + at, scales->window = ws + at + (arrays.lse ? heads * a.Tq : 0), scales->heads = (int)heads;
    return attn_width(a, [&](auto width) {
        constexpr int W = decltype(width)::value;
        return attn_launch("attention scales", arrays.lse ? attn_scale_kernel<W, true> : attn_scale_kernel<W, false>, heads * runs,
                           n_arrays + (a.table ? 1 : 0), kAttnThreads, 0, st, a, arrays, *scales, n_arrays, runs);
    });
}
// Runs of rows whose scales are found by workgroups of their own: 256 rows or more, 64 at most.  (16 at most:
// 64 queries of 2 heads against 16384 keys 48 us, with 64 37.  Runs of 64 rows: 128 heads of 1024 rows 158 us forward
// and 539 backward, with 256 154 and 520; 4 heads of 512 21 us, with 256 23.)
static int scale_runs(long Tq, long Tk) { return (int)std::max(1L, std::min(cdiv(std::max(Tq, Tk), 256), 64L)); }
// Into how many runs the walked axis (`rows` long) is cut, so that `whole` workgroups become enough to fill
// every CU `resident` times (twice as often where a causal mask makes them uneven); runs of `shortest` rows at least.
// Up to a quarter of that where the workgroups are fewer than the CUs, until they are as many.  Both sides (64 columns):
// cut / whole, forward 8 heads of 4096 146 / 187 us, of 1024 35 / 57, 4 heads of 512 22 / 33, 64 heads of 512 stay whole: 39,
// 45 in three; backward (before its last step for speed) 64 heads of 512 123 / 133, 8 of 4096 479 / 708, 8 of 1024 96 / 203
// (causal 96 / 202, and 118 in twice as many), 4 of 512 62 / 123; 16 heads of 2047 under a causal mask, 128 columns, 491 / 720.
static int axis_splits(long whole, long rows, int resident, int causal, long shortest) {
    if (whole <= 0) return 1;
    const long want = (long)kNumCU * resident * (causal ? 2 : 1);
    return (int)std::max({1L, std::min({cdiv(want, whole), rows / shortest, 16L}), std::min({kNumCU / whole, rows / (shortest / 4), 64L})});
}
static int padded_dim(int D) { return D <= 32 ? 32 : D <= 64 ? 64 : 128; }

// The rule of the buckets: per side (all of them, or half when positions after the query have their
// own) the first half one distance each, then logarithmic up to max_distance.  Bucket e of the
// logarithmic part begins at the smallest n with (n / first)^(side - first) >= (max / first)^e; the
// logarithms are compared in double with a slack far below the gap between whole distances, so that
// the exact ties of the rule (first 8, max 128: at 16, 32, 64) fall where the real numbers say.
static int bucket_rule(const char* what, int buckets, int bidirectional, int max_distance, BucketRule* r) {
    CGT_ARG_CHECK(buckets >= (bidirectional ? 4 : 2) && buckets <= kMaxBuckets && (!bidirectional || buckets % 2 == 0),
                  "%s: %d buckets (%s, and %d at most)", what, buckets,
                  bidirectional ? "an even number, 4 at least, where positions after the query have their own" : "2 at least", kMaxBuckets);
    r->buckets = buckets;
    r->bidirectional = bidirectional != 0;
    r->max_distance = max_distance;
    r->side = bidirectional ? buckets / 2 : buckets;
    r->first = r->side / 2;
    CGT_ARG_CHECK(max_distance > r->first && max_distance <= kMaxDistance, "%s: max_distance %d must be above %d and at most %d", what, max_distance,
                  r->first, kMaxDistance);
    const int logs = r->side - r->first;
    int n = r->first;
    for (int e = 1; e < logs; ++e) {
        const double want = e * std::log((double)max_distance / r->first);
        while (n < max_distance && logs * std::log((double)n / r->first) < want - 1e-11) ++n;
        r->edge[e] = n;
    }
    return CGT_AMD_OK;
}

static int attn_setup(const char* what, Attn* a, long B, long H, long Tq, long Tk, long D, int layout, const float* table, long buckets,
                      int bidirectional, long max_distance, double scale, int causal, long q_offset, double p, const long long* rng, unsigned channel) {
    CGT_ARG_CHECK(B >= 0 && H >= 0 && Tq >= 0 && Tk >= 0, "%s: negative extent", what);
    CGT_ARG_CHECK(D >= 1 && D <= 128, "%s: heads of %ld columns (1 to 128)", what, D);
    CGT_ARG_CHECK(Tq < (1L << 29) && Tk < (1L << 29) && q_offset >= -kMaxOffset && q_offset <= kMaxOffset, "%s: lengths and offset must be below 2^29", what);
    CGT_ARG_CHECK(B < (1L << 22) && H < (1L << 22) && B * H < (1L << 22), "%s: too many heads", what);
    CGT_ARG_CHECK(layout == 0 || layout == 1, "%s: layout %d (0: heads before positions, 1: after them)", what, layout);
    CGT_ARG_CHECK(std::isfinite(scale), "%s: scale must be finite", what);
    if (!dropout_rate(p, what, &a->rate)) return CGT_AMD_ERR_ARG;
    CGT_ARG_CHECK(rng || a->rate.threshold == 0, "%s: dropout needs the generator's state", what);
    a->table = table;
    if (table) {
        if (int rc = bucket_rule(what, (int)std::min(buckets, 1L << 20), bidirectional, (int)std::min(max_distance, 1L << 20), &a->rule)) return rc;
    }
    a->B = (int)B, a->H = (int)H, a->Tq = (int)Tq, a->Tk = (int)Tk, a->D = (int)D;
    a->causal = causal != 0, a->q_offset = (int)q_offset, a->scale = (float)scale, a->rng = rng, a->channel = channel;
    a->q_b = H * Tq * D, a->k_b = H * Tk * D;
    a->q_h = layout ? D : Tq * D, a->k_h = layout ? D : Tk * D;
    a->q_t = a->k_t = layout ? H * D : D;
    return CGT_AMD_OK;
}

static int attention_fwd(const float* q, const float* k, const float* v, const float* table, long B, long H, long Tq, long Tk, long D, int layout,
                         long buckets, int bidirectional, long max_distance, double scale, int causal, long q_offset, const int* q_offsets,
                         const int* q_lengths, const int* k_lengths, double p, const long long* rng, unsigned channel, float* o, float* lse,
                         void* stream) {
    const StreamTurn turn(stream);
    Attn a = {};
    if (int rc = attn_setup("attention", &a, B, H, Tq, Tk, D, layout, table, buckets, bidirectional, max_distance, scale, causal, q_offset, p, rng, channel))
        return rc;
    if (B * H * Tq == 0) return CGT_AMD_OK;
    CGT_ARG_CHECK(q && o && lse && (Tk == 0 || (k && v)), "attention: null pointer");
    a.q = q, a.k = k, a.v = v, a.q_lengths = q_lengths, a.k_lengths = k_lengths, a.q_offsets = q_offsets;
    hipStream_t st = as_stream(stream);
    // Up to eight queries read k and v once, on the vector units; more go through the matrix cores, whose
    // scales take a walk over k and v of their own.  Both sides, vector / matrix: 16 heads of 16 sequences (64 columns)
    // against 8192 keys, 1 query 188 / 370 us, 4 203 / 372, 8 268 / 373; against 512 keys 20 / 41, 24 / 41, 34 / 41;
    // 128 columns, 8 queries 483 / 739; one sequence, 8192 keys, 1 query 19 / 48.
    const bool token = Tq <= 8 && a.rate.threshold == 0;
    const int DP = padded_dim(a.D), tiles = token ? 1 : (int)cdiv(Tq, kAttnCols);
    const long heads = B * H, whole = heads * tiles;
    // Too few workgroups to fill the chip: the keys are cut too.
    const int splits = token ? (whole >= 4 * kNumCU ? 1 : (int)std::max(1L, std::min({cdiv(8L * kNumCU, whole), Tk / 128, 64L})))
                             : axis_splits(whole, Tk, DP == 128 ? 2 : 3, a.causal, 512);
    CGT_ARG_CHECK(whole * splits < (1L << 31) && heads * scale_runs(Tq, Tk) < (1L << 31), "attention: too many workgroups");
    // workspace: the scales of k's and v's rows and the bias window, then the pieces of a split key axis
    const size_t rows = splits > 1 ? (size_t)heads * Tq * splits : 0, window_floats = table && !token ? (size_t)bias_window(a.rule) * H : 0;
    const size_t shared_floats = token ? 0 : (2 * scale_floats(heads, Tk) + window_floats + 1) & ~(size_t)1;
    float* part = nullptr;
    float2* ml = nullptr;
    Scales scales = {};
    if (rows + shared_floats) {
        float* ws = stream_workspace(stream, kWsAttention, (shared_floats + rows * (D + 2)) * sizeof(float), "attention");
        if (!ws) return CGT_AMD_ERR_NOMEM;
        ml = reinterpret_cast<float2*>(ws + shared_floats);
        part = ws + shared_floats + 2 * rows;
        if (!token) {
            if (int rc = launch_scales(a, {{k, v}, {1, 1}, nullptr}, 2, scale_runs(Tk, Tk), ws, &scales, st)) return rc;
        }
    }
    const size_t window_bytes = table ? bias_window(a.rule) * sizeof(float) : 0;
    const int rc = attn_dispatch(a, [&](auto width, auto bias, auto drop) {
        constexpr int W = decltype(width)::value;
        constexpr bool bias_ = decltype(bias)::value, drop_ = decltype(drop)::value;
        if constexpr (!drop_) {
            if (token)
                return a.Tq == 1 ? attn_launch("attention (one query)", attn_token_kernel<W, 1, bias_>, whole * splits, 1, kAttnThreads, window_bytes, st,
                                               a, o, lse, part, ml, splits)
                     : a.Tq <= 4 ? attn_launch("attention (few queries)", attn_token_kernel<W, 4, bias_>, whole * splits, 1, kAttnThreads, window_bytes, st,
                                               a, o, lse, part, ml, splits)
                                 : attn_launch("attention (few queries)", attn_token_kernel<W, 8, bias_>, whole * splits, 1, kAttnThreads, window_bytes, st,
                                               a, o, lse, part, ml, splits);
        }
        const size_t lds_bytes = Tile<W>::kRowBytes + Tile<W>::kColBytes + 2 * kAttnRows * sizeof(float) + window_bytes;
        return attn_launch("attention forward", attn_fwd_kernel<W, bias_, drop_>, whole * splits, 1, kAttnThreads, lds_bytes, st, a, scales, o, lse, part, ml,
                           tiles, splits);
    });
    if (rc != CGT_AMD_OK) return rc;
    if (splits > 1) {
        const int rc = attn_width(a, [&](auto width) {
            constexpr int W = decltype(width)::value;
            constexpr int teams = kAttnThreads / (W / 4);
            return splits >= kJoinTeams ? attn_launch("attention join", attn_join_kernel<W, teams>, heads * Tq, 1, kAttnThreads, 0, st, a, o, lse, part, ml, splits)
                                        : attn_launch("attention join", attn_join_kernel<W, 1>, cdiv(heads * Tq, teams), 1, kAttnThreads, 0, st, a, o, lse, part, ml, splits);
        });
        if (rc != CGT_AMD_OK) return rc;
    }
    return CGT_AMD_OK;
}

static int attention_bwd(const float* q, const float* k, const float* v, const float* table, const float* o, const float* lse, const float* go, long B,
                         long H, long Tq, long Tk, long D, int layout, long buckets, int bidirectional, long max_distance, double scale, int causal,
                         long q_offset, const int* q_offsets, const int* q_lengths, const int* k_lengths, double p, const long long* rng,
                         unsigned channel, float* gq, float* gk, float* gv, float* gtable, void* stream) {
    const StreamTurn turn(stream);
    Attn a = {};
    if (int rc = attn_setup("attention backward", &a, B, H, Tq, Tk, D, layout, table, buckets, bidirectional, max_distance, scale, causal, q_offset, p, rng,
                            channel))
        return rc;
    CGT_ARG_CHECK(!table || gtable, "attention backward: null pointer");
    const long heads = B * H;
    if (heads == 0 || (Tq == 0 && Tk == 0) || Tq == 0) {
        if (table)
            if (int rc = cgt_amd_fill_u32(gtable, 0u, buckets * H, stream)) return rc;
        if (heads * Tk == 0) return CGT_AMD_OK;
        CGT_ARG_CHECK(gk && gv, "attention backward: null pointer");
        if (int rc = cgt_amd_fill_u32(gk, 0u, heads * Tk * D, stream)) return rc;
        return cgt_amd_fill_u32(gv, 0u, heads * Tk * D, stream);
    }
    CGT_ARG_CHECK(q && o && lse && go && gq && (Tk == 0 || (k && v && gk && gv)), "attention backward: null pointer");
    a.q = q, a.k = k, a.v = v, a.q_lengths = q_lengths, a.k_lengths = k_lengths, a.q_offsets = q_offsets;
    hipStream_t st = as_stream(stream);
    const int DP = padded_dim(a.D), qtiles = (int)cdiv(Tq, kAttnCols), ktiles = (int)cdiv(Tk, kAttnCols);
    const int runs = scale_runs(Tq, Tk);
    CGT_ARG_CHECK(heads * qtiles < (1L << 31) && heads * ktiles < (1L << 31) && heads * runs < (1L << 31), "attention backward: too many workgroups");
    const int qsplits = axis_splits(heads * qtiles, Tk, DP == 128 ? 1 : 2, a.causal, 256), ksplits = axis_splits(heads * ktiles, Tq, DP == 128 ? 1 : 2, a.causal, 256);
    // workspace: the rows' scales, the bias window, row products, the table's partial rows, partial gradients (of the queries,
    // then of the keys)
    const long parts = B * qtiles * qsplits;
    const size_t window_floats = table ? (size_t)bias_window(a.rule) * H : 0, range_floats = 2 * (scale_floats(heads, Tk) + scale_floats(heads, Tq)) + heads * Tq + window_floats;
    const size_t table_floats = table ? (size_t)(parts * H * buckets) : 0;
    const size_t part_floats = std::max(qsplits > 1 ? (size_t)qsplits * heads * Tq * D : 0, ksplits > 1 ? (size_t)ksplits * 2 * heads * Tk * D : 0);
    float* ws = stream_workspace(stream, kWsAttention, (range_floats + heads * Tq + table_floats + part_floats) * sizeof(float), "attention backward");
    if (!ws) return CGT_AMD_ERR_NOMEM;
    float *delta = ws + range_floats, *part_table = delta + heads * Tq, *part = part_table + table_floats;
    Scales scales = {};
    int rc = launch_scales(a, {{k, v, q, go}, {1, 1, 0, 0}, lse}, 4, runs, ws, &scales, st);
    if (rc != CGT_AMD_OK) return rc;
    const size_t window_bytes = table ? bias_window(a.rule) * sizeof(float) : 0;
    rc = attn_dispatch(a, [&](auto width, auto bias, auto drop) {
        constexpr int W = decltype(width)::value;
        constexpr bool bias_ = decltype(bias)::value, drop_ = decltype(drop)::value;
        const size_t lds_bytes = 2 * Tile<W>::kRowBytes + Tile<W>::kColBytes + 2 * kAttnRows * sizeof(float) + (bias_ ? 4 * kSquare * sizeof(float) : 0) + 5 * window_bytes;
        return attn_launch("attention backward (queries)", attn_bwd_q_kernel<W, bias_, drop_>, heads * qtiles * qsplits, 1, kAttnThreads, lds_bytes, st, a, scales,
                           o, lse, go, gq, part, delta, part_table, qtiles, qsplits);
    });
    if (rc != CGT_AMD_OK) return rc;
    auto add_up = [&](float* out0, float* out1, long T, int splits, long s_b, long s_h, long s_t) {
        return attn_width(a, [&](auto width) {
            constexpr int W = decltype(width)::value;
            return attn_launch("attention backward (partial sums)", attn_sum_kernel<W>, cdiv(heads * T, kAttnThreads / (W / 4)), out1 ? 2 : 1, kAttnThreads, 0, st,
                               a, part, out0, out1, (int)T, splits, s_b, s_h, s_t);
        });
    };
    if (qsplits > 1) {
        rc = add_up(gq, nullptr, Tq, qsplits, a.q_b, a.q_h, a.q_t);
        if (rc != CGT_AMD_OK) return rc;
    }
    if (table) {
        attn_table_kernel<<<dim3((unsigned)cdiv(H * buckets, 16)), kAttnThreads, 0, st>>>(part_table, (int)parts, a.H, a.rule.buckets, gtable);
        CGT_LAUNCH_CHECK("attention backward (table)");
    }
    if (ktiles) {
        rc = attn_dispatch(a, [&](auto width, auto bias, auto drop) {
            constexpr int W = decltype(width)::value;
            constexpr bool bias_ = decltype(bias)::value, drop_ = decltype(drop)::value;
            const size_t lds_bytes = 2 * Tile<W>::kRowBytes + 2 * Tile<W>::kColBytes + (4 * kAttnRows + (drop_ ? kAttnThreads : 0)) * sizeof(float) + window_bytes;
            return attn_launch("attention backward (keys)", attn_bwd_kv_kernel<W, bias_, drop_>, heads * ktiles * ksplits, 1, kAttnThreads, lds_bytes, st, a, scales,
                               lse, delta, go, gk, gv, part, ktiles, ksplits);
        });
        if (rc != CGT_AMD_OK) return rc;
        if (ksplits > 1) {
            rc = add_up(gk, gv, Tk, ksplits, a.k_b, a.k_h, a.k_t);
            if (rc != CGT_AMD_OK) return rc;
        }
    }
    return CGT_AMD_OK;
}

}  // namespace cgt_amd

using namespace cgt_amd;

CGT_API int cgt_amd_rel_bucket(long rel, int buckets, int bidirectional, int max_distance) {
    BucketRule r;
    if (bucket_rule("rel_bucket", buckets, bidirectional, max_distance, &r)) return -1;
    const long lim = 2L * kMaxDistance;
    return bucket_of(r, (int)std::max(-lim, std::min(lim, rel)));
}

CGT_API int cgt_amd_rel_attention_fwd_f32(const float* q, const float* k, const float* v, const float* table, long B, long H, long Tq, long Tk, long D,
                                          int layout, long buckets, int bidirectional, long max_distance, double scale, int causal, long q_offset,
                                          const int* q_lengths, const int* k_lengths, double p, const long long* rng, unsigned channel,
                                          float* o, float* lse, void* stream) {
    return attention_fwd(q, k, v, table, B, H, Tq, Tk, D, layout, buckets, bidirectional, max_distance, scale, causal, q_offset, nullptr, q_lengths, k_lengths,
                         p, rng, channel, o, lse, stream);
}

CGT_API int cgt_amd_rel_attention_at_fwd_f32(const float* q, const float* k, const float* v, const float* table, long B, long H, long Tq, long Tk, long D,
                                             int layout, long buckets, int bidirectional, long max_distance, double scale, int causal,
                                             const int* q_offsets, const int* q_lengths, const int* k_lengths, double p, const long long* rng,
                                             unsigned channel, float* o, float* lse, void* stream) {
    CGT_ARG_CHECK(q_offsets || B == 0, "attention: null pointer (offsets)");
    return attention_fwd(q, k, v, table, B, H, Tq, Tk, D, layout, buckets, bidirectional, max_distance, scale, causal, 0, q_offsets, q_lengths, k_lengths,
                         p, rng, channel, o, lse, stream);
}

CGT_API int cgt_amd_rel_attention_bwd_f32(const float* q, const float* k, const float* v, const float* table, const float* o, const float* lse,
                                          const float* go, long B, long H, long Tq, long Tk, long D, int layout, long buckets, int bidirectional,
                                          long max_distance, double scale, int causal, long q_offset, const int* q_lengths, const int* k_lengths,
                                          double p, const long long* rng, unsigned channel, float* gq, float* gk, float* gv, float* gtable, void* stream) {
    return attention_bwd(q, k, v, table, o, lse, go, B, H, Tq, Tk, D, layout, buckets, bidirectional, max_distance, scale, causal, q_offset, nullptr, q_lengths,
                         k_lengths, p, rng, channel, gq, gk, gv, gtable, stream);
}

CGT_API int cgt_amd_rel_attention_at_bwd_f32(const float* q, const float* k, const float* v, const float* table, const float* o, const float* lse,
                                             const float* go, long B, long H, long Tq, long Tk, long D, int layout, long buckets, int bidirectional,
                                             long max_distance, double scale, int causal, const int* q_offsets, const int* q_lengths,
                                             const int* k_lengths, double p, const long long* rng, unsigned channel, float* gq, float* gk, float* gv,
                                             float* gtable, void* stream) {
    CGT_ARG_CHECK(q_offsets || B == 0, "attention backward: null pointer (offsets)");
    return attention_bwd(q, k, v, table, o, lse, go, B, H, Tq, Tk, D, layout, buckets, bidirectional, max_distance, scale, causal, 0, q_offsets, q_lengths,
                         k_lengths, p, rng, channel, gq, gk, gv, gtable, stream);
}
