// policy_attention.hpp - what the attention kernels share (policy_attention.hip forward, policy_attention_dq.hip and
// policy_attention_dkv.hip backward): the launch block, packed rows, tiles on their way from memory to LDS, scores.
//
// The query heads that share a key head are packed with the steps into one axis of rows, row m = step m / group, head
// m % group of the key head's group, so a tile of rows fills whatever the two numbers are, and each key is read once for
// all of its heads. Scores are computed transposed, keys x rows: a lane of the 32 x 32 product then holds 16 keys of ONE
// row, so that the softmax runs within a lane (and its partner 32 lanes away), and the probabilities, rounded, are the
// second operand of the product with the values as they stand.
#pragma once

#include <climits>
#include <cmath>

#include "policy.hpp"

namespace goi {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kMaxBuckets = 64, kMaxBiasTable = 4096;

// A row's part of what the backward kernels hand over: its largest score in powers of two (+infinity for a row without keys,
// so that exp2(s - top) is 0), the inverse of its sum, delta = out . dout times that, and the keys it sees.
struct RowInfo {
    float top, inv, delta;
    int lo, hi;
};
// The same for 32 rows: the keys that any row sees [lo, hi), those that every row sees [full_lo, full_hi), and the range
// of the rows' positions plus origin.
struct BlockInfo {
    int lo, hi, full_lo, full_hi, pos_lo, pos_hi, pad0, pad1;
};

struct AttnRun {
    GoiAttention a;
    int group;   // query heads per key head
    int rows;    // packed rows of a key head: q_steps * group
    int tiles;   // row tiles (forward, dq) or key tiles (dkv) of a key head
    int splits;  // forward: the key axis is cut into `splits` ranges of `span` keys, joined afterwards
    int span;
    int origin;  // index of distance 0 in buckets
    int blocks;  // 32-row blocks of a key head
    float c;     // scale * log2(e)
    float* part_o;   // forward, splits > 1: [splits][world, key head, row][dim] unnormalised outputs
    float2* part_ml; // and [splits][world, key head, row] maximum (powers of two) and sum
    RowInfo* row_info;      // backward: [world, key head][rows]
    BlockInfo* block_info;  // [world, key head][blocks]
    float* part_bias;       // [world, row tile][heads * n_buckets]
};

// Host side (policy_attention.hip): checks, sizes and launches.
hipError_t launch_attention_dq(const AttnRun& A, int waves, hipStream_t st);
hipError_t launch_attention_dkv(const AttnRun& A, int waves, hipStream_t st);
int attention_dim_tile(int dim);  // 32, 64 or 128

__device__ __forceinline__ int history(const AttnRun& A, int n) {
    return A.a.lengths ? min(max(A.a.lengths[n], 0), A.a.k_steps) : A.a.k_steps;
}

struct Row {
    bool valid;    // m < rows
    int i, hl;     // step and head within the group
    int pos;       // position + origin
    int lo, hi;    // keys seen; lo = hi = 0 if none
};

__device__ __forceinline__ Row make_row(const AttnRun& A, int n, int L, int m) {
    Row r;
    r.valid = m < A.rows;
    r.i = r.valid ? m / A.group : 0;
    r.hl = r.valid ? m - r.i * A.group : 0;
    const int p = L - A.a.q_steps + r.i;
    r.pos = p + A.origin;
    r.lo = A.a.first ? max(A.a.first[(int64_t)n * A.a.q_steps + r.i], 0) : 0;
    r.hi = A.a.causal ? min(p + 1, L) : L;
    if (!r.valid || r.hi <= r.lo) r.lo = r.hi = 0;
    return r;
}

__device__ __forceinline__ BlockInfo make_block(const Row& r) {
    BlockInfo b;
    b.lo = wave_min(r.hi > r.lo ? r.lo : INT_MAX);
    b.hi = wave_max(r.hi);
    b.full_lo = wave_max(r.valid ? r.lo : 0);
    b.full_hi = wave_min(r.valid ? r.hi : INT_MAX);
    b.pos_lo = wave_min(r.valid ? r.pos : INT_MAX);
    b.pos_hi = wave_max(r.valid ? r.pos : INT_MIN);
    b.pad0 = b.pad1 = 0;
    return b;
}

// ROWS rows of `dim` elements on their way to an LDS tile: load() issues the loads (of addresses inside the tensor, whatever
// the row), store() writes the tile with zeros in the rows outside [lo, hi) and past dim.
template <typename T, int DP, int ROWS, int NT>
struct KeyStage {
    static constexpr int N = ROWS * (DP / 8) / NT;
    static_assert(ROWS * (DP / 8) % NT == 0, "whole chunks a thread");
    int4_t x[N];
    __device__ __forceinline__ void load(const T* base, int64_t stride, int row0, int lo, int hi, int dim, int tid) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const int c = tid + j * NT, row = c / (DP / 8), ch = c % (DP / 8);
            const int key = min(max(row0 + row, lo), hi - 1);
            x[j] = *reinterpret_cast<const int4_t*>(base + key * stride + (ch * 8 < dim ? ch * 8 : 0));
        }
    }
    __device__ __forceinline__ void store(T* tile, int row0, int lo, int hi, int dim, int tid) const {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const int c = tid + j * NT, row = c / (DP / 8), ch = c % (DP / 8);
            const bool in = row0 + row >= lo && row0 + row < hi && ch * 8 < dim;
            reinterpret_cast<int4_t*>(tile)[chunk_at<DP>(row, ch)] = in ? x[j] : int4_t{0, 0, 0, 0};
        }
    }
};

// A lane's second operand over one row of memory: elements 16 s + 8 (lane >> 5) .. of it, zeros past dim or without a row
template <typename T, int DP>
__device__ __forceinline__ void load_operand(half8<T> (&f)[DP / 16], const T* row, bool valid, int dim, int lane) {
#pragma unroll
    for (int s = 0; s < DP / 16; ++s) {
        const int d = 16 * s + 8 * (lane >> 5);
        union {
            int4_t i;
            half8<T> h;
        } u;
        u.i = int4_t{0, 0, 0, 0};
        if (valid && d < dim) u.i = *reinterpret_cast<const int4_t*>(row + d);
        f[s] = u.h;
    }
}

// The bias table of key head g's group in LDS, [group][n_distances], in powers of two. Finite entries are held within
// +-1.7e38, so that a type's lowest value, a usual mask, stays finite here and a row of such entries alone is still a row of
// equal scores, as in the formula.
__device__ __forceinline__ void stage_bias(const AttnRun& A, int g, float* table, int tid, int nt) {
    const GoiAttention& a = A.a;
    for (int x = tid; x < A.group * a.n_distances; x += nt) {
        const int hl = x / a.n_distances, dist = x - hl * a.n_distances;
        const int b = min(max(a.buckets[dist], 0), a.n_buckets - 1);
        const int64_t at = (int64_t)(g * A.group + hl) * a.n_buckets + b;
        float v;
        if (a.bias_type == GOI_F32) v = static_cast<const float*>(a.bias)[at];
        else if (a.bias_type == GOI_F16) v = (float)static_cast<const f16*>(a.bias)[at];
        else v = (float)static_cast<const bf16*>(a.bias)[at];
        const float y = v * kLog2e;
        table[x] = fabsf(v) <= 3.4028235e38f ? fminf(fmaxf(y, -1.7e38f), 1.7e38f) : y;
    }
}

// The place in a table of n distances of every pair of a 32-key block at key0 with rows at positions pos_lo .. pos_hi, or -1
// where it is not one place.
__device__ __forceinline__ int one_distance(int key0, int pos_lo, int pos_hi, int n) {
    const int a = min(max(pos_lo - (key0 + 31), 0), n - 1), b = min(max(pos_hi - key0, 0), n - 1);
    return a == b ? a : -1;
}

// Scores of 32 keys (tile rows row0 .. + 31) with the lane's row: the raw products of the 16 keys that the lane holds
template <typename T, int DP>
__device__ __forceinline__ float16_t raw_scores(const T* tile, int row0, const half8<T> (&f)[DP / 16], int lane) {
    float16_t s;
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = 0.0f;
#pragma unroll
    for (int x = 0; x < DP / 16; ++x) s = mfma(row_fragment<T, DP>(tile, row0, x, lane), f[x], s);
    return s;
}

// s * c + bias of the lane's 16 keys from key0 on (keys x rows layout). bias: the row's table, or null
__device__ __forceinline__ void scale_scores(float16_t& s, float c, const float* bias, int n_dist, int key0, int pos,
                                             int pos_lo, int pos_hi, int half) {
    if (!bias) {
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] *= c;
        return;
    }
    const int one = one_distance(key0, pos_lo, pos_hi, n_dist);
    if (one >= 0) {
        const float b = bias[one];
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = s[r] * c + b;
    } else {
#pragma unroll
        for (int r = 0; r < 16; ++r)
            s[r] = s[r] * c + bias[min(max(pos - key0 - mfma_row(r, half), 0), n_dist - 1)];
    }
}

// the lane's half of a row of d0 .. : 4 consecutive elements per register group, as the transposed products hold them
template <typename T, int DP>
__device__ __forceinline__ void store_row(T* row, const float16_t (&o)[DP / 32], float f, int dim, int half) {
#pragma unroll
    for (int b = 0; b < DP / 32; ++b)
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            const int d = 32 * b + 8 * x + 4 * half;
            half4<T> y;
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] = (T)(o[b][4 * x + e] * f);
            if (d < dim) *reinterpret_cast<half4<T>*>(row + d) = y;
        }
}

template <int N>
__device__ __forceinline__ void clear(float16_t (&o)[N]) {
#pragma unroll
    for (int b = 0; b < N; ++b)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[b][r] = 0.0f;
}

}  // namespace goi
