// policy_attention_dq.hip - the attention's backward pass over rows: dq, the bias' gradient, and for the pass over keys
// (policy_attention_dkv.hip) each row's statistics, delta and range of keys. The probabilities are computed again.
//
// With P = 2^(s - top) / sum, dP = dout v^T and dS = P (dP - delta): dq = scale dS k, dbias[h, b] = the sum of dS over the pairs
// at a distance of bucket b. Two passes, one that keeps rows and one that keeps keys, compute the scores twice (7 products
// where one pass needs 5) and need no atomics: results do not depend on the order in which blocks run.
#include "policy_attention.hpp"

namespace goi {
namespace {

template <typename T, int DP, int NW>
__global__ void __launch_bounds__(64 * NW) k_attention_dq(const AttnRun A) {
    constexpr int NT = 64 * NW, KT = NW == 1 && DP == 128 ? 32 : 64, KB = KT / 32, NBUF = NW == 1 ? 1 : 2;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    __shared__ int range[2][NW];
    T* const tiles = reinterpret_cast<T*>(lds);  // [NBUF][keys, values][KT][DP]
    float* const table = reinterpret_cast<float*>(lds + NBUF * 2 * KT * DP * sizeof(T));
    const GoiAttention& a = A.a;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, half = lane >> 5;

    int place = xcd_place(blockIdx.x, gridDim.x);
    const int tile = A.tiles - 1 - place % A.tiles;
    place /= A.tiles;
    const int n = place / a.kv_heads, g = place - n * a.kv_heads;
    const int L = history(A, n), m0 = (tile * NW + wave) * 32, m = m0 + (lane & 31);
    const Row row = make_row(A, n, L, m);
    const BlockInfo blk = make_block(row);
    if (lane == 0) {
        range[0][wave] = blk.lo;
        range[1][wave] = blk.hi;
        if (m0 < A.rows) A.block_info[(int64_t)(n * a.kv_heads + g) * A.blocks + m0 / 32] = blk;
    }
    // the bias by distance, the bucket of each distance, and each lane's own sums by bucket
    const float* bias = nullptr;
    uint8_t* const bucket = reinterpret_cast<uint8_t*>(table + A.group * a.n_distances);
    float* const sums = reinterpret_cast<float*>(bucket + (a.n_distances + 15) / 16 * 16) + wave * a.n_buckets * 64 + lane;
    if (a.bias) {
        stage_bias(A, g, table, tid, NT);
        for (int x = tid; x < a.n_distances; x += NT) bucket[x] = (uint8_t)min(max(a.buckets[x], 0), a.n_buckets - 1);
        for (int b = 0; b < a.n_buckets; ++b) sums[b * 64] = 0.0f;
        bias = table + row.hl * a.n_distances;
    }
    const int head = g * A.group + row.hl;
    half8<T> q[DP / 16], go[DP / 16];
    load_operand<T, DP>(q, static_cast<const T*>(a.q) + n * a.q_strides[0] + row.i * a.q_strides[1] + head * a.q_strides[2],
                        row.valid, a.dim, lane);
    load_operand<T, DP>(go, static_cast<const T*>(a.dout) + n * a.dout_strides[0] + row.i * a.dout_strides[1] +
                                head * a.dout_strides[2], row.valid, a.dim, lane);
    float top = INFINITY, inv = 0.0f, delta = 0.0f;  // delta: out . dout / sum
    {
        half8<T> out[DP / 16];
        load_operand<T, DP>(out, static_cast<const T*>(a.out) + n * a.out_strides[0] + row.i * a.out_strides[1] +
                                     head * a.out_strides[2], row.valid, a.dim, lane);
#pragma unroll
        for (int s = 0; s < DP / 16; ++s)
#pragma unroll
            for (int e = 0; e < 8; ++e) delta += (float)out[s][e] * (float)go[s][e];
        delta += other_half(delta);
        if (row.hi > row.lo) {
            const float2 st =
                reinterpret_cast<const float2*>(a.stats)[((int64_t)n * a.heads + head) * a.q_steps + row.i];
            if (st.y != 0.0f) {  // 0: only scores of minus infinity
                top = st.x;
                inv = 1.0f / st.y;
            }
        }
        delta = inv != 0.0f ? delta * inv : 0.0f;
        if (row.valid && half == 0)
            A.row_info[(int64_t)(n * a.kv_heads + g) * A.rows + m] = RowInfo{top, inv, delta, row.lo, row.hi};
    }
    __syncthreads();
    int lo = INT_MAX, hi = 0;
    for (int w = 0; w < NW; ++w) {
        lo = min(lo, range[0][w]);
        hi = max(hi, range[1][w]);
    }

    float16_t dq[DP / 32];
    clear(dq);
    if (lo < hi) {
        const T* const kp = static_cast<const T*>(a.k) + n * a.k_strides[0] + g * a.k_strides[2];
        const T* const vp = static_cast<const T*>(a.v) + n * a.v_strides[0] + g * a.v_strides[2];
        KeyStage<T, DP, KT, NT> ks, vs;
        ks.load(kp, a.k_strides[1], lo, lo, hi, a.dim, tid);
        vs.load(vp, a.v_strides[1], lo, lo, hi, a.dim, tid);
        ks.store(tiles, lo, lo, hi, a.dim, tid);
        vs.store(tiles + KT * DP, lo, lo, hi, a.dim, tid);
        __syncthreads();
        int buf = 0;
        for (int k0 = lo; k0 < hi; k0 += KT) {
            const bool more = k0 + KT < hi;
            if (more) {
                ks.load(kp, a.k_strides[1], k0 + KT, lo, hi, a.dim, tid);
                vs.load(vp, a.v_strides[1], k0 + KT, lo, hi, a.dim, tid);
            }
            const T* const kt = tiles + buf * 2 * KT * DP;
            const T* const vt = kt + KT * DP;
#pragma unroll
            for (int b = 0; b < KB; ++b) {
                const int key0 = k0 + 32 * b;
                if (key0 >= blk.hi || key0 + 32 <= blk.lo) continue;
                float16_t s = raw_scores<T, DP>(kt, 32 * b, q, lane);
                const float16_t dp = raw_scores<T, DP>(vt, 32 * b, go, lane);
                scale_scores(s, A.c, bias, a.n_distances, key0, row.pos, blk.pos_lo, blk.pos_hi, half);
#pragma unroll
                for (int r = 0; r < 16; ++r) s[r] = exp2_fast(s[r] - top) * (dp[r] * inv - delta);
                if (key0 < blk.full_lo || key0 + 32 > blk.full_hi) {
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        const int key = key0 + mfma_row(r, half);
                        s[r] = key >= row.lo && key < row.hi ? s[r] : 0.0f;
                    }
                }
                if (bias) {
                    // the lane's own sums, one word a bucket: no two lanes share one, so the order of additions is the
                    // program's
                    const int one = one_distance(key0, blk.pos_lo, blk.pos_hi, a.n_distances);
                    if (one >= 0) {
                        float t = 0.0f;
#pragma unroll
                        for (int r = 0; r < 16; ++r) t += s[r];
                        __hip_atomic_fetch_add(sums + bucket[one] * 64, t, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
                    } else {
#pragma unroll
                        for (int r = 0; r < 16; ++r) {
                            const int d = min(max(row.pos - key0 - mfma_row(r, half), 0), a.n_distances - 1);
                            __hip_atomic_fetch_add(sums + bucket[d] * 64, s[r], __ATOMIC_RELAXED,
                                                   __HIP_MEMORY_SCOPE_WORKGROUP);
                        }
                    }
                }
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    const half8<T> ds = to_operand<T>(s, x);
#pragma unroll
                    for (int d = 0; d < DP / 32; ++d)
                        dq[d] = mfma(column_fragment<T, DP>(kt, 32 * b + 16 * x, 32 * d, lane), ds, dq[d]);
                }
            }
            if (NBUF == 1) __syncthreads();
            else buf ^= 1;
            if (more) {
                ks.store(tiles + buf * 2 * KT * DP, k0 + KT, lo, hi, a.dim, tid);
                vs.store(tiles + buf * 2 * KT * DP + KT * DP, k0 + KT, lo, hi, a.dim, tid);
            }
            __syncthreads();
        }
    }
    if (row.valid) {
        T* const to = static_cast<T*>(a.dq) + n * a.dq_strides[0] + row.i * a.dq_strides[1] + head * a.dq_strides[2];
        store_row<T, DP>(to, dq, a.scale, a.dim, half);
    }
    if (a.bias) {
        __syncthreads();
        // the block's sums: of the lanes whose row is of head hl, over all waves
        const float* const all = reinterpret_cast<const float*>(bucket + (a.n_distances + 15) / 16 * 16);
        float* const part = A.part_bias + ((int64_t)n * A.tiles + tile) * a.heads * a.n_buckets + g * A.group * a.n_buckets;
        for (int x = tid; x < A.group * a.n_buckets; x += NT) {
            const int hl = x / a.n_buckets, b = x - hl * a.n_buckets;
            float t = 0.0f;
            for (int w = 0; w < NW; ++w) {
                const int first = (hl - (tile * NW + w) * 32 % A.group + A.group) % A.group;
                const float* const own = all + (w * a.n_buckets + b) * 64;
                for (int l = first; l < 32; l += A.group) t += own[l] + own[l + 32];
            }
            part[x] = t;
        }
    }
}

template <typename T, int DP, int NW>
hipError_t launch(const AttnRun& A, hipStream_t st) {
    constexpr int KT = NW == 1 && DP == 128 ? 32 : 64, NBUF = NW == 1 ? 1 : 2;
    size_t lds = NBUF * 2 * KT * DP * sizeof(T);
    if (A.a.bias)
        lds += (size_t)A.group * A.a.n_distances * sizeof(float) + (A.a.n_distances + 15) / 16 * 16 +
               (size_t)NW * A.a.n_buckets * 64 * sizeof(float);
    (void)hipFuncSetAttribute(reinterpret_cast<const void*>(k_attention_dq<T, DP, NW>),
                              hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    hipLaunchKernelGGL((k_attention_dq<T, DP, NW>), dim3((unsigned)((int64_t)A.a.n_worlds * A.a.kv_heads * A.tiles)),
                       dim3(64 * NW), lds, st, A);
    return hipGetLastError();
}

template <typename T, int DP>
hipError_t launch(const AttnRun& A, int waves, hipStream_t st) {
    return waves == 1 ? launch<T, DP, 1>(A, st) : waves == 2 ? launch<T, DP, 2>(A, st) : launch<T, DP, 4>(A, st);
}

template <typename T>
hipError_t launch(const AttnRun& A, int waves, hipStream_t st) {
    const int dp = attention_dim_tile(A.a.dim);
    return dp == 32 ? launch<T, 32>(A, waves, st) : dp == 64 ? launch<T, 64>(A, waves, st) : launch<T, 128>(A, waves, st);
}

}  // namespace

hipError_t launch_attention_dq(const AttnRun& A, int waves, hipStream_t st) {
    return A.a.type == GOI_BF16 ? launch<bf16>(A, waves, st) : launch<f16>(A, waves, st);
}

}  // namespace goi
