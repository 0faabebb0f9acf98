// policy_attention_dq.hip - the attention's backward pass over rows: dq, the bias' gradient, and for the pass over keys
// (policy_attention_dkv.hip) each row's statistics, delta and range of keys. The probabilities are computed again.
//
// With P = 2^(s - top) / sum, dP = dout v^T and dS = P (dP - delta): dq = scale dS k, dbias[h, b] = the sum of dS over the pairs
// at a distance of bucket b. Two passes, one that keeps rows and one that keeps keys, compute the scores twice (7 products
// where one pass needs 5) and need no atomics: results do not depend on the order in which blocks run.
#include "policy_attention.hpp"

namespace goi {
namespace {

// dq of a wave's 32 rows pair by pair
template <typename T>
__device__ void careful_dq(const AttnRun& A, int n, int g, int L, int m0, const float* table, const Row& mine, float my_top,
                           float my_inv, float my_delta, int lane) {
    for (int r = 0; r < 32 && m0 + r < A.rows; ++r) {
        const int i = step_of(A, m0 + r), hl = m0 + r - i * A.group, head = g * A.group + hl;
        const int lo = __shfl(mine.lo, r), hi = __shfl(mine.hi, r);
        const float top = __shfl(my_top, r), inv = __shfl(my_inv, r), delta = __shfl(my_delta, r);
        const float2 q = two_elements(A.q.at<T>(n, i, head), A.dim, lane);
        const float2 go = two_elements(A.dout.at<T>(n, i, head), A.dim, lane);
        const float* const bias = A.bias ? table + hl * A.table + kPad : nullptr;
        float2 dq = make_float2(0.0f, 0.0f);
        for (int key = lo; key < hi; ++key) {
            const float2 k = two_elements(A.k.at<T>(n, key, g), A.dim, lane), v = two_elements(A.v.at<T>(n, key, g), A.dim, lane);
            const float s = careful_score(A, q, k, bias, L - A.q_steps + i - key);
            const float ds = exp2_fast(s - top) * (wave_sum(go.x * v.x + go.y * v.y) * inv - delta);
            dq.x += ds * k.x;
            dq.y += ds * k.y;
        }
        T* const to = A.dq.at<T>(n, i, head);
        if (lane < A.dim) to[lane] = (T)(dq.x * A.scale);
        if (lane + 64 < A.dim) to[lane + 64] = (T)(dq.y * A.scale);
    }
}

template <typename T, int DP, int NW>
__global__ void __launch_bounds__(64 * NW, DP == 128 && NW == 1 ? 1 : 2) k_attention_dq(const AttnRun A) {
    constexpr int NT = 64 * NW, KT = tile_rows(DP, NW), KB = KT / 32, NBUF = tile_buffers(NW);
    extern __shared__ __attribute__((aligned(16))) char lds[];
    __shared__ int range[2][NW];
    T* const tiles = reinterpret_cast<T*>(lds);  // [NBUF][keys, values][KT][DP]
    float* const table = reinterpret_cast<float*>(lds + NBUF * 2 * KT * DP * sizeof(T));
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), half = lane >> 5;

    const int place = xcd_place(blockIdx.x, gridDim.x), g = place / A.per_head, block = place - g * A.per_head;
    // the bias by distance, each lane's own sums by bucket, and the place of each distance's bucket in them. A bucket's 64 lanes are
    // kSumPitch words apart from the next's: adding up many buckets over the lanes, at the end, is then free of bank conflicts
    float* const all = table + A.group * A.table;  // [NW][n_buckets][kSumPitch]
    float* const sums = all + wave * A.n_buckets * kSumPitch + lane;
    uint16_t* const bucket = reinterpret_cast<uint16_t*>(all + NW * A.n_buckets * kSumPitch);  // [A.table]
    if (A.bias) {
        stage_bias(A, g, table, tid, NT);
        for (int x = tid; x < A.table; x += NT)
            bucket[x] = (uint16_t)(min(max(A.buckets[min(max(x - kPad, 0), A.n_distances - 1)], 0), A.n_buckets - 1) * kSumPitch);
        for (int b = 0; b < A.n_buckets; ++b) sums[b * kSumPitch] = 0.0f;
    }
    // a lane's rows are of the same head in all of a block's items (the host gives a block one item where they are not)
    const int end = (int)((int64_t)(block + 1) * A.items / A.per_head);
    for (int item = (int)((int64_t)block * A.items / A.per_head); item < end; ++item) {
        const int n = item / A.tiles, tile = A.tiles - 1 - (item - n * A.tiles);
        const int L = history(A, n), m0 = (tile * NW + wave) * 32, m = m0 + (lane & 31);
        Row row = make_row(A, n, L, m);
        const BlockInfo blk = make_block(A, L, m0, row);
        row.pos = min(max(row.pos, blk.pos_lo), blk.pos_hi);  // also where there is no row
        if (lane == 0) {
            range[0][wave] = blk.lo;
            range[1][wave] = blk.hi;
            if (m0 < A.rows) A.block_info[(int64_t)(n * A.kv_heads + g) * A.blocks + m0 / 32] = blk;
        }
        const float* const bias = A.bias ? table + row.hl * A.table + kPad : nullptr;
        const int head = g * A.group + row.hl;
        half8<T> q[DP / 16], go[DP / 16];
        load_operand<T, DP>(q, A.q.at<T>(n, row.i, head), row.valid, A.dim, lane);
        load_operand<T, DP>(go, A.dout.at<T>(n, row.i, head), row.valid, A.dim, lane);
        float top = INFINITY, inv = 0.0f, delta = 0.0f;  // delta: out . dout / sum
        {
            half8<T> out[DP / 16];
            load_operand<T, DP>(out, A.out.at<T>(n, row.i, head), row.valid, A.dim, lane);
            float2 st = make_float2(0.0f, 0.0f);
            if (row.hi > row.lo) st = A.stats[((int64_t)n * A.heads + head) * A.q_steps + row.i];
#pragma unroll
            for (int s = 0; s < DP / 16; ++s)
#pragma unroll
                for (int e = 0; e < 8; ++e) delta += (float)out[s][e] * (float)go[s][e];
            delta = half_sum(delta);
            if (st.y != 0.0f) {  // 0: only scores of minus infinity, or no key
                top = st.x;
                inv = 1.0f / st.y;
            }
            delta = inv != 0.0f ? delta * inv : 0.0f;
            if (row.valid && half == 0)
                A.row_info[(int64_t)(n * A.kv_heads + g) * A.rows + m] = RowInfo{top, inv, delta, row.lo, row.hi};
        }
        __syncthreads();
        int lo = INT_MAX, hi = 0;
        for (int w = 0; w < NW; ++w) {
            lo = min(lo, range[0][w]);
            hi = max(hi, range[1][w]);
        }
        lo = __builtin_amdgcn_readfirstlane(lo);
        hi = __builtin_amdgcn_readfirstlane(hi);

        float16_t dq[DP / 32];
        clear(dq);
        bool careful = false;
        if (lo < hi) {
            KeyStage<T, DP, KT, NT> ks(A.k, n, g, A.dim, tid), vs(A.v, n, g, A.dim, tid);
            ks.load(lo, hi, tid);
            vs.load(lo, hi, tid);
            ks.store(tiles, lo, hi, tid);
            vs.store(tiles + KT * DP, lo, hi, tid);
            __syncthreads();
            int buf = 0;
            for (int k0 = lo; k0 < hi; k0 += KT) {
                const bool more = k0 + KT < hi;
                if (more) {
                    ks.load(k0 + KT, hi, tid);
                    vs.load(k0 + KT, hi, tid);
                }
                const T* const kt = tiles + buf * 2 * KT * DP;
                const T* const vt = kt + KT * DP;
#pragma unroll
                for (int b = 0; b < KB; ++b) {
                    const int key0 = k0 + 32 * b;
                    if (key0 >= blk.hi || key0 + 32 <= blk.lo) continue;
                    float16_t s = raw_scores<T, DP>(kt, 32 * b, q, lane);
                    const float16_t dp = raw_scores<T, DP>(vt, 32 * b, go, lane);
                    scale_scores(s, A.c, bias, A.n_distances, key0, row.pos, blk.pos_lo, blk.pos_hi, half);
#pragma unroll
                    for (int r = 0; r < 16; ++r) s[r] = exp2_fast(s[r] - top) * (dp[r] * inv - delta);
                    if (key0 < blk.full_lo || key0 + 32 > blk.full_hi) {
#pragma unroll
                        for (int r = 0; r < 16; ++r) {
                            const int key = key0 + mfma_row(r, half);
                            s[r] = key >= row.lo && key < row.hi ? s[r] : 0.0f;
                        }
                        careful = careful || !finite_rows<T, DP>(kt, 32 * b, lane);
                    }
                    if (bias) {
                        // the lane's own sums, one word a bucket: no two lanes share one, so the order of additions is the
                        // program's
                        const int one = one_distance(key0, blk.pos_lo, blk.pos_hi, A.n_distances);
                        if (one >= 0) {
                            float t = 0.0f;
#pragma unroll
                            for (int r = 0; r < 16; ++r) t += s[r];
                            __hip_atomic_fetch_add(sums + bucket[kPad + one], t, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
                        } else {
                            const uint16_t* const to = bucket + (kPad + row.pos - key0 - 4 * half - 27);
#pragma unroll
                            for (int r = 0; r < 16; ++r)
                                __hip_atomic_fetch_add(sums + to[27 - mfma_row(r, 0)], s[r], __ATOMIC_RELAXED,
                                                       __HIP_MEMORY_SCOPE_WORKGROUP);
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
                    ks.store(tiles + buf * 2 * KT * DP, k0 + KT, hi, tid);
                    vs.store(tiles + buf * 2 * KT * DP + KT * DP, k0 + KT, hi, tid);
                }
                __syncthreads();
            }
        }
        if (row.valid) store_row<T, DP>(A.dq.at<T>(n, row.i, head), dq, A.scale, A.dim, half);
        if (careful) careful_dq<T>(A, n, g, L, m0, table, row, top, inv, delta, lane);
        __syncthreads();  // the next item overwrites what this one read
    }
    if (A.bias) {
        // the block's sums: of the lanes whose row is of head hl, over all waves
        const int tile = A.tiles - 1 - (int)((int64_t)block * A.items / A.per_head) % A.tiles;
        float* const part = A.part_bias + (int64_t)block * A.heads * A.n_buckets + g * A.group * A.n_buckets;
        for (int x = tid; x < A.group * A.n_buckets; x += NT) {
            const int hl = x / A.n_buckets, b = x - hl * A.n_buckets;
            float t = 0.0f;
            for (int w = 0; w < NW; ++w) {
                const int first = (hl - (tile * NW + w) * 32 % A.group + A.group) % A.group;
                const float* const own = all + (w * A.n_buckets + b) * kSumPitch;
                for (int l = first; l < 32; l += A.group) t += own[l] + own[l + 32];
            }
            part[x] = t;
        }
    }
}

template <typename T, int DP, int NW>
hipError_t launch(const AttnRun& A, hipStream_t st) {
    const size_t lds = attention_dq_lds(A, NW);
    (void)hipFuncSetAttribute(reinterpret_cast<const void*>(k_attention_dq<T, DP, NW>),
                              hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    hipLaunchKernelGGL((k_attention_dq<T, DP, NW>), dim3((unsigned)(A.kv_heads * A.per_head)), dim3(64 * NW), lds, st, A);
    return hipGetLastError();
}

template <typename T, int DP>
hipError_t launch(const AttnRun& A, int waves, hipStream_t st) {
    return waves == 1 ? launch<T, DP, 1>(A, st) : waves == 2 ? launch<T, DP, 2>(A, st) : launch<T, DP, 4>(A, st);
}

template <typename T>
hipError_t launch(const AttnRun& A, int waves, hipStream_t st) {
    const int dp = attention_dim_tile(A.dim);
    return dp == 32 ? launch<T, 32>(A, waves, st) : dp == 64 ? launch<T, 64>(A, waves, st) : launch<T, 128>(A, waves, st);
}

}  // namespace

hipError_t launch_attention_dq(const AttnRun& A, int waves, hipStream_t st) {
    return A.type == GOI_BF16 ? launch<bf16>(A, waves, st) : launch<f16>(A, waves, st);
}

}  // namespace goi
