// policy_attention_dkv.hip - the attention's backward pass over keys: dk = scale dS^T q and dv = P^T dout, summed over the
// query heads that share the key head. A wave keeps 32 keys (their k and v as the second operands, dk and dv as sums) and runs over
// the packed rows, whose tiles of q and dout the block's waves share in LDS; the scores come out rows x keys, so a lane
// holds 16 rows of ONE key and P and dS, rounded, are second operands as they stand (policy_attention.hpp).
#include "policy_attention.hpp"

namespace goi {
namespace {

// A tile of packed rows on its way to LDS. Rows that see no key are stored as zeros: what they hold (the steps after an
// episode's end, say) must not reach a sum.
template <typename T, int DP, int ROWS, int NT>
struct RowStage {
    static constexpr int N = ROWS * (DP / 8) / NT;
    int4_t q[N], go[N];
    bool in[N];
    __device__ __forceinline__ void load(const AttnRun& A, const T* qp, const T* gp, const RowInfo* info, int m0, int tid) {
        const GoiAttention& a = A.a;
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const int c = tid + j * NT, ch = c % (DP / 8), m = min(m0 + c / (DP / 8), A.rows - 1);
            const int i = m / A.group, hl = m - i * A.group, d = ch * 8 < a.dim ? ch * 8 : 0;
            q[j] = *reinterpret_cast<const int4_t*>(qp + i * a.q_strides[1] + hl * a.q_strides[2] + d);
            go[j] = *reinterpret_cast<const int4_t*>(gp + i * a.dout_strides[1] + hl * a.dout_strides[2] + d);
            in[j] = info[m].hi > info[m].lo && m0 + c / (DP / 8) < A.rows && ch * 8 < a.dim;
        }
    }
    __device__ __forceinline__ void store(T* qt, T* gt, int tid) const {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const int c = tid + j * NT, at = chunk_at<DP>(c / (DP / 8), c % (DP / 8));
            reinterpret_cast<int4_t*>(qt)[at] = in[j] ? q[j] : int4_t{0, 0, 0, 0};
            reinterpret_cast<int4_t*>(gt)[at] = in[j] ? go[j] : int4_t{0, 0, 0, 0};
        }
    }
};

// What the waves need of each row of a tile, in LDS
template <int ROWS>
struct RowValues {
    float top[ROWS], inv[ROWS], delta[ROWS];
    int lo[ROWS], hi[ROWS], pos[ROWS], table[ROWS];  // pos: position + origin; table: the head's offset in the bias table
};

template <typename T, int DP, int NW>
__global__ void __launch_bounds__(64 * NW) k_attention_dkv(const AttnRun A) {
    constexpr int NT = 64 * NW, RT = NW == 1 && DP == 128 ? 32 : 64, RB = RT / 32, NBUF = NW == 1 ? 1 : 2;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    __shared__ __attribute__((aligned(16))) RowValues<RT> values[NBUF];
    T* const tiles = reinterpret_cast<T*>(lds);  // [NBUF][q, dout][RT][DP]
    float* const table = reinterpret_cast<float*>(lds + NBUF * 2 * RT * DP * sizeof(T));
    const GoiAttention& a = A.a;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, half = lane >> 5;

    int place = xcd_place(blockIdx.x, gridDim.x);
    const int tile = place % A.tiles;  // in a causal window the first keys are seen by the most rows: they go first
    place /= A.tiles;
    const int n = place / a.kv_heads, g = place - n * a.kv_heads;
    const int L = history(A, n);
    const int block0 = tile * 32 * NW, block1 = min(block0 + 32 * NW, L);  // the block's keys
    const int key0 = block0 + wave * 32, key = key0 + (lane & 31);
    const int64_t pair = (int64_t)n * a.kv_heads + g;
    const RowInfo* const info = A.row_info + pair * A.rows;
    const BlockInfo* const blocks = A.block_info + pair * A.blocks;
    const T* const qp = static_cast<const T*>(a.q) + n * a.q_strides[0] + g * A.group * a.q_strides[2];
    const T* const gp = static_cast<const T*>(a.dout) + n * a.dout_strides[0] + g * A.group * a.dout_strides[2];
    if (a.bias) stage_bias(A, g, table, tid, NT);
    half8<T> k[DP / 16], v[DP / 16];
    load_operand<T, DP>(k, static_cast<const T*>(a.k) + n * a.k_strides[0] + key * a.k_strides[1] + g * a.k_strides[2],
                        key < L, a.dim, lane);
    load_operand<T, DP>(v, static_cast<const T*>(a.v) + n * a.v_strides[0] + key * a.v_strides[1] + g * a.v_strides[2],
                        key < L, a.dim, lane);
    float16_t dk[DP / 32], dv[DP / 32];
    clear(dk);
    clear(dv);

    // the next tile of RT rows at or after m0 with a row that sees a key of the block
    const auto seek = [&](int m0) {
        for (; m0 < A.rows; m0 += RT) {
            bool any = false;
            for (int b = 0; b < RB; ++b) {
                const int x = m0 / 32 + b;
                if (x < A.blocks) any = any || (blocks[x].lo < block1 && blocks[x].hi > block0);
            }
            if (any) break;
        }
        return m0;
    };
    RowStage<T, DP, RT, NT> stage;
    RowInfo mine{INFINITY, 0.0f, 0.0f, 0, 0};
    int my_pos = 0, my_table = 0;
    const auto load_values = [&](int m0) {
        const int m = m0 + tid;
        mine = RowInfo{INFINITY, 0.0f, 0.0f, 0, 0};
        if (tid < RT && m < A.rows) {
            mine = info[m];
            const int i = m / A.group;
            my_pos = L - a.q_steps + i + A.origin;
            my_table = (m - i * A.group) * a.n_distances;
        }
    };
    const auto store_values = [&](RowValues<RT>& to) {
        if (tid < RT) {
            to.top[tid] = mine.top;
            to.inv[tid] = mine.inv;
            to.delta[tid] = mine.delta;
            to.lo[tid] = mine.lo;
            to.hi[tid] = mine.hi;
            to.pos[tid] = my_pos;
            to.table[tid] = my_table;
        }
    };

    // in a causal order the rows before position block0 see none of the block's keys
    int m0 = 0;
    if (a.causal) m0 = (int)(min((int64_t)max(block0 - (L - a.q_steps), 0) * A.group, (int64_t)A.rows) / RT * RT);
    m0 = block0 < block1 ? seek(m0) : A.rows;
    if (m0 < A.rows) {
        stage.load(A, qp, gp, info, m0, tid);
        load_values(m0);
        stage.store(tiles, tiles + RT * DP, tid);
        store_values(values[0]);
    }
    __syncthreads();
    int buf = 0;
    while (m0 < A.rows) {
        const int next = seek(m0 + RT);
        if (next < A.rows) {
            stage.load(A, qp, gp, info, next, tid);
            load_values(next);
        }
        const T* const qt = tiles + buf * 2 * RT * DP;
        const T* const gt = qt + RT * DP;
        const RowValues<RT>& val = values[buf];
#pragma unroll
        for (int b = 0; b < RB; ++b) {
            const int x = m0 / 32 + b;
            if (x >= A.blocks) continue;
            const BlockInfo blk = blocks[x];
            if (blk.lo >= key0 + 32 || blk.hi <= key0) continue;
            float16_t p = raw_scores<T, DP>(qt, 32 * b, k, lane);
            float16_t ds = raw_scores<T, DP>(gt, 32 * b, v, lane);
            const bool full = key0 >= blk.full_lo && key0 + 32 <= blk.full_hi;
            const int one = a.bias ? one_distance(key0, blk.pos_lo, blk.pos_hi, a.n_distances) : 0;
#pragma unroll
            for (int r4 = 0; r4 < 4; ++r4) {
                const int row = 32 * b + 8 * r4 + 4 * half;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int r = 4 * r4 + e;
                    float s = p[r] * A.c;
                    if (a.bias) {
                        const int d = one >= 0 ? one : min(max(val.pos[row + e] - key, 0), a.n_distances - 1);
                        s += table[val.table[row + e] + d];
                    }
                    const float prob = exp2_fast(s - val.top[row + e]);
                    p[r] = prob * val.inv[row + e];
                    ds[r] = prob * (ds[r] * val.inv[row + e] - val.delta[row + e]);
                }
                if (!full) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int r = 4 * r4 + e;
                        const bool sees = key >= val.lo[row + e] && key < val.hi[row + e];
                        p[r] = sees ? p[r] : 0.0f;
                        ds[r] = sees ? ds[r] : 0.0f;
                    }
                }
            }
#pragma unroll
            for (int x2 = 0; x2 < 2; ++x2) {
                const half8<T> pf = to_operand<T>(p, x2), sf = to_operand<T>(ds, x2);
#pragma unroll
                for (int d = 0; d < DP / 32; ++d) {
                    dv[d] = mfma(column_fragment<T, DP>(gt, 32 * b + 16 * x2, 32 * d, lane), pf, dv[d]);
                    dk[d] = mfma(column_fragment<T, DP>(qt, 32 * b + 16 * x2, 32 * d, lane), sf, dk[d]);
                }
            }
        }
        if (NBUF == 1) __syncthreads();
        else buf ^= 1;
        if (next < A.rows) {
            stage.store(tiles + buf * 2 * RT * DP, tiles + buf * 2 * RT * DP + RT * DP, tid);
            store_values(values[buf]);
        }
        __syncthreads();
        m0 = next;
    }
    if (key >= a.k_steps) return;
    T* const to_k = static_cast<T*>(a.dk) + n * a.dk_strides[0] + key * a.dk_strides[1] + g * a.dk_strides[2];
    T* const to_v = static_cast<T*>(a.dv) + n * a.dv_strides[0] + key * a.dv_strides[1] + g * a.dv_strides[2];
    store_row<T, DP>(to_k, dk, a.scale, a.dim, half);
    store_row<T, DP>(to_v, dv, 1.0f, a.dim, half);
}

template <typename T, int DP, int NW>
hipError_t launch(const AttnRun& A, hipStream_t st) {
    constexpr int RT = NW == 1 && DP == 128 ? 32 : 64, NBUF = NW == 1 ? 1 : 2;
    const size_t lds = NBUF * 2 * RT * DP * sizeof(T) + (A.a.bias ? (size_t)A.group * A.a.n_distances * sizeof(float) : 0);
    (void)hipFuncSetAttribute(reinterpret_cast<const void*>(k_attention_dkv<T, DP, NW>),
                              hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    hipLaunchKernelGGL((k_attention_dkv<T, DP, NW>), dim3((unsigned)((int64_t)A.a.n_worlds * A.a.kv_heads * A.tiles)),
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

hipError_t launch_attention_dkv(const AttnRun& A, int waves, hipStream_t st) {
    return A.a.type == GOI_BF16 ? launch<bf16>(A, waves, st) : launch<f16>(A, waves, st);
}

}  // namespace goi
