// policy_int8.hip - product in 8-bit integers with a scale for each row and each channel (include/goi_policy.h), on the
// 8-bit matrix instructions with int32 sums: exact, so neither the tiling nor the order shows in the result.
#include <algorithm>

#include "policy.hpp"

namespace goi {
namespace {

typedef int int16v __attribute__((ext_vector_type(16)));

__device__ __forceinline__ int16v mfma(int4_t a, int4_t b, int16v c) {
    return __builtin_amdgcn_mfma_i32_32x32x32_i8(a, b, c, 0, 0, 0);
}

// 16 bytes of a row from k on, zeros past width
__device__ __forceinline__ int4_t row_bytes(const int8_t* row, int k, int width) {
    if (k + 16 <= width) return *reinterpret_cast<const int4_t*>(row + k);
    union {
        int4_t v;
        int8_t b[16];
    } u;
    u.v = int4_t{0, 0, 0, 0};
    for (int e = 0; k + e < width; ++e) u.b[e] = row[k + e];
    return u.v;
}

__device__ __forceinline__ float bias_at(const GoiInt8& a, int n) {
    if (!a.bias) return 0.0f;
    if (a.bias_type == GOI_F32) return static_cast<const float*>(a.bias)[n];
    if (a.bias_type == GOI_F16) return (float)static_cast<const f16*>(a.bias)[n];
    return (float)static_cast<const bf16*>(a.bias)[n];
}

// Few rows: a block takes 16 channels and up to 16 MB rows. Its four waves share the channels' weights along k, 64 bytes a step,
// straight from memory into the operands, and add their sums up in LDS: each weight is read once. Bound by the weights'
// bytes, or by latency.
template <typename T, int MB>
__global__ void __launch_bounds__(256) k_int8_few(const GoiInt8 a) {
    __shared__ int4_t shared[4][MB][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int n0 = blockIdx.x * 16, m0 = blockIdx.y * 16 * MB, n = n0 + (lane & 15);
    const int8_t* const w = a.w + (int64_t)min(n, a.channels - 1) * a.w_stride;
    int4_t c[MB];
#pragma unroll
    for (int b = 0; b < MB; ++b) c[b] = int4_t{0, 0, 0, 0};
#pragma unroll 4
    for (int k = wave * 64 + 16 * (lane >> 4); k - 16 * (lane >> 4) < a.width; k += 256) {
        const int4_t x = row_bytes(w, k, a.width);
#pragma unroll
        for (int b = 0; b < MB; ++b) {
            const int m = min(m0 + 16 * b + (lane & 15), a.rows - 1);
            c[b] = __builtin_amdgcn_mfma_i32_16x16x64_i8(x, row_bytes(a.x + (int64_t)m * a.x_stride, k, a.width), c[b], 0, 0, 0);
        }
    }
#pragma unroll
    for (int b = 0; b < MB; ++b) shared[wave][b][lane] = c[b];
    __syncthreads();
    // wave w finishes row block w: lane l has row l & 15 and channels 4 (l >> 4) .. + 3
    for (int b = wave; b < MB; b += 4) {
        const int4_t s = (shared[0][b][lane] + shared[1][b][lane]) + (shared[2][b][lane] + shared[3][b][lane]);
        const int m = m0 + 16 * b + (lane & 15), at = n0 + 4 * (lane >> 4);
        if (m >= a.rows) continue;
        const float f = a.x_scales[m];
        T* const y = static_cast<T*>(a.y) + (int64_t)m * a.y_stride;
        for (int e = 0; e < 4; ++e)
            if (at + e < a.channels) y[at + e] = (T)((float)s[e] * f * a.w_scales[at + e] + bias_at(a, at + e));
    }
}

// Many rows: tiles of BM rows and BN channels, four waves of half of each, 128 bytes of k a step through two LDS tiles: the next
// step's loads are in flight while this one is multiplied.
template <typename T, int BM, int BN>
__global__ void __launch_bounds__(256) k_int8(const GoiInt8 a, int tiles_n) {
    constexpr int WM = BM / 2, WN = BN / 2, RM = WM / 32, RN = WN / 32, NX = BM * 8 / 256, NW = BN * 8 / 256;
    extern __shared__ __attribute__((aligned(16))) char lds[];  // [2][BM + BN][128]
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, half = lane >> 5;
    const int place = xcd_place(blockIdx.x, gridDim.x);
    const int m0 = place / tiles_n * BM, n0 = place % tiles_n * BN;
    int4_t xs[NX], ws[NW];
    const auto load = [&](int k0) {
#pragma unroll
        for (int j = 0; j < NX; ++j) {
            const int c = tid + j * 256, m = min(m0 + (c >> 3), a.rows - 1);
            xs[j] = row_bytes(a.x + (int64_t)m * a.x_stride, k0 + 16 * (c & 7), a.width);
        }
#pragma unroll
        for (int j = 0; j < NW; ++j) {
            const int c = tid + j * 256, n = min(n0 + (c >> 3), a.channels - 1);
            ws[j] = row_bytes(a.w + (int64_t)n * a.w_stride, k0 + 16 * (c & 7), a.width);
        }
    };
    const auto store = [&](int buf) {
        int4_t* const x = reinterpret_cast<int4_t*>(lds + buf * (BM + BN) * 128);
        int4_t* const w = x + BM * 8;
#pragma unroll
        for (int j = 0; j < NX; ++j) x[chunk_at<64>((tid + j * 256) >> 3, tid & 7)] = xs[j];
#pragma unroll
        for (int j = 0; j < NW; ++j) w[chunk_at<64>((tid + j * 256) >> 3, tid & 7)] = ws[j];
    };
    int16v c[RM][RN];
#pragma unroll
    for (int i = 0; i < RM; ++i)
#pragma unroll
        for (int j = 0; j < RN; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) c[i][j][r] = 0;
    load(0);
    store(0);
    __syncthreads();
    int buf = 0;
    for (int k0 = 0; k0 < a.width; k0 += 128) {
        const bool more = k0 + 128 < a.width;
        if (more) load(k0 + 128);
        const int4_t* const x = reinterpret_cast<const int4_t*>(lds + buf * (BM + BN) * 128);
        const int4_t* const w = x + BM * 8;
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            int4_t fx[RM], fw[RN];
#pragma unroll
            for (int i = 0; i < RM; ++i) fx[i] = x[chunk_at<64>((wave >> 1) * WM + 32 * i + (lane & 31), 2 * s + half)];
#pragma unroll
            for (int j = 0; j < RN; ++j) fw[j] = w[chunk_at<64>((wave & 1) * WN + 32 * j + (lane & 31), 2 * s + half)];
#pragma unroll
            for (int i = 0; i < RM; ++i)
#pragma unroll
                for (int j = 0; j < RN; ++j) c[i][j] = mfma(fx[i], fw[j], c[i][j]);
        }
        buf ^= 1;
        if (more) store(buf);
        __syncthreads();
    }
#pragma unroll
    for (int j = 0; j < RN; ++j) {
        const int n = n0 + (wave & 1) * WN + 32 * j + (lane & 31);
        if (n >= a.channels) continue;
        const float f = a.w_scales[n], b = bias_at(a, n);
#pragma unroll
        for (int i = 0; i < RM; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int m = m0 + (wave >> 1) * WM + 32 * i + mfma_row(r, half);
                if (m < a.rows) static_cast<T*>(a.y)[(int64_t)m * a.y_stride + n] = (T)((float)c[i][j][r] * a.x_scales[m] * f + b);
            }
    }
}

template <typename T, int BM, int BN>
void launch_tiles(const GoiInt8& a, hipStream_t st) {
    const int tiles_m = (a.rows + BM - 1) / BM, tiles_n = (a.channels + BN - 1) / BN;
    (void)hipFuncSetAttribute(reinterpret_cast<const void*>(k_int8<T, BM, BN>), hipFuncAttributeMaxDynamicSharedMemorySize,
                              2 * (BM + BN) * 128);
    hipLaunchKernelGGL((k_int8<T, BM, BN>), dim3((unsigned)((int64_t)tiles_m * tiles_n)), dim3(256), 2 * (BM + BN) * 128, st, a,
                       tiles_n);
}

template <typename T>
void launch(const GoiInt8& a, hipStream_t st) {
    const dim3 few((a.channels + 15) / 16, 1);
    if (a.rows <= 16) hipLaunchKernelGGL((k_int8_few<T, 1>), few, dim3(256), 0, st, a);
    else if (a.rows <= 32) hipLaunchKernelGGL((k_int8_few<T, 2>), few, dim3(256), 0, st, a);
    else if (a.rows <= 64) hipLaunchKernelGGL((k_int8_few<T, 4>), few, dim3(256), 0, st, a);
    else if ((int64_t)((a.rows + 127) / 128) * ((a.channels + 127) / 128) >= 256) launch_tiles<T, 128, 128>(a, st);
    else launch_tiles<T, 64, 64>(a, st);
}

}  // namespace
}  // namespace goi

using namespace goi;

extern "C" int32_t goi_linear_int8(const GoiInt8* a, void* hip_stream) {
    const char* const who = "goi_linear_int8";
    if (!a) return policy_error(GOI_E_ARG, "%s: null argument", who);
    if (a->rows < 0 || a->channels < 0 || a->width < 1) return policy_error(GOI_E_ARG, "%s: negative sizes or no width", who);
    if (a->width > 131071) return policy_error(GOI_E_UNSUPPORTED, "%s: width above 131071", who);
    if (a->type != GOI_F32 && a->type != GOI_F16 && a->type != GOI_BF16)
        return policy_error(GOI_E_UNSUPPORTED, "%s: unknown type", who);
    if (a->bias && a->bias_type != a->type && a->bias_type != GOI_F32)
        return policy_error(GOI_E_UNSUPPORTED, "%s: the bias is of another 16-bit type", who);
    if (a->rows == 0 || a->channels == 0) return GOI_OK;
    if (!a->x || !a->w || !a->x_scales || !a->w_scales || !a->y) return policy_error(GOI_E_ARG, "%s: null argument", who);
    if (((uintptr_t)a->x | (uintptr_t)a->w | (uintptr_t)a->x_stride | (uintptr_t)a->w_stride) & 15)
        return policy_error(GOI_E_ARG, "%s: x and w need 16-byte aligned rows", who);
    if ((int64_t)((a->rows + 63) / 64) * ((a->channels + 63) / 64) > 0x7fffffff)
        return policy_error(GOI_E_UNSUPPORTED, "%s: more than 2^31 tiles", who);
    const hipStream_t st = static_cast<hipStream_t>(hip_stream);
    if (a->type == GOI_F32) launch<float>(*a, st);
    else if (a->type == GOI_F16) launch<f16>(*a, st);
    else launch<bf16>(*a, st);
    return launch_error(who);
}
