// fp8_quant_kernels.hip -- everything around the 8-bit matrix product (fp8_gemm_kernels.hip) that is bound by memory: quantising rows and
// weights to E4M3 with a scale per group of 128 (formats: fp8_common.h), RMSNorm + residual with a quantised result, and the way back.
// One pass over the data everywhere: a group of 128 is 16 lanes x 8 elements, its maximum four DPP rotations inside a 16-lane row, and the
// values stay in registers between the maximum and the conversion.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/dynam3d_hip.h"
#include "d3d_common.h"
#include "fp8_common.h"

namespace {

__device__ __forceinline__ void store_scale(void* scale, int64_t idx, int kind, uint32_t code, float s) {
    if (kind == 0) ((uint8_t*)scale)[idx] = (uint8_t)code;
    else ((float*)scale)[idx] = s;
}

// ---- rows -> E4M3 ---------------------------------------------------------------------------------------------------------------------
template <int DT>
__global__ void __launch_bounds__(256)
k_fp8_quant_rows(const void* __restrict__ x, uint8_t* __restrict__ q, void* __restrict__ scale, int rows, int K, int KB, int64_t ldx, int64_t ldq,
                 int64_t lds, int kind) {
    const int64_t g = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4);
    if (g >= (int64_t)rows * KB) return;                         // (whole 16-lane rows leave together)
    const int row = (int)(g / KB), kb = (int)(g - (int64_t)row * KB);
    const int k = kb * FP8_G + (threadIdx.x & 15) * 8;
    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (k < K) fp_load8<DT>(x, (int64_t)row * ldx + k, v);
    float a = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) a = fmaxf(a, fp8_finite_abs(v[i]));
    a = row16_max(a);
    uint32_t o[2], code;
    float s;
    fp8_quantize_pack<8>(v, a, kind, o, code, s);
    if (k < K) *reinterpret_cast<uint2*>(q + (int64_t)row * ldq + k) = make_uint2(o[0], o[1]);
    if ((threadIdx.x & 15) == 0) store_scale(scale, (int64_t)row * lds + kb, kind, code, s);
}

// ---- RMSNorm [+ residual] -> E4M3 --------------------------------------------------------------------------------------------------------
// A workgroup per row, NCH chunks of 8 elements per thread held in registers (the row is read once), as many waves as that leaves: 2 chunks up to D = 4096, 3 up to
// 6144, 4 up to 16384.  HBM bound: 6568 x 3072 bf16 + residual 26.5 us = 5.3 TB/s.  One chunk per thread (more waves, each with its own reductions) took 20.5 us
// for 6568 x 3072 without residual against 17.1, 18.9 for 2000 x 8192 against 16.1; 256 threads for every D 34.0 for 30000 x 1024 against 23.1.
template <int DT, int NCH>
__global__ void __launch_bounds__(512)
k_fp8_rms_norm(const void* __restrict__ x, const void* __restrict__ residual, const float* __restrict__ w, void* __restrict__ sum,
               uint8_t* __restrict__ q, void* __restrict__ scale, int D, int64_t ldx, int64_t ldr, int64_t ldsum, int64_t ldq, int64_t lds,
               float eps, int kind) {
    __shared__ float part[8];
    const int lane = threadIdx.x, row = blockIdx.x, T = blockDim.x;
    float v[NCH][8];
    float ss = 0.f;
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
        const int k = (c * T + lane) * 8;
        if (k < D) {
            fp_load8<DT>(x, (int64_t)row * ldx + k, v[c]);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[c][i] = 0.f;
        }
    }
    if (residual) {
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
            const int k = (c * T + lane) * 8;
            if (k < D) {
                float r[8];
                fp_load8<DT>(residual, (int64_t)row * ldr + k, r);
#pragma unroll
                for (int i = 0; i < 8; ++i) v[c][i] += r[i];
                if constexpr (DT != 2) {                         // the stream is kept in 16 bits: what the next layer reads is what is normalised
#pragma unroll
                    for (int i = 0; i < 8; i += 2) {
                        const uint32_t u = fp_pack2<DT>(v[c][i], v[c][i + 1]);
                        v[c][i] = fp_to_f32<DT>((uint16_t)(u & 0xffffu));
                        v[c][i + 1] = fp_to_f32<DT>((uint16_t)(u >> 16));
                    }
                }
                fp_store8<DT>(sum, (int64_t)row * ldsum + k, v[c]);
            }
        }
    }
#pragma unroll
    for (int c = 0; c < NCH; ++c)
#pragma unroll
        for (int i = 0; i < 8; ++i) ss += v[c][i] * v[c][i];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) ss += __shfl_xor(ss, o, 64);
    if ((lane & 63) == 0) part[lane >> 6] = ss;
    __syncthreads();
    ss = part[0];
    for (int i = 1; i < T >> 6; ++i) ss += part[i];
    const float r = 1.f / sqrtf(ss / (float)D + eps);
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
        const int k = (c * T + lane) * 8;
        float a = 0.f;
        if (k < D) {
            float g[8];
            fp_load8<2>(w, k, g);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                v[c][i] = v[c][i] * r * g[i];
                a = fmaxf(a, fp8_finite_abs(v[c][i]));
            }
        }
        a = row16_max(a);
        uint32_t o[2], code;
        float s;
        fp8_quantize_pack<8>(v[c], a, kind, o, code, s);
        if (k < D) {
            *reinterpret_cast<uint2*>(q + (int64_t)row * ldq + k) = make_uint2(o[0], o[1]);
            if ((lane & 15) == 0) store_scale(scale, (int64_t)row * lds + k / FP8_G, kind, code, s);
        }
    }
}

// ---- weights -> E4M3, one scale per 128 x 128 block (once per weight) -----------------------------------------------------------------------
template <int DT>
__global__ void __launch_bounds__(256)
k_fp8_quant_block(const void* __restrict__ w, uint8_t* __restrict__ q, void* __restrict__ scale, int rows, int K, int64_t ldw, int64_t ldq, int64_t lds,
                  int kind) {
    __shared__ float part[4];
    const int r0 = blockIdx.y * FP8_G + (threadIdx.x >> 4);
    const int k = blockIdx.x * FP8_G + (threadIdx.x & 15) * 8;
    float v[8][8];
    float a = 0.f;
#pragma unroll
    for (int p = 0; p < 8; ++p) {
        const int row = r0 + p * 16;
        if (row < rows && k < K) {
            fp_load8<DT>(w, (int64_t)row * ldw + k, v[p]);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[p][i] = 0.f;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) a = fmaxf(a, fp8_finite_abs(v[p][i]));
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) a = fmaxf(a, __shfl_xor(a, o, 64));
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = a;
    __syncthreads();
    a = fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3]));
    uint32_t code = 0;
    float s = 0.f;
#pragma unroll
    for (int p = 0; p < 8; ++p) {
        const int row = r0 + p * 16;
        uint32_t o[2];
        fp8_quantize_pack<8>(v[p], a, kind, o, code, s);
        if (row < rows && k < K) *reinterpret_cast<uint2*>(q + (int64_t)row * ldq + k) = make_uint2(o[0], o[1]);
    }
    if (threadIdx.x == 0) store_scale(scale, (int64_t)blockIdx.y * lds + blockIdx.x, kind, code, s);
}

// ---- E4M3 -> bf16 / fp16 / float32: x = q * s, rounded once -----------------------------------------------------------------------------------
template <int DT>
__global__ void __launch_bounds__(256)
k_fp8_dequantize(const uint8_t* __restrict__ q, const void* __restrict__ scale, void* __restrict__ x, int rows, int K, int K16, int64_t ldq, int64_t lds,
                 int64_t ldx, int group_rows_log2, int kind) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= (int64_t)rows * K16) return;
    const int row = (int)(i / K16), k = (int)(i - (int64_t)row * K16) * 16;
    const uint4 r = *reinterpret_cast<const uint4*>(q + (int64_t)row * ldq + k);
    const int64_t si = (int64_t)(row >> group_rows_log2) * lds + k / FP8_G;
    const float s = kind == 0 ? e8m0_value(((const uint8_t*)scale)[si]) : ((const float*)scale)[si];
    const uint32_t u[4] = {r.x, r.y, r.z, r.w};
    float v[16];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)u[j], false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)u[j], true);
        v[4 * j] = lo[0] * s;
        v[4 * j + 1] = lo[1] * s;
        v[4 * j + 2] = hi[0] * s;
        v[4 * j + 3] = hi[1] * s;
    }
    fp_store8<DT>(x, (int64_t)row * ldx + k, v);
    fp_store8<DT>(x, (int64_t)row * ldx + k + 8, v + 8);
}

int32_t bad(const char* msg) {
    d3d_set_error_(msg);
    return D3D_EINVAL;
}

bool aligned(const void* p, int64_t ld, int32_t elem_bytes) { return ((uintptr_t)p & 15) == 0 && (ld * elem_bytes) % 16 == 0; }
int32_t elem_bytes(int32_t dtype) { return dtype == 2 ? 4 : 2; }
bool blocks_ok(int64_t n, int64_t threads = 256) { return n * threads < (int64_t)1 << 32; }        // (a launch has less than 2^32 threads)

#define D3D_BY_DTYPE(dtype, CALL) \
    do {                          \
        if ((dtype) == 0) {       \
            CALL(0);              \
        } else if ((dtype) == 1) { \
            CALL(1);              \
        } else {                  \
            CALL(2);              \
        }                         \
    } while (0)

}  // namespace

extern "C" {

int32_t d3d_fp8_quantize(const void* x, void* q, void* scale, int32_t rows, int32_t K, int64_t ldx, int64_t ldq, int64_t lds, int32_t dtype,
                         int32_t scale_kind, void* stream) {
    if (rows < 0 || K < 0 || K % 16 || dtype < 0 || dtype > 2 || scale_kind < 0 || scale_kind > 1) return bad("d3d_fp8_quantize: bad sizes (K must be a multiple of 16) or types");
    if (rows == 0 || K == 0) return D3D_OK;
    if (!x || !q || !scale || !aligned(x, ldx, elem_bytes(dtype)) || !aligned(q, ldq, 1)) return bad("d3d_fp8_quantize: rows must start on 16 bytes");
    const int KB = (int)(((int64_t)K + FP8_G - 1) / FP8_G);            // (K up to 2^31 - 16)
    const int64_t nb = ((int64_t)rows * KB + 15) / 16;
    if (!blocks_ok(nb)) return bad("d3d_fp8_quantize: too many groups for one launch");
#define CALL(DT) \
    hipLaunchKernelGGL((k_fp8_quant_rows<DT>), dim3((uint32_t)nb), dim3(256), 0, (hipStream_t)stream, x, (uint8_t*)q, scale, rows, K, KB, ldx, ldq, lds, scale_kind)
    D3D_BY_DTYPE(dtype, CALL);
#undef CALL
    D3D_LAUNCH_CHECK();
}

int32_t d3d_fp8_quantize_weight(const void* w, void* q, void* scale, int32_t rows, int32_t K, int64_t ldw, int64_t ldq, int64_t lds, int32_t dtype,
                                int32_t scale_kind, void* stream) {
    if (rows < 0 || K < 0 || K % 16 || dtype < 0 || dtype > 2 || scale_kind < 0 || scale_kind > 1) return bad("d3d_fp8_quantize_weight: bad sizes (K must be a multiple of 16) or types");
    if (rows == 0 || K == 0) return D3D_OK;
    if (!w || !q || !scale || !aligned(w, ldw, elem_bytes(dtype)) || !aligned(q, ldq, 1)) return bad("d3d_fp8_quantize_weight: rows must start on 16 bytes");
    const int KB = (int)(((int64_t)K + FP8_G - 1) / FP8_G), NB = (int)(((int64_t)rows + FP8_G - 1) / FP8_G);
    if (NB > 65535) return bad("d3d_fp8_quantize_weight: more than 65535 blocks of rows");
#define CALL(DT) \
    hipLaunchKernelGGL((k_fp8_quant_block<DT>), dim3(KB, NB), dim3(256), 0, (hipStream_t)stream, w, (uint8_t*)q, scale, rows, K, ldw, ldq, lds, scale_kind)
    D3D_BY_DTYPE(dtype, CALL);
#undef CALL
    D3D_LAUNCH_CHECK();
}

int32_t d3d_fp8_dequantize(const void* q, const void* scale, void* x, int32_t rows, int32_t K, int64_t ldq, int64_t lds, int64_t ldx, int32_t group_rows,
                           int32_t dtype, int32_t scale_kind, void* stream) {
    if (rows < 0 || K < 0 || K % 16 || dtype < 0 || dtype > 2 || scale_kind < 0 || scale_kind > 1 || (group_rows != 1 && group_rows != FP8_G))
        return bad("d3d_fp8_dequantize: bad sizes (K must be a multiple of 16) or types");
    if (rows == 0 || K == 0) return D3D_OK;
    if (!x || !q || !scale || !aligned(x, ldx, elem_bytes(dtype)) || !aligned(q, ldq, 1)) return bad("d3d_fp8_dequantize: rows must start on 16 bytes");
    const int64_t nb = ((int64_t)rows * (K / 16) + 255) / 256;
    if (!blocks_ok(nb)) return bad("d3d_fp8_dequantize: too many elements for one launch");
#define CALL(DT)                                                                                                                                        \
    hipLaunchKernelGGL((k_fp8_dequantize<DT>), dim3((uint32_t)nb), dim3(256), 0, (hipStream_t)stream, (const uint8_t*)q, scale, x, rows, K, K / 16, ldq, lds, ldx, \
                       group_rows == 1 ? 0 : 7, scale_kind)
    D3D_BY_DTYPE(dtype, CALL);
#undef CALL
    D3D_LAUNCH_CHECK();
}

int32_t d3d_fp8_rms_norm(const void* x, const void* residual, const float* w, void* sum, void* q, void* scale, int32_t rows, int32_t D, int64_t ldx,
                         int64_t ldr, int64_t ldsum, int64_t ldq, int64_t lds, float eps, int32_t dtype, int32_t scale_kind, void* stream) {
    if (rows < 0 || D <= 0 || D % 16 || D > 16384 || dtype < 0 || dtype > 2 || scale_kind < 0 || scale_kind > 1)
        return bad("d3d_fp8_rms_norm: bad sizes (D must be a multiple of 16, at most 16384) or types");
    if (rows == 0) return D3D_OK;
    const int32_t eb = elem_bytes(dtype);
    if (!x || !q || !scale || !w || ((uintptr_t)w & 15) || !aligned(x, ldx, eb) || !aligned(q, ldq, 1)) return bad("d3d_fp8_rms_norm: rows must start on 16 bytes");
    if (residual && (!sum || !aligned(residual, ldr, eb) || !aligned(sum, ldsum, eb))) return bad("d3d_fp8_rms_norm: residual and sum rows must start on 16 bytes");
    const int32_t nch = D <= 4096 ? 2 : D <= 6144 ? 3 : 4, threads = (D + nch * 512 - 1) / (nch * 512) * 64;
    if (!blocks_ok(rows, threads)) return bad("d3d_fp8_rms_norm: too many rows for one launch");
#define ROWS(DT, NCH)                                                                                                                            \
    hipLaunchKernelGGL((k_fp8_rms_norm<DT, NCH>), dim3((uint32_t)rows), dim3(threads), 0, (hipStream_t)stream, x, residual, w, sum, (uint8_t*)q, scale, D, ldx, \
                       ldr, ldsum, ldq, lds, eps, scale_kind)
#define CALL(DT)                           \
    do {                                   \
        if (nch == 2) ROWS(DT, 2);         \
        else if (nch == 3) ROWS(DT, 3);    \
        else ROWS(DT, 4);                  \
    } while (0)
    D3D_BY_DTYPE(dtype, CALL);
#undef CALL
#undef ROWS
    D3D_LAUNCH_CHECK();
}

}  // extern "C"
