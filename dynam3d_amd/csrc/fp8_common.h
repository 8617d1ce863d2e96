// fp8_common.h -- the 8-bit number format of fp8_quant_kernels.hip and fp8_gemm_kernels.hip: OCP E4M3 values (largest 448, no infinity, one
// NaN) in groups of 128 along K, one scale per group (activations: per row; weights: per 128 x 128 block).
//
//   scale kinds   0  E8M0: s = 2^max(-126, ceil(log2(amax / 448))), stored as the byte e + 127.  A power of two divides without rounding,
//                    and v_mfma_scale_* applies it to the operand inside the matrix core: no vector work in the K loop.
//                 1  float32: s = max(amax / 448, 2^-126), divided by with IEEE rounding.
//   amax runs over the FINITE members of the group; a member that is not finite becomes E4M3's NaN and stays visible in every product.
#pragma once
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace {

constexpr int FP8_G = 128;            // elements per scale along K

__device__ __forceinline__ float fp8_finite_abs(float v) {
    const float a = __builtin_fabsf(v);
    return a < __builtin_inff() ? a : 0.f;
}

// byte of the E8M0 scale for a group maximum (finite, >= 0).  448 = 1.75 * 2^8: one binade more when the significand exceeds 1.75.
__device__ __forceinline__ uint32_t e8m0_of_amax(float amax) {
    const uint32_t u = __float_as_uint(amax);
    const int code = (int)(u >> 23) - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
    return (uint32_t)(code < 1 ? 1 : code);
}
__device__ __forceinline__ float e8m0_value(uint32_t code) {                 // 2^(code - 127); 0 = 2^-127 (a float32 denormal), 255 = NaN
    return code == 255u ? __builtin_nanf("") : code == 0u ? __uint_as_float(0x00400000u) : __uint_as_float(code << 23);
}
__device__ __forceinline__ float e8m0_inverse(uint32_t code) {               // 2^(127 - code) for the codes e8m0_of_amax makes (1 .. 247)
    return __uint_as_float((254u - code) << 23);
}

// two float32 -> two E4M3 bytes in the low / high half of `old` (round to nearest even; |v| <= 448 or NaN: v_cvt_pk_fp8_f32 never saturates here)
template <bool HI>
__device__ __forceinline__ uint32_t fp8_pack2(float a, float b, uint32_t old) {
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(a, b, (int)old, HI);
}

// Quantises N values (N % 4 == 0) of one group with its maximum known; returns the packed bytes in `out`, the scale through `code` / `s`.
template <int N>
__device__ __forceinline__ void fp8_quantize_pack(const float* v, float amax, int kind, uint32_t* out, uint32_t& code, float& s) {
    float t[N];
    if (kind == 0) {
        code = e8m0_of_amax(amax);
        s = e8m0_value(code);
        const float inv = e8m0_inverse(code);
#pragma unroll
        for (int i = 0; i < N; ++i) t[i] = v[i] * inv;                       // exact (a power of two; the result is far from denormal, or rounds to 0)
    } else {
        code = 0;
        s = fmaxf(amax / 448.f, 0x1p-126f);
        if (s >= 0x1p-80f) {
            // v / s correctly rounded, without a division per value: r = 1 / s rounded, t = v r is off by two steps at most, and each
            // t += r (v - t s), the remainder exact, makes it the neighbour and then the nearest (Markstein).  (The remainder of a v that does not round
            // to 0 in E4M3, |v| >= 2^-10 s, is far from the denormals here.)  fp16 4617 x 4112 with float32 scales: 30.2 us with divisions and the threads of
            // the time, 22.4; quantising 6568 x 3072 18.5 -> 15.9.
            const float r = 1.f / s;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                t[i] = v[i] * r;
                t[i] = __builtin_fmaf(__builtin_fmaf(-t[i], s, v[i]), r, t[i]);
                t[i] = __builtin_fmaf(__builtin_fmaf(-t[i], s, v[i]), r, t[i]);
            }
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) t[i] = v[i] / s;
        }
    }
#pragma unroll
    for (int i = 0; i < N; ++i)
        if (!(__builtin_fabsf(v[i]) < __builtin_inff())) t[i] = __builtin_nanf("");
#pragma unroll
    for (int i = 0; i < N; i += 4) out[i / 4] = fp8_pack2<true>(t[i + 2], t[i + 3], fp8_pack2<false>(t[i], t[i + 1], 0u));
}

// maximum over the 16 lanes of a DPP row, in every lane
__device__ __forceinline__ float row16_max(float v) {
#define D3D_ROW_MAX(ctrl) v = fmaxf(v, __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(v), ctrl, 0xf, 0xf, true)))
    D3D_ROW_MAX(0x128);      // row_ror:8
    D3D_ROW_MAX(0x124);
    D3D_ROW_MAX(0x122);
    D3D_ROW_MAX(0x121);
#undef D3D_ROW_MAX
    return v;
}

// element types of the 16 / 32-bit side: 0 bf16, 1 fp16, 2 float32
template <int DT>
struct FpElem {
    static constexpr int BYTES = DT == 2 ? 4 : 2;
};
template <int DT>
__device__ __forceinline__ float fp_to_f32(uint16_t v) {
    if constexpr (DT == 0) return __uint_as_float((uint32_t)v << 16);
    else return __half2float(__ushort_as_half(v));
}
// two values, rounded to nearest even (hardware converters: NaN-safe)
template <int DT>
__device__ __forceinline__ uint32_t fp_pack2(float lo, float hi) {
    if constexpr (DT == 0) {
        typedef __bf16 b2 __attribute__((ext_vector_type(2)));
        typedef float f2 __attribute__((ext_vector_type(2)));
        const b2 r = __builtin_convertvector(f2{lo, hi}, b2);
        return *reinterpret_cast<const uint32_t*>(&r);
    } else {
        const __half2 h = __halves2half2(__float2half_rn(lo), __float2half_rn(hi));
        return *reinterpret_cast<const uint32_t*>(&h);
    }
}
// 8 consecutive elements (16-byte aligned; float32: 32 bytes)
template <int DT>
__device__ __forceinline__ void fp_load8(const void* base, int64_t idx, float* v) {
    if constexpr (DT == 2) {
        const float4 a = *reinterpret_cast<const float4*>((const float*)base + idx), b = *reinterpret_cast<const float4*>((const float*)base + idx + 4);
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
        const uint4 r = *reinterpret_cast<const uint4*>((const uint16_t*)base + idx);
        const uint32_t u[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = fp_to_f32<DT>((uint16_t)(u[i] & 0xffffu));
            v[2 * i + 1] = fp_to_f32<DT>((uint16_t)(u[i] >> 16));
        }
    }
}
template <int DT>
__device__ __forceinline__ void fp_store8(void* base, int64_t idx, const float* v) {
    if constexpr (DT == 2) {
        *reinterpret_cast<float4*>((float*)base + idx) = make_float4(v[0], v[1], v[2], v[3]);
        *reinterpret_cast<float4*>((float*)base + idx + 4) = make_float4(v[4], v[5], v[6], v[7]);
    } else {
        *reinterpret_cast<uint4*>((uint16_t*)base + idx) =
            make_uint4(fp_pack2<DT>(v[0], v[1]), fp_pack2<DT>(v[2], v[3]), fp_pack2<DT>(v[4], v[5]), fp_pack2<DT>(v[6], v[7]));
    }
}

}  // namespace
