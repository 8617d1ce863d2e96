// fp8_gemm_kernels.hip -- the 8-bit "NT" matrix product of the language model's linears on gfx950:
//
//   y[m, n] = sum_b sx[m, b] sw[n / 128, b] sum_{k in block b} xq[m, k] wq[n, k]     (+ bias[n] + residual[m, n], or SwiGLU over two halves)
//
// xq (M, K), wq (N, K) E4M3, one scale per row and 128 columns of x and per 128 x 128 block of w (fp8_common.h: E8M0 or float32).  Sums are
// float32; the result is rounded once, to bf16 / fp16 / float32 -- or, behind SwiGLU, quantised again for the product that follows.
//
// What the 8-bit matrix instructions round (measured, all shapes alike): 8 neighbouring products are aligned to the largest of them and cut 13
// bits below it, then added to the float32 accumulator.  A product loses less than 2^-13 of the largest beside it, at most 7 * 2^-13 sum |x w| in
// all and ~2^-14 of a result of random signs: far inside half a step of bf16 (2^-9), below one of fp16 (2^-12), but not of float32, and not of a 16-bit
// result of which most has cancelled.  A float32 result, and any other that the caller asks for, is therefore computed EXACTly: E4M3 converted to bf16 in
// registers (exact), products on the bf16 matrix instruction (exact, aligned to 24 bits), half the rate.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <atomic>
#include <type_traits>
#include <utility>

#include "../../include/dynam3d_hip.h"
#include "d3d_common.h"
#include "fp8_common.h"

namespace {

using v8i = __attribute__((ext_vector_type(8))) int;
using v4i = __attribute__((ext_vector_type(4))) int;
using v4f = __attribute__((ext_vector_type(4))) float;

struct GemmArgs {
    const uint8_t *x, *w;
    const void *sx, *sw;
    const void *bias, *res;
    void *out, *out_scale;
    float* ws;                       // split K: [slices][M][ldws] float32, else null
    int64_t ldx, ldw, ldsx, ldsw, ldr, ldo, ldos, ldws;
    int M, N, K, KB;                 // N = rows of w (SwiGLU: 2 I); KB = groups along K = K tiles
    int I;                           // SwiGLU: columns of the result
    int tiles_m, tiles_n, splits;
    int out_type;                    // 0 bf16, 1 fp16, 2 float32, 3 E4M3 + scale (SwiGLU)
    int exact;                       // asked for: EXACT for every result type
    int vec;                         // rows of out / res allow 4-column vector accesses
};

__device__ uint4 g_zero16;           // what the lanes behind the end of a ragged K read: an E4M3 zero can meet no NaN

// One 1 KiB piece (8 rows x 128 B) of an operand tile into LDS, 16 bytes per lane, no registers in between.  In asm so that the compiler does
// not drain it in front of every LDS read (it counts the builtin as a pending LDS write); the K loops wait for it explicitly.
// The wait states are the assembly's own business too: 1 behind a write of m0, 5 between a vector instruction that writes the scalar base (a v_readlane, where the base
// was spilled) and the load -- the instructions and the s_nop in front of it make 5 whatever the compiler puts before.
__device__ __forceinline__ void dma_piece(uint32_t voff, const uint8_t* base, uint32_t dst) {
    const uint32_t d = __builtin_amdgcn_readfirstlane(dst);
    uint32_t keep;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %2\n\ts_nop 2\n\tglobal_load_lds_dwordx4 %1, %3\n\ts_mov_b32 m0, %0"
                 : "=&s"(keep) : "v"(voff), "s"(d), "s"(base) : "memory");
}
__device__ __forceinline__ void dma_piece_at(const uint8_t* addr, uint32_t dst) {
    const uint32_t d = __builtin_amdgcn_readfirstlane(dst);
    uint32_t keep;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off\n\ts_mov_b32 m0, %0"
                 : "=&s"(keep) : "v"(addr), "s"(d) : "memory");
}
__device__ __forceinline__ void dma_piece_once(uint32_t voff, const uint8_t* base, uint32_t dst) {      // data read once: not kept in the caches
    const uint32_t d = __builtin_amdgcn_readfirstlane(dst);
    uint32_t keep;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %2\n\ts_nop 2\n\tglobal_load_lds_dwordx4 %1, %3 nt\n\ts_mov_b32 m0, %0"
                 : "=&s"(keep) : "v"(voff), "s"(d), "s"(base) : "memory");
}
// one scale per lane (a byte, or a float32) into the dwords behind LDS dst
template <int KIND>
__device__ __forceinline__ void dma_scale(uint32_t voff, const uint8_t* base, uint32_t dst) {
    const uint32_t d = __builtin_amdgcn_readfirstlane(dst);
    uint32_t keep;
    if constexpr (KIND == 0)
        asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %2\n\ts_nop 2\n\tglobal_load_lds_ubyte %1, %3\n\ts_mov_b32 m0, %0"
                     : "=&s"(keep) : "v"(voff), "s"(d), "s"(base) : "memory");
    else
        asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %2\n\ts_nop 2\n\tglobal_load_lds_dword %1, %3\n\ts_mov_b32 m0, %0"
                     : "=&s"(keep) : "v"(voff), "s"(d), "s"(base) : "memory");
}
__device__ __forceinline__ uint32_t lds_addr(const void* p) { return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void*)p; }

__device__ __forceinline__ v8i frag(const uint8_t* lo, const uint8_t* hi) {
    const v4i a = *reinterpret_cast<const v4i*>(lo), b = *reinterpret_cast<const v4i*>(hi);
    return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
}
// 16 x 16 x 128 product of two E4M3 fragments: lane l holds 32 k-values of row l & 15 (the same 32 of both operands); E8M0 scales per lane
__device__ __forceinline__ v4f mma_scaled(const v8i& a, const v8i& b, v4f c, uint32_t sa, uint32_t sb) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 0, 0, 0, (int)sa, 0, (int)sb);
}
__device__ __forceinline__ v4f mma_plain(const v8i& a, const v8i& b, v4f c) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 0, 0, 0, 0, 0, 0);          // (zero scale operands: the unscaled instruction)
}

// the EXACT product: the same fragments as 4 x 8 bf16 values, 4 x v_mfma_f32_16x16x32_bf16
using bf8 = __attribute__((ext_vector_type(8))) __bf16;
using bf2 = __attribute__((ext_vector_type(2))) __bf16;
__device__ __forceinline__ bf8 to_bf16(int lo, int hi) {
    const bf2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((uint32_t)lo, 1.f, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((uint32_t)lo, 1.f, true);
    const bf2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((uint32_t)hi, 1.f, false), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((uint32_t)hi, 1.f, true);
    return bf8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
__device__ __forceinline__ float scale_value(uint32_t v, int kind) { return kind == 0 ? e8m0_value(v) : __uint_as_float(v); }

// Two scales may multiply out of float32's range though sx sw d does not leave it (sx = 2^70, sw = 2^60, d = 2^-18; or d = 0).
// Float32 scales in the tile kernel: their powers of two ride in the instruction as E8M0 codes (it takes any two, measured), and what multiplies the
// sum is the product of the rests, in [1, 4).  Scalings by powers of two: the same bits as d (sx sw) where that is an ordinary number.  (A tile of 16 rows of w has
// one scale there: the lane's operand row and its result columns share it.)
__device__ __forceinline__ void split_scale(float s, uint32_t& code, float& rest) {
    code = min(max((__float_as_uint(s) >> 23) & 255u, 1u), 254u);
    rest = __builtin_ldexpf(s, 127 - (int)code);                       // (a denormal keeps its bits below 1; 0, infinity and NaN stay)
}
// The EXACT product has no scale operands, and in the kernel for few rows 16 rows of w may have two scales: sx * sw first while it is a normal number, else d takes the smaller one first -- that overflows only where the
// result does, and bits it loses, below 2^-149, are bits that x or w times its scale could not hold either.
struct ScalePair {
    float first, second;                                               // (1, sx sw), or (the smaller, the larger)
    __device__ __forceinline__ ScalePair(float sx, float sw) {
        const float s = sx * sw;
        const bool x_less = __builtin_fabsf(sx) < __builtin_fabsf(sw), plain = __builtin_fabsf(s) >= 0x1p-126f && __builtin_fabsf(s) < __builtin_inff();
        first = plain ? 1.f : x_less ? sx : sw;
        second = plain ? s : x_less ? sw : sx;
    }
    __device__ __forceinline__ float add(float d, float acc) const { return __builtin_fmaf(d * first, second, acc); }
};
// all 16 products of these scales are normal numbers, in every lane (NaN: whichever way, the sum becomes NaN)
__device__ __forceinline__ bool all_plain(const float* sx, const float* sw) {
    float hx = 0.f, hw = 0.f, lx = __builtin_inff(), lw = __builtin_inff();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        hx = fmaxf(hx, __builtin_fabsf(sx[i])), lx = fminf(lx, __builtin_fabsf(sx[i]));
        hw = fmaxf(hw, __builtin_fabsf(sw[i])), lw = fminf(lw, __builtin_fabsf(sw[i]));
    }
    return __all(hx * hw < __builtin_inff() && lx * lw >= 0x1p-126f);
}

// __expf rounds x log2(e) before the power: its error grows to |x| 2^-24 (5e-6 at 88), far inside the rounding of an 8- or 16-bit result.  A float32 result (FULL) gets
// e^x = 2^n 2^f with f = x log2(e) - n from two fused operations (log2(e) in two parts): within 2^-22 for every x, of a negative argument so that it cannot overflow.
// (expf would do, but this file is compiled with -ffp-contract=fast, which fuses expf's own reduction apart: 2.6e-6 at 80.)
__device__ __forceinline__ float exp_below_0(float x) {
    x = fmaxf(x, -150.f);                                              // (2^-216: 0)
    const float n = __builtin_rintf(x * 0x1.715476p+0f), f = __builtin_fmaf(x, 0x1.4ae0cp-26f, __builtin_fmaf(x, 0x1.715476p+0f, -n));
    return __builtin_ldexpf(__builtin_amdgcn_exp2f(f), (int)n);
}
template <bool FULL>
__device__ __forceinline__ float silu(float x) {
    if constexpr (FULL) {
        const float e = exp_below_0(-__builtin_fabsf(x));
        return x * ((x < 0.f ? e : 1.f) / (1.f + e));
    } else {
        return x / (1.f + __expf(-x));
    }
}

// ---- epilogue: 4 consecutive columns n .. n + 3 of row m ------------------------------------------------------------------------------------
template <int DT>
__device__ __forceinline__ void finish4(const GemmArgs& a, float* v, int m, int n, int ncols) {
    const int64_t o = (int64_t)m * a.ldo + n, r = (int64_t)m * a.ldr + n;
    if (a.vec && n + 3 < ncols) {
        if (a.bias) {
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] += DT == 2 ? ((const float*)a.bias)[n + i] : fp_to_f32<DT>(((const uint16_t*)a.bias)[n + i]);
        }
        if constexpr (DT == 2) {
            if (a.res) {
                const float4 t = *reinterpret_cast<const float4*>((const float*)a.res + r);
                v[0] += t.x; v[1] += t.y; v[2] += t.z; v[3] += t.w;
            }
            *reinterpret_cast<float4*>((float*)a.out + o) = make_float4(v[0], v[1], v[2], v[3]);
        } else {
            if (a.res) {
                const uint2 t = *reinterpret_cast<const uint2*>((const uint16_t*)a.res + r);
                v[0] += fp_to_f32<DT>((uint16_t)(t.x & 0xffffu)); v[1] += fp_to_f32<DT>((uint16_t)(t.x >> 16));
                v[2] += fp_to_f32<DT>((uint16_t)(t.y & 0xffffu)); v[3] += fp_to_f32<DT>((uint16_t)(t.y >> 16));
            }
            *reinterpret_cast<uint2*>((uint16_t*)a.out + o) = make_uint2(fp_pack2<DT>(v[0], v[1]), fp_pack2<DT>(v[2], v[3]));
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (n + i >= ncols) break;
        float t = v[i];
        if constexpr (DT == 2) {
            if (a.bias) t += ((const float*)a.bias)[n + i];
            if (a.res) t += ((const float*)a.res)[r + i];
            ((float*)a.out)[o + i] = t;
        } else {
            if (a.bias) t += fp_to_f32<DT>(((const uint16_t*)a.bias)[n + i]);
            if (a.res) t += fp_to_f32<DT>(((const uint16_t*)a.res)[r + i]);
            ((uint16_t*)a.out)[o + i] = (uint16_t)(fp_pack2<DT>(t, t) & 0xffffu);
        }
    }
}
__device__ __forceinline__ void finish4(const GemmArgs& a, float* v, int m, int n, int ncols) {
    if (a.out_type == 0) finish4<0>(a, v, m, n, ncols);
    else if (a.out_type == 1) finish4<1>(a, v, m, n, ncols);
    else finish4<2>(a, v, m, n, ncols);
}

// K tiles of a slice in the order they are worked off: a ragged last tile comes FIRST, so that only the prologue's loads know about the end of K
struct KOrder {
    int n, kb, first;
    __device__ __forceinline__ KOrder(int b, int e, bool ragged_end) : n(e - b), kb(b), first(ragged_end ? e - 1 : -1) {}
    __device__ __forceinline__ int tile(int p) const { return first < 0 ? kb + p : (p == 0 ? first : kb + p - 1); }
};

// ================================================================================================================================
// Tile kernel: BM x BN x 128 per workgroup of 4 waves (64 x 64 each), two K tiles in LDS, two workgroups per CU.
//   * A K tile is one scale group: 128 B per row, the operand of ONE v_mfma_*_16x16x128.  Rows are XOR-swizzled in 16-byte chunks
//     (chunk ^= row & 7, applied to the DMA's source address), so the two ds_read_b128 of a fragment are conflict-free.
//   * w is the first operand: a lane owns 4 consecutive columns of one row of the result.
//   * E8M0: the scales ride in the instruction.  float32 scales, and EXACT: each K tile's product is multiplied by sx * sw and added (split_scale, ScalePair).
// SwiGLU: the tile holds BN / 2 columns of the result; its w rows alternate 16 gate and 16 up rows, so that one lane holds both.
// ================================================================================================================================
template <int KIND, bool SWI, bool EXACT, int BM, int BN>
__global__ void __launch_bounds__(256, 2)
k_fp8_gemm_tile(const GemmArgs a) {
    constexpr int WC = BN / 64, PA = BM / 32, PW = BN / 32;          // waves along N; DMA pieces per wave
    static_assert((BM / 64) * WC == 4, "four waves");
    constexpr int STAGE = (BM + BN) * FP8_G, OUT_N = SWI ? BN / 2 : BN, ESZ = KIND == 0 ? 1 : 4;
    extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wr = wave / WC, wc = wave % WC, fi = lane & 15, fg = lane >> 4;
    const int ncols = SWI ? a.I : a.N;

    // tile of this workgroup: slices outermost; inside, consecutive workgroups of an XCD share rows of x and w (8 row tiles per group)
    const int nt = a.tiles_m * a.tiles_n;
    const int slice = __builtin_amdgcn_readfirstlane((int)blockIdx.x / nt);
    int t = (int)blockIdx.x - slice * nt;
    {
        const int xcd = t & 7, q = nt >> 3, r = nt & 7;
        t = (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + (t >> 3);
    }
    constexpr int GM = 8;
    const int g0 = t / (GM * a.tiles_n) * GM, gs = min(GM, a.tiles_m - g0), ti = t % (GM * a.tiles_n);
    const int row0 = __builtin_amdgcn_readfirstlane((g0 + ti % gs) * BM), col0 = __builtin_amdgcn_readfirstlane(ti / gs * OUT_N);
    const int kb0 = slice * a.KB / a.splits, kb1 = (slice + 1) * a.KB / a.splits;
    const KOrder order(kb0, kb1, kb1 == a.KB && a.K % FP8_G);

    // w row behind row r of the LDS tile
    auto wrow = [&](int r) {
        if constexpr (SWI) {
            const int c = min(col0 + (r >> 6) * 32 + ((r >> 5) & 1) * 16 + (r & 15), a.I - 1);
            return (r & 16) ? a.I + c : c;
        } else {
            return min(col0 + r, a.N - 1);
        }
    };
    const uint8_t* xbase = a.x + (int64_t)row0 * a.ldx;
    const uint8_t* wbase = a.w + (SWI ? 0 : (int64_t)col0 * a.ldw);
    const int wsub = SWI ? 0 : col0;
    uint32_t xo[PA], wo[PW];
#pragma unroll
    for (int p = 0; p < PA; ++p) {
        const int r = (wave + p * 4) * 8 + (lane >> 3);
        xo[p] = (uint32_t)((int64_t)(min(row0 + r, a.M - 1) - row0) * a.ldx + ((lane & 7) ^ (r & 7)) * 16);
    }
#pragma unroll
    for (int p = 0; p < PW; ++p) {
        const int r = (wave + p * 4) * 8 + (lane >> 3);
        wo[p] = (uint32_t)((int64_t)(wrow(r) - wsub) * a.ldw + ((lane & 7) ^ (r & 7)) * 16);
    }
    const uint32_t lds0 = lds_addr(smem);
    auto stage = [&](int p) {
        const int kt = order.tile(p);
        const uint32_t dst = lds0 + (uint32_t)(p & 1) * STAGE + (uint32_t)wave * 1024u;
        const int64_t k0 = (int64_t)kt * FP8_G;
        if (kt * FP8_G + FP8_G > a.K) {                               // the ragged tile: chunks behind K read zeros
            const int chunk = (lane & 7) ^ ((lane >> 3) & 7);
            const bool in = kt * FP8_G + chunk * 16 < a.K;
#pragma unroll
            for (int q = 0; q < PA; ++q) dma_piece_at(in ? xbase + k0 + xo[q] : (const uint8_t*)&g_zero16, dst + (uint32_t)q * 4096u);
#pragma unroll
            for (int q = 0; q < PW; ++q) dma_piece_at(in ? wbase + k0 + wo[q] : (const uint8_t*)&g_zero16, dst + BM * FP8_G + (uint32_t)q * 4096u);
        } else {
#pragma unroll
            for (int q = 0; q < PA; ++q) dma_piece(xo[q], xbase + k0, dst + (uint32_t)q * 4096u);
#pragma unroll
            for (int q = 0; q < PW; ++q) dma_piece(wo[q], wbase + k0, dst + BM * FP8_G + (uint32_t)q * 4096u);
        }
    };

    // Scales of this lane's rows: x row per i, w row (E8M0: of the lane's operand row; float32: of its 4 result columns, one block) per j.  They come through LDS, a
    // DMA per wave for 64 of the 256 rows: a load per use (8 per wave, 16 rows each) kept the address pipe busier than the operands (823 x 9216 x 3072 44.5 us and
    // 51.9 with float32 scales, now 34.4 - 37.4 and 41.3; 1024 x 3072 x 8192 72.4, now 57.2).  Loads two K tiles ahead, behind a second barrier, gained nothing (39.6).
    // SwiGLU has no LDS left for them (two workgroups fill it) and loads each into its register.
    constexpr bool LDS_SCALES = !SWI;
    const uint8_t* sxb = (const uint8_t*)a.sx + (int64_t)row0 * a.ldsx * ESZ;
    uint32_t sxo[4], swo[4];
    if constexpr (LDS_SCALES) {
        const int r = (wave & 1) * 64 + lane;                          // waves 0, 1: x rows, 2, 3: w rows
        sxo[0] = (uint32_t)(wave < 2 ? min(r, a.M - 1 - row0) * (int)a.ldsx * ESZ : (wrow(r) >> 7) * (int)a.ldsw * ESZ);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            sxo[i] = (uint32_t)(min(wr * 64 + i * 16 + fi, a.M - 1 - row0) * (int)a.ldsx * ESZ);
            swo[i] = (uint32_t)((wrow(wc * 64 + i * 16 + fi) >> 7) * (int)a.ldsw * ESZ);
        }
    }
    uint32_t sx[4], sw[4], nsx[4], nsw[4];
    auto load_scales = [&](int p) {
        const int kt = order.tile(p);
        const uint8_t *px = sxb + kt * ESZ, *pw = (const uint8_t*)a.sw + kt * ESZ;
        if constexpr (LDS_SCALES) {
            dma_scale<KIND>(sxo[0], wave < 2 ? px : pw, lds0 + 2 * STAGE + (uint32_t)(p & 1) * 1024u + (uint32_t)wave * 256u);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                nsx[i] = KIND == 0 ? (uint32_t)px[sxo[i]] : *(const uint32_t*)(px + sxo[i]);
                nsw[i] = KIND == 0 ? (uint32_t)pw[swo[i]] : *(const uint32_t*)(pw + swo[i]);
            }
        }
    };

    v4f acc[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = v4f{0.f, 0.f, 0.f, 0.f};

    if (order.n > 0) {
        load_scales(0);
        stage(0);
    }
    constexpr bool CARE = EXACT || KIND == 1;                         // scales as numbers: their products may not be
    float fx[4], fw[4];
    v8i af[4], bf[4];                                                 // (EXACT reads its fragments by halves)
    auto arrive = [&](int p) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();                                 // tile p has landed everywhere, tile p - 1 has been read everywhere
        if constexpr (!LDS_SCALES) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                sx[i] = nsx[i];
                sw[i] = nsw[i];
                asm volatile("" : "+v"(sx[i]), "+v"(sw[i]));          // the compiler's own wait for the scales belongs HERE, not behind the next DMA
            }
        }
        if (p + 1 < order.n) {
            load_scales(p + 1);
            stage(p + 1);
        }
        if constexpr (LDS_SCALES) {
            const uint32_t* ls = reinterpret_cast<const uint32_t*>(smem + 2 * STAGE + (p & 1) * 1024);
#pragma unroll
            for (int i = 0; i < 4; ++i) sx[i] = ls[wr * 64 + i * 16 + fi], sw[i] = ls[128 + wc * 64 + i * 16 + fi];
        }
    };
    auto fetch = [&](int p) {
        if constexpr (!EXACT) {
            const uint8_t* la = smem + (p & 1) * STAGE;
            const uint8_t* lb = la + BM * FP8_G;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int rb = wc * 64 + i * 16 + fi, ra = wr * 64 + i * 16 + fi, s = fi & 7;
                bf[i] = frag(lb + rb * FP8_G + ((fg ^ s) << 4), lb + rb * FP8_G + (((fg + 4) ^ s) << 4));
                af[i] = frag(la + ra * FP8_G + ((fg ^ s) << 4), la + ra * FP8_G + (((fg + 4) ^ s) << 4));
            }
        }
        if constexpr (CARE) {
#pragma unroll
            for (int i = 0; i < 4; ++i) fx[i] = scale_value(sx[i], KIND), fw[i] = scale_value(sw[i], KIND);
        }
    };
    auto multiply = [&](int p, auto plain) {                          // plain: sx * sw is a normal number for all pairs of the wave
        if constexpr (EXACT) {
            const uint8_t* la = smem + (p & 1) * STAGE;
            const uint8_t* lb = la + BM * FP8_G;
#pragma unroll
            for (int jh = 0; jh < 4; jh += 2) {                       // two of the wave's four column tiles at a time: the sums of a K tile are 32 registers
                v4f d[4][2];
#pragma unroll
                for (int i = 0; i < 4; ++i) d[i][0] = d[i][1] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    __builtin_amdgcn_sched_barrier(0);                // (loads and conversions of later steps are not pulled up: registers)
                    v4i ax[4], bx[2];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        if (i < 2) bx[i] = *reinterpret_cast<const v4i*>(lb + (wc * 64 + (jh + i) * 16 + fi) * FP8_G + (((fg + 4 * h) ^ (fi & 7)) << 4));
                        ax[i] = *reinterpret_cast<const v4i*>(la + (wr * 64 + i * 16 + fi) * FP8_G + (((fg + 4 * h) ^ (fi & 7)) << 4));
                    }
#pragma unroll
                    for (int g = 0; g < 4; g += 2) {
                        const bf8 b0 = to_bf16(bx[0][g], bx[0][g + 1]), b1 = to_bf16(bx[1][g], bx[1][g + 1]);
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const bf8 ah = to_bf16(ax[i][g], ax[i][g + 1]);
                            d[i][0] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b0, ah, d[i][0], 0, 0, 0);
                            d[i][1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b1, ah, d[i][1], 0, 0, 0);
                        }
                    }
                }
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const ScalePair s(fx[i], fw[jh + j]);
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            acc[i][jh + j][r] = plain ? __builtin_fmaf(d[i][j][r], fx[i] * fw[jh + j], acc[i][jh + j][r]) : s.add(d[i][j][r], acc[i][jh + j][r]);
                    }
            }
        } else {
            if constexpr (KIND == 1 && !plain) {                      // the codes to sx, sw, the rests to fx, fw
#pragma unroll
                for (int i = 0; i < 4; ++i) split_scale(fx[i], sx[i], fx[i]), split_scale(fw[i], sw[i], fw[i]);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if constexpr (KIND == 0) {
                        acc[i][j] = mma_scaled(bf[j], af[i], acc[i][j], sw[j], sx[i]);
                    } else {
                        const v4f zero = v4f{0.f, 0.f, 0.f, 0.f}, d = plain ? mma_plain(bf[j], af[i], zero) : mma_scaled(bf[j], af[i], zero, sw[j], sx[i]);
                        const float s = fx[i] * fw[j];
#pragma unroll
                        for (int r = 0; r < 4; ++r) acc[i][j][r] = __builtin_fmaf(d[r], s, acc[i][j][r]);
                    }
                }
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    };
    // Products of scales that are not plain are rare (zeros beside small weights make them, 2^-126 * sw): the first one sends the wave to a second loop that takes care of
    // them.  Both loops meet the workgroup's other waves at one barrier per K tile.  (6568 x 3072 x 8192, float32 scales: 207 us, without the question 197, in the careful
    // form for every K tile 216; both forms in one loop spilled.)
    int p = 0;
    if constexpr (CARE) {
        bool plain = true;
        while (p < order.n) {
            arrive(p);
            fetch(p);
            plain = all_plain(fx, fw);
            if (!plain) break;
            multiply(p++, std::true_type{});
        }
        while (!plain) {
            fetch(p);
            multiply(p++, std::false_type{});
            if (p == order.n) break;
            arrive(p);
        }
    } else {
        for (; p < order.n; ++p) {
            arrive(p);
            fetch(p);
            multiply(p, std::true_type{});
        }
    }

    // ---- epilogue: lane holds row row0 + wr * 64 + i * 16 + fi, operand columns wc * 64 + j * 16 + fg * 4 .. + 3
    if (a.splits > 1) {                                               // raw float32 sums, column = row of w; k_fp8_gemm_finish adds the slices in order
        float* ws = a.ws + (int64_t)slice * a.M * a.ldws;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int m = row0 + wr * 64 + i * 16 + fi;
            if (m >= a.M) continue;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int c = SWI ? col0 + wc * 32 + (j >> 1) * 16 + fg * 4 : col0 + wc * 64 + j * 16 + fg * 4;
                const int64_t o = (int64_t)m * a.ldws + (SWI && (j & 1) ? a.ldws / 2 : 0) + c;
                if (c < ncols) *reinterpret_cast<v4f*>(ws + o) = acc[i][j];      // (rows of ws are padded to 8 columns)
            }
        }
        return;
    }
    if constexpr (!SWI) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int m = row0 + wr * 64 + i * 16 + fi;
            if (m >= a.M) continue;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float v[4] = {acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3]};
                finish4(a, v, m, col0 + wc * 64 + j * 16 + fg * 4, ncols);
            }
        }
    } else {
        float v[4][8];
        float* amax = reinterpret_cast<float*>(smem);                 // [4 waves][64 rows]
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int r = 0; r < 4; ++r) v[i][j * 4 + r] = acc[i][2 * j + 1][r] * silu<EXACT>(acc[i][2 * j][r]);
        if (a.out_type != 3) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int m = row0 + wr * 64 + i * 16 + fi;
                if (m >= a.M) continue;
#pragma unroll
                for (int j = 0; j < 2; ++j) finish4(a, &v[i][j * 4], m, col0 + wc * 32 + j * 16 + fg * 4, ncols);
            }
            return;
        }
        // the tile's 128 columns are one group of the result: its maximum over 4 lanes, then over the 4 waves
        static_assert(!SWI || (BM == 64 && BN == 256), "one group of 128 columns per workgroup");
        __builtin_amdgcn_s_barrier();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float x = 0.f;
#pragma unroll
            for (int r = 0; r < 8; ++r)
                if (col0 + wc * 32 + (r >> 2) * 16 + fg * 4 < ncols) x = fmaxf(x, fp8_finite_abs(v[i][r]));       // (I % 16 == 0 here)
            x = fmaxf(x, __shfl_xor(x, 16, 64));
            x = fmaxf(x, __shfl_xor(x, 32, 64));
            if (fg == 0) amax[wc * 64 + i * 16 + fi] = x;
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int lr = i * 16 + fi, m = row0 + lr;
            const float x = fmaxf(fmaxf(amax[lr], amax[64 + lr]), fmaxf(amax[128 + lr], amax[192 + lr]));
            uint32_t o[2], code;
            float s;
            fp8_quantize_pack<8>(v[i], x, KIND, o, code, s);
            if (m >= a.M) continue;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int c = col0 + wc * 32 + j * 16 + fg * 4;
                if (c < ncols) *reinterpret_cast<uint32_t*>((uint8_t*)a.out + (int64_t)m * a.ldo + c) = o[j];
            }
            if (wc == 0 && fg == 0) {
                if (KIND == 0) ((uint8_t*)a.out_scale)[(int64_t)m * a.ldos + col0 / FP8_G] = (uint8_t)code;
                else ((float*)a.out_scale)[(int64_t)m * a.ldos + col0 / FP8_G] = s;
            }
        }
    }
}

// ================================================================================================================================
// Large products, E8M0 scales, results of 8 or 16 bits: 256 x 256 x 128 per workgroup of FOUR waves, 128 x 128 each, one wave per SIMD.
//   * 64 products of 16x16x128 per wave and K tile on 256 accumulators, out of 16 fragments that stay in registers; LDS is read 128 KiB per K tile.  With
//     128 x 64 per wave (eight waves) it was 192, the two waves of a SIMD met at the barriers, and 8192^3 took 538 us instead of 440.
//   * Two barriers per K tile: behind the first every wave has read tile p and its buffer takes the DMA of tile p + 2; behind the second tile p + 1
//     has landed.
//   * 16x16x128 products: the matrix pipe alone runs 4.3 PFLOP/s on them and 3.6 - 3.9 on 32x32x64 (power), measured on random data.
//   * Rows are permuted inside blocks of 64: row 4 f + c of a block is row f of tile c, for x and w alike.  A lane then holds 16 NEIGHBOURING columns of a row
//     (it stores them with no trip through LDS), and the scales of its rows in four tiles are neighbours: they come by DMA too, a dword per row, are
//     read as one 16-byte piece, and packed into a register of which the instruction picks the byte.
//   * What bounds it: power, then waits.  8192^3 402 - 440 us, 2.5 - 2.7 PFLOP/s; the matrix pipe is busy 70 % of the cycles there, at 1.8 GHz (6568 x 9216 x 3072, 24 K tiles and a round of 168 tiles at the end: 53 %); 16 % are waits for loads and at
//     the barriers; with a quarter of the CUs at work a K tile takes 0.97 us instead of 1.7.  One workgroup
//     for several output tiles, loading the next one's operands while it stores, gained nothing (172.7 and 171.8 us for 6568 x 9216 x 3072).
// DT: 0 bf16, 1 fp16, 3 E4M3 + scale (SwiGLU).  Rows of out and residual allow 16-byte accesses, columns come in eights (the host's choice of this kernel).
// ================================================================================================================================
// 1 KiB (16 bytes per lane from base + off), or one byte per lane into a dword, to LDS dst + IMM; base and dst in scalar registers.  (m0 is not kept: nothing else
// in the kernel below uses it.  2 wait states of its own: the bases are made, by v_readfirstlane, a dozen products or an s_nop 4 ahead -- and none is spilled.  With 5 here, 18
// times per K tile, 6568 x 9216 x 3072 took 163.5 us instead of 160.)
template <int IMM>
__device__ __forceinline__ void dma_to(uint32_t off, const uint8_t* base, uint32_t dst) {
    asm volatile("s_add_u32 m0, %1, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %2" ::"v"(off), "s"(dst), "s"(base), "n"(IMM) : "memory", "scc");
}
template <int IMM>
__device__ __forceinline__ void dma_byte_to(uint32_t off, const uint8_t* base, uint32_t dst) {
    asm volatile("s_add_u32 m0, %1, %3\n\ts_nop 0\n\tglobal_load_lds_ubyte %0, %2" ::"v"(off), "s"(dst), "s"(base), "n"(IMM) : "memory", "scc");
}

template <class F, int... I>
__device__ __forceinline__ void each(F&& f, std::integer_sequence<int, I...>) { (f(std::integral_constant<int, I>{}), ...); }
template <int N, class F>
__device__ __forceinline__ void each(F&& f) { each(f, std::make_integer_sequence<int, N>{}); }

template <bool SWI, int DT>
__global__ void __launch_bounds__(256, 1)
k_fp8_gemm_big(const GemmArgs a) {
    constexpr int BM = 256, BN = 256, BUF = (BM + BN) * FP8_G, OUT_N = SWI ? BN / 2 : BN;
    extern __shared__ __attribute__((aligned(16))) uint8_t smem[];     // [2][x 256 x 128 | w 256 x 128], scales [2][x 256 | w 256] dwords
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave >> 1, wn = wave & 1, fi = lane & 15, fg = lane >> 4, lr = lane >> 3;
    const int ncols = SWI ? a.I : a.N, nk = a.KB;
    const int nwg = a.tiles_m * a.tiles_n;
    int wg = blockIdx.x;
    {
        const int xcd = wg & 7, q = nwg >> 3, r = nwg & 7;
        wg = (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + (wg >> 3);
    }
    constexpr int GM = 4;                                              // 4 row tiles share the w tiles of an XCD: 4 + 8 operand panels for its 32 workgroups
    const int g0 = wg / (GM * a.tiles_n) * GM, gs = min(GM, a.tiles_m - g0), ti = wg % (GM * a.tiles_n);
    const int row0 = __builtin_amdgcn_readfirstlane((g0 + ti % gs) * BM), col0 = __builtin_amdgcn_readfirstlane(ti / gs * OUT_N);

    // DMA: piece q of a wave is LDS rows (wave + 4 q) * 8 .. + 7 of an operand tile; offsets from the tile's origin, rows behind the end read the last
    // one again (their results are not stored).  Chunk swizzle ^ (LDS row & 7).
    const int chunk = (lane & 7) ^ lr;
    const uint8_t* xbase = a.x + (int64_t)row0 * a.ldx;
    const uint8_t* wbase = a.w + (SWI ? 0 : (int64_t)col0 * a.ldw);
    uint32_t xo[8], wo[8];
#pragma unroll
    for (int q = 0; q < 8; ++q) {
        const int r = (q >> 1) * 64 + ((wave & 1) * 8 + lr) * 4 + (wave >> 1) + 2 * (q & 1);
        xo[q] = (uint32_t)min(r, a.M - 1 - row0) * (uint32_t)a.ldx + (chunk << 4);
        if constexpr (SWI) {                                           // (column tiles 0, 1 of a block of 64 gate, 2, 3 up)
            const int c = min(col0 + (q >> 1) * 32 + ((wave & 1) * 8 + lr) * 2 + (wave >> 1), a.I - 1);
            wo[q] = (uint32_t)((q & 1) ? a.I + c : c) * (uint32_t)a.ldw + (chunk << 4);
        } else {
            wo[q] = (uint32_t)min(r, a.N - 1 - col0) * (uint32_t)a.ldw + (chunk << 4);
        }
    }
    // scales: wave v loads those of rows 64 v + lane of x and of w
    const uint8_t* sxb = (const uint8_t*)a.sx + (int64_t)row0 * a.ldsx;
    const uint32_t sxo = (uint32_t)(min(wave * 64 + lane, a.M - 1 - row0) * (int)a.ldsx);
    const int sc = min(col0 + (SWI ? wave * 32 + (lane >> 2) * 2 + (lane & 1) : wave * 64 + lane), ncols - 1);
    const uint32_t swo = (uint32_t)(((SWI && (lane & 2) ? a.I + sc : sc) >> 7) * (int)a.ldsw);
    // Position p of the K loop is K tile p; where K ends inside a tile, that tile comes FIRST (position 0) and only the prologue knows about the end of K
    const int ragged = __builtin_amdgcn_readfirstlane(a.K % FP8_G ? 1 : 0);
    const uint32_t lds0 = __builtin_amdgcn_readfirstlane(lds_addr(smem) + (uint32_t)wave * 1024u);
    struct From { const uint8_t *x, *w, *sx, *sw; uint32_t d, ds; };
    auto from = [&](int p, int buf) {                                  // position p to buffer buf (all in scalar registers)
        const int k = __builtin_amdgcn_readfirstlane(p < ragged ? nk - 1 : p - ragged);
        auto scalar = [](const uint8_t* p) {
            const uint64_t u = (uint64_t)p;
            return (const uint8_t*)(((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(u >> 32)) << 32) | (uint32_t)__builtin_amdgcn_readfirstlane((int)u));
        };
        return From{scalar(xbase + (int64_t)k * FP8_G), scalar(wbase + (int64_t)k * FP8_G), scalar(sxb + k), scalar((const uint8_t*)a.sw + k),
                    (uint32_t)__builtin_amdgcn_readfirstlane((int)(lds0 + (uint32_t)buf * BUF)),
                    (uint32_t)__builtin_amdgcn_readfirstlane((int)(lds_addr(smem) + (uint32_t)wave * 256u + 2u * BUF + (uint32_t)buf * 2048u))};
    };
    auto dma = [&](auto q, const From& f) {                            // piece q of 18: 8 of x, 8 of w, the scales of x and of w
        if constexpr (q < 8) dma_to<q * 4096>(xo[q], f.x, f.d);
        else if constexpr (q < 16) dma_to<q * 4096>(wo[q - 8], f.w, f.d);
        else if constexpr (q == 16) dma_byte_to<0>(sxo, f.sx, f.ds);
        else dma_byte_to<1024>(swo, f.sw, f.ds);
    };
    // the scales of the lane's four rows in block c of the wave's x (c = 0, 1) or w (2, 3)
    auto scales4 = [&](int c, int p) { return *reinterpret_cast<const v4i*>(smem + 2 * BUF + (p & 1) * 2048 + (c < 2 ? wm * 2 + c : 4 + wn * 2 + c - 2) * 256 + fi * 16); };
    auto pack = [](const v4i& v) { return (uint32_t)(v[0] | (v[1] << 8) | (v[2] << 16) | (v[3] << 24)); };

    v4f acc[8][8];
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[i][j] = v4f{0.f, 0.f, 0.f, 0.f};
    v8i af[8], bf[8];
    uint32_t sx[2], sw[2];
    auto rd = [&](const uint8_t* t) { return frag(t + fi * FP8_G + ((fg ^ (fi & 7)) << 4), t + fi * FP8_G + (((fg + 4) ^ (fi & 7)) << 4)); };
    auto xt = [&](int p, int i) { return smem + (p & 1) * BUF + (wm * 128 + i * 16) * FP8_G; };
    auto wt = [&](int p, int j) { return smem + (p & 1) * BUF + (BM + wn * 128 + j * 16) * FP8_G; };
    // One K tile: 64 products, x tiles 0 - 3 and then 4 - 7 against the w tiles in turn: in this order the fragments come free one after the other, and each is
    // read anew (for the next tile, x tiles 4 - 7 for this one) some 30 products ahead of its use.  Reads and loads are spread evenly: per product (32
    // cycles) the four waves get one 16-byte read each out of LDS and half a piece out of the caches, so a run of either would stall the products (with
    // the loads behind one another the kernel took 8 - 10 % longer).  (The last two tiles load the last one again, for nobody: no branch in the loop.)
    constexpr int FREE = 13, LANDED = 32;
    v4i raw;
    auto tile = [&](int p) {
        const From f = from(min(p + 2, nk - 1), p & 1);
        each<64>([&](auto s_) {
            constexpr int s = s_, j = (s >> 2) & 7, i = (s >> 5) * 4 + (s & 3);
            acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(bf[j], af[i], acc[i][j], 0, 0, j & 3, (int)sw[j >> 2], i & 3, (int)sx[i >> 2]);
            if constexpr (s == 0) bf[7] = rd(wt(p, 7));
            if constexpr (s == 2) raw = scales4(1, p);
            if constexpr (s == 4 || s == 6 || s == 8 || s == 10) af[2 + s / 2] = rd(xt(p, 2 + s / 2));
            if constexpr (s == 6) sx[1] = pack(raw);
            if constexpr (s == FREE) {                                 // every wave has read tile p
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                __builtin_amdgcn_s_barrier();
            }
            each<18>([&](auto q) {
                if constexpr (s == FREE + q * 3 - q / 12) dma(q, f);
            });
            if constexpr (s == LANDED) {                               // tile p + 1 has landed: all but the first loads of tile p + 2
                asm volatile("s_waitcnt vmcnt(%0)" ::"n"((LANDED - FREE) / 3 + 1) : "memory");
                __builtin_amdgcn_s_barrier();
            }
            if constexpr (s >= 33 && s < 41 && (s - 33) % 2 == 0) af[(s - 33) / 2] = rd(xt(p + 1, (s - 33) / 2));
            if constexpr (s == 42) raw = scales4(0, p + 1);
            each<7>([&](auto c) {
                if constexpr (s == 41 + c * 13 / 4 + (c > 4)) bf[c] = rd(wt(p + 1, c));
            });
            if constexpr (s == 46) sx[0] = pack(raw), raw = scales4(2, p + 1);
            if constexpr (s == 52) sw[0] = pack(raw), raw = scales4(3, p + 1);
            if constexpr (s == 63) sw[1] = pack(raw);
            __builtin_amdgcn_sched_barrier(0);
        });
    };

    // nk >= 2 (the host's choice of this kernel)
    const From f0 = from(0, 0), f1 = from(1, 1);
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_nop 4" ::: "memory");                              // the bases have reached the scalar registers
    __builtin_amdgcn_sched_barrier(0);
    if (ragged) {                                                      // the chunks behind K read zeros
        const bool in = (nk - 1) * FP8_G + chunk * 16 < a.K;
#pragma unroll
        for (int q = 0; q < 8; ++q) {
            dma_piece_at(in ? xbase + (int64_t)(nk - 1) * FP8_G + xo[q] : (const uint8_t*)&g_zero16, lds0 + (uint32_t)q * 4096u);
            dma_piece_at(in ? wbase + (int64_t)(nk - 1) * FP8_G + wo[q] : (const uint8_t*)&g_zero16, lds0 + (uint32_t)(BM * FP8_G) + (uint32_t)q * 4096u);
        }
    } else {
        each<16>([&](auto q) { dma(q, f0); });
    }
    dma(std::integral_constant<int, 16>{}, f0), dma(std::integral_constant<int, 17>{}, f0);
    each<18>([&](auto q) { dma(q, f1); });
    asm volatile("s_waitcnt vmcnt(18)" ::: "memory");
    __builtin_amdgcn_s_barrier();
#pragma unroll
    for (int c = 0; c < 7; ++c) bf[c] = rd(wt(0, c));
#pragma unroll
    for (int c = 0; c < 4; ++c) af[c] = rd(xt(0, c));
    sx[0] = pack(scales4(0, 0)), sw[0] = pack(scales4(2, 0)), sw[1] = pack(scales4(3, 0));
    int p = 0;
    do tile(p);
    while (++p < nk);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");                   // (no load into LDS outlives the wave)

    // ---- epilogue.  Lane: row (i >> 2) * 64 + 4 fi + (i & 3) of the wave's 128; of each block h of 64 w rows, columns 16 fg + 4 r + j (SwiGLU: 8 fg + 2 r + j)
    int elane = lane;
    asm volatile("" : "+v"(elane));                                   // (what follows from it is not worked out before the K loop and kept: registers)
    const int ef = elane & 15, eg = elane >> 4, mrow = wm * 128 + ef * 4;
    constexpr int NC = SWI ? 8 : 16, ND = DT == 3 ? 0 : DT;
    auto row_of = [&](int i) { return mrow + (i >> 2) * 64 + (i & 3); };
    auto col_of = [&](int h) { return col0 + (SWI ? (wn * 2 + h) * 32 + eg * 8 : wn * 128 + h * 64 + eg * 16); };
    auto keep = [&](int i, int h) {                                    // the sums stay where the products left them until here, row by row
#pragma unroll
        for (int c = 0; c < 4; ++c) asm volatile("" : "+a"(acc[i][h * 4 + c]));
    };
    if constexpr (DT == 3) {                                           // the tile's 128 columns are one group of the result
        __builtin_amdgcn_s_barrier();                                  // every wave has read its last fragments
        float* amax = reinterpret_cast<float*>(smem);                  // [2 waves][256 rows]
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            float x = 0.f;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                keep(i, h);
                float y = 0.f;
#pragma unroll
                for (int c = 0; c < 8; ++c) {
                    const float v = acc[i][h * 4 + 2 + (c & 1)][c >> 1] * silu<false>(acc[i][h * 4 + (c & 1)][c >> 1]);
                    acc[i][h * 4 + (c & 1)][c >> 1] = v;
                    y = fmaxf(y, fp8_finite_abs(v));
                }
                x = fmaxf(x, col_of(h) < ncols ? y : 0.f);             // (I % 16 == 0: all of the lane's columns or none)
            }
            x = fmaxf(x, __shfl_xor(x, 16, 64));
            x = fmaxf(x, __shfl_xor(x, 32, 64));
            if (eg == 0) amax[wn * 256 + row_of(i)] = x;
            __builtin_amdgcn_sched_barrier(0);
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int lrow = row_of(i), m = row0 + lrow;
            const float x = fmaxf(amax[lrow], amax[256 + lrow]);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float v[8];
#pragma unroll
                for (int c = 0; c < 8; ++c) v[c] = acc[i][h * 4 + (c & 1)][c >> 1];
                uint32_t o[2], code;
                float s;
                fp8_quantize_pack<8>(v, x, 0, o, code, s);
                if (m < a.M) {
                    if (col_of(h) < ncols) *reinterpret_cast<uint2*>((uint8_t*)a.out + (int64_t)m * a.ldo + col_of(h)) = make_uint2(o[0], o[1]);
                    if (h == 0 && wn == 0 && eg == 0) ((uint8_t*)a.out_scale)[(int64_t)m * a.ldos + col0 / FP8_G] = (uint8_t)code;
                }
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    } else {
        // Bias and residual are added whether they are there or not (zeros): only their loads are conditional -- branches around the sums would cost
        // copies of all 256.  Offsets from the tile's origin in 32 bits: one register per address.
        const uint8_t* rbase = (const uint8_t*)a.res + ((int64_t)row0 * a.ldr + col0) * 2;
        uint8_t* obase = (uint8_t*)a.out + ((int64_t)row0 * a.ldo + col0) * 2;
        auto half = [](const uint4& u, int c) {                        // 16-bit element c of 8
            const uint32_t w = (c >> 1) == 0 ? u.x : (c >> 1) == 1 ? u.y : (c >> 1) == 2 ? u.z : u.w;
            return fp_to_f32<ND>((uint16_t)(c & 1 ? w >> 16 : w & 0xffffu));
        };
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int n = col_of(h);
            const bool in0 = n < ncols, in1 = NC == 16 && n + 8 < ncols;
            const uint32_t on = (uint32_t)(n - col0) * 2u;
            uint4 bias[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
            if (!SWI && a.bias && in0) bias[0] = *reinterpret_cast<const uint4*>((const uint16_t*)a.bias + n);
            if (!SWI && a.bias && in1) bias[1] = *reinterpret_cast<const uint4*>((const uint16_t*)a.bias + n + 8);
            uint4 t[8][2];                                             // the residual: 16 loads requested together
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                t[i][0] = t[i][1] = make_uint4(0, 0, 0, 0);
                if (!SWI && a.res && row0 + row_of(i) < a.M) {
                    const uint8_t* r = rbase + ((uint32_t)row_of(i) * (uint32_t)a.ldr * 2u + on);
                    if (in0) t[i][0] = *reinterpret_cast<const uint4*>(r);
                    if (in1) t[i][1] = *reinterpret_cast<const uint4*>(r + 16);
                }
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                __builtin_amdgcn_sched_barrier(0);
                keep(i, h);
                float v[NC];
#pragma unroll
                for (int c = 0; c < NC; ++c) {
                    if constexpr (SWI) v[c] = acc[i][h * 4 + 2 + (c & 1)][c >> 1] * silu<false>(acc[i][h * 4 + (c & 1)][c >> 1]);
                    else v[c] = acc[i][h * 4 + (c & 3)][c >> 2] + half(bias[c >> 3], c & 7) + half(t[i][c >> 3], c & 7);
                }
                uint8_t* o = obase + ((uint32_t)row_of(i) * (uint32_t)a.ldo * 2u + on);
                const bool m_in = row0 + row_of(i) < a.M;
                if (m_in && in0) fp_store8<ND>(o, 0, v);
                if (m_in && in1) fp_store8<ND>(o, 8, v + NC - 8);
            }
        }
    }
}

// ================================================================================================================================
// Few rows (M <= 16 MT): the weights stream once.
//   * A workgroup owns R neighbouring rows of w (SwiGLU: R gate rows and the R up rows beside them), R chosen so that the grid is one or a few whole
//     workgroups per CU; its waves take the K blocks in turn (block b to wave b mod waves: side by side they read neighbouring 128 B of the same
//     rows).  A wave requests up to nb blocks before it waits, so that a CU has ~100 KB in flight: what bounds it is memory, then the launch.
//   * The blocks go to the wave's own corner of LDS by DMA, 8 rows x 128 B per instruction, not cached (nt): that pattern reads 28 MB of cold weights
//     in 6.1 us, fragments loaded straight into registers (16 rows x 64 B) in 7.2 and more registers.  No barrier: each wave reads what it loaded.
//   * x, at most MT x 16 rows out of L2, takes the same way, once per workgroup; the scales of a batch of blocks are one load each for x and w, a lane
//     per scale, handed round with cross-lane reads (a byte load per use cost 1 us of 10: the address pipe takes 16 cycles per instruction).
//   * 16-bit results take the 8-bit instruction; float32 ones, up to 32 rows those that are quantised again, and all where the caller says so, the EXACT product (see the top).
//   * The waves' sums meet in LDS and are added in wave order; one thread then has 4 neighbouring columns of a row.
// ================================================================================================================================
template <int KIND, bool SWI, bool EXACT, int MT, int NJ, int U, int WAVES>
__global__ void __launch_bounds__(WAVES * 64)
k_fp8_gemm_rows(const GemmArgs a, int R /* <= 16 NJ, a multiple of 4 */, int nb /* blocks in flight per wave, <= U */) {
    constexpr int NT = SWI ? 2 : 1, NW = NJ * NT, T = MT * NW, ESZ = KIND == 0 ? 1 : 4, SLOT = (NW + MT) * 2048;
    static_assert(U * MT <= 4, "one lane per x scale of a batch");
    extern __shared__ __attribute__((aligned(16))) uint8_t smem[];     // [waves][nb][NT][NJ][16 rows of w][128 B], [MT][16 rows of x][128 B]; then [waves][T][64] sums
    v4f* red = reinterpret_cast<v4f*>(smem);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), nw = (int)blockDim.x >> 6;
    const int fi = lane & 15, fg = lane >> 4, lr = lane >> 3;
    const int ncols = SWI ? a.I : a.N, n0 = (int)blockIdx.x * R, rows = min(R, ncols - n0);
    const int chunk = (lane & 7) ^ lr;                                 // source chunk of this lane in every piece of 8 rows
    const uint32_t wo = (uint32_t)(lr * a.ldw) + chunk * 16, xo = (uint32_t)(lr * a.ldx) + chunk * 16;
    // lane -> x scale (block u, row): u * MT * 16 + row; lane -> w scale: u * 4 + half * 2 + (0: the block of 128 of the first row, 1: of the last)
    const uint8_t* sxl = (const uint8_t*)a.sx + (int64_t)min(lane % (MT * 16), a.M - 1) * a.ldsx * ESZ;
    const uint8_t* swl = (const uint8_t*)a.sw + (int64_t)(((SWI && (lane & 2) ? a.I : 0) + n0 + (lane & 1 ? rows - 1 : 0)) >> 7) * a.ldsw * ESZ;
    // lane of the w scale of its operand row (E8M0 in the instruction) or of its 4 result columns (they lie in one block)
    int swi_lane[NW];
#pragma unroll
    for (int t = 0; t < NW; ++t) {
        const int half = t / NJ, first = (half ? a.I : 0) + n0, r = first + min((t % NJ) * 16 + (!EXACT && KIND == 0 ? fi : fg * 4), rows - 1);
        swi_lane[t] = half * 2 + ((r >> 7) != (first >> 7) ? 1 : 0);
    }
    v4f acc[T];
#pragma unroll
    for (int t = 0; t < T; ++t) acc[t] = v4f{0.f, 0.f, 0.f, 0.f};

    auto scale_at = [&](const uint8_t* p, int kb) { return KIND == 0 ? (uint32_t)p[kb] : ((const uint32_t*)p)[kb]; };
    auto frag_at = [&](const uint8_t* p, int h) { return *reinterpret_cast<const v4i*>(p + fi * FP8_G + (((fg + 4 * h) ^ (fi & 7)) << 4)); };
    const uint8_t* mine = smem + (uint32_t)wave * nb * SLOT;
    const uint32_t dst0 = lds_addr(smem) + (uint32_t)wave * nb * SLOT;
    for (int b0 = wave; b0 < a.KB; b0 += nw * nb) {
        const uint32_t vx = scale_at(sxl, min(b0 + lane / (MT * 16) * nw, a.KB - 1)), vw = scale_at(swl, min(b0 + (lane >> 2) * nw, a.KB - 1));
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");             // the reads of the blocks before have left LDS
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int b = b0 + u * nw;
            if (u >= nb || b >= a.KB) continue;
            const bool in = b * FP8_G + chunk * 16 < a.K, ragged = b * FP8_G + FP8_G > a.K;
            const uint32_t dst = dst0 + (uint32_t)(u * SLOT);
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int q = 0; q < NJ * 2; ++q) {
                    if (q * 8 >= rows) break;                          // (the same for the whole workgroup)
                    const uint8_t* base = a.w + ((int64_t)(n0 + q * 8 + (t ? a.I : 0)) * a.ldw + (int64_t)b * FP8_G);
                    if (q * 8 + lr < rows) {                           // rows of the neighbour are not read; their part of LDS feeds results that nobody stores
                        if (ragged) dma_piece_at(in ? base + wo : (const uint8_t*)&g_zero16, dst + (t * NJ * 2 + q) * 1024);
                        else dma_piece_once(wo, base, dst + (t * NJ * 2 + q) * 1024);
                    }
                }
#pragma unroll
            for (int q = 0; q < MT * 2; ++q) {
                if (q * 8 >= a.M) break;
                const uint8_t* base = a.x + ((int64_t)q * 8 * a.ldx + (int64_t)b * FP8_G);
                if (q * 8 + lr < a.M) {
                    if (ragged) dma_piece_at(in ? base + xo : (const uint8_t*)&g_zero16, dst + (NW * 2 + q) * 1024);
                    else dma_piece(xo, base, dst + (NW * 2 + q) * 1024);
                }
            }
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (u >= nb || b0 + u * nw >= a.KB) continue;
            const uint8_t* slot = mine + u * SLOT;
            v4i x[MT][2];
            uint32_t sx[MT], sw[NW];
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                x[i][0] = frag_at(slot + (NW + i) * 2048, 0);
                x[i][1] = frag_at(slot + (NW + i) * 2048, 1);
                sx[i] = __shfl(vx, (u * MT + i) * 16 + fi, 64);
            }
#pragma unroll
            for (int t = 0; t < NW; ++t) sw[t] = __shfl(vw, u * 4 + swi_lane[t], 64);
            if constexpr (!EXACT) {
#pragma unroll
                for (int t = 0; t < NW; ++t) {
                    const v8i w = __builtin_shufflevector(frag_at(slot + t * 2048, 0), frag_at(slot + t * 2048, 1), 0, 1, 2, 3, 4, 5, 6, 7);
#pragma unroll
                    for (int i = 0; i < MT; ++i) {
                        const v8i xv = __builtin_shufflevector(x[i][0], x[i][1], 0, 1, 2, 3, 4, 5, 6, 7);
                        if constexpr (KIND == 0) {
                            acc[i * NW + t] = mma_scaled(w, xv, acc[i * NW + t], sw[t], sx[i]);
                        } else {
                            const v4f d = mma_plain(w, xv, v4f{0.f, 0.f, 0.f, 0.f});
                            const ScalePair s(__uint_as_float(sx[i]), __uint_as_float(sw[t]));
#pragma unroll
                            for (int r = 0; r < 4; ++r) acc[i * NW + t][r] = s.add(d[r], acc[i * NW + t][r]);
                        }
                    }
                }
            } else {
                bf8 xh[MT][4];
#pragma unroll
                for (int i = 0; i < MT; ++i)
#pragma unroll
                    for (int g = 0; g < 4; ++g) xh[i][g] = to_bf16(x[i][g >> 1][(g & 1) * 2], x[i][g >> 1][(g & 1) * 2 + 1]);
#pragma unroll
                for (int t = 0; t < NW; ++t) {
                    v4f d[MT];
#pragma unroll
                    for (int i = 0; i < MT; ++i) d[i] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const v4i w = frag_at(slot + t * 2048, h);
#pragma unroll
                        for (int g = 0; g < 2; ++g) {
                            const bf8 wh = to_bf16(w[g * 2], w[g * 2 + 1]);
#pragma unroll
                            for (int i = 0; i < MT; ++i) d[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wh, xh[i][h * 2 + g], d[i], 0, 0, 0);
                        }
                    }
#pragma unroll
                    for (int i = 0; i < MT; ++i) {
                        const ScalePair s(scale_value(sx[i], KIND), scale_value(sw[t], KIND));
#pragma unroll
                        for (int r = 0; r < 4; ++r) acc[i * NW + t][r] = s.add(d[i][r], acc[i * NW + t][r]);
                    }
                }
            }
        }
    }
    __syncthreads();                                                   // every wave has read its blocks: LDS becomes the sums
#pragma unroll
    for (int t = 0; t < T; ++t) red[(wave * T + t) * 64 + lane] = acc[t];
    __syncthreads();
    for (int e = tid; e < MT * NJ * 64; e += (int)blockDim.x) {        // (m tile, column tile, lane): 4 columns of one row
        const int i = e / (NJ * 64), j = (e >> 6) % NJ, l = e & 63, m = i * 16 + (l & 15), c = j * 16 + (l >> 4) * 4, n = n0 + c;
        if (m >= a.M || c >= rows) continue;
        float v[NT][4];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const v4f* p = red + (i * NW + t * NJ + j) * 64 + l;
            v4f s = p[0];
#pragma unroll
            for (int q = 1; q < WAVES; ++q)
                if (q < nw) s += p[q * T * 64];
#pragma unroll
            for (int r = 0; r < 4; ++r) v[t][r] = s[r];
        }
        if constexpr (SWI) {
            if (a.out_type == 3) {                                     // k_fp8_gemm_finish needs 128 columns for a scale
                *reinterpret_cast<v4f*>(a.ws + (int64_t)m * a.ldws + n) = v4f{v[0][0], v[0][1], v[0][2], v[0][3]};
                *reinterpret_cast<v4f*>(a.ws + (int64_t)m * a.ldws + a.ldws / 2 + n) = v4f{v[1][0], v[1][1], v[1][2], v[1][3]};
                continue;
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) v[0][r] = v[1][r] * silu<EXACT>(v[0][r]);
        }
        finish4(a, v[0], m, n, n0 + rows);
    }
}

// ---- split K: the slices float32 sums, added in slice order, and the epilogue ---------------------------------------------------------------
// 8 columns per thread; 16 threads are one group of 128 columns of the quantised result.
__global__ void __launch_bounds__(256)
k_fp8_gemm_finish(const GemmArgs a, int swi, int c8 /* threads per row: a multiple of 16 */, int kind) {
    const int64_t idx = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (idx >= (int64_t)a.M * c8) return;                              // (whole 16-lane rows leave together)
    const int m = (int)(idx / c8), n = (int)(idx - (int64_t)m * c8) * 8, ncols = swi ? a.I : a.N;
    float v[8] = {}, u[8] = {};
    if (n < ncols) {
        const float* p = a.ws + (int64_t)m * a.ldws + n;
        const int64_t step = (int64_t)a.M * a.ldws;
        for (int s = 0; s < a.splits; ++s, p += step) {
            float t[8];
            fp_load8<2>(p, 0, t);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] += t[i];
            if (swi) {
                fp_load8<2>(p + a.ldws / 2, 0, t);
#pragma unroll
                for (int i = 0; i < 8; ++i) u[i] += t[i];
            }
        }
        if (swi) {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = u[i] * (a.out_type == 2 || a.exact ? silu<true>(v[i]) : silu<false>(v[i]));
        }
        if (a.out_type != 3) {
            finish4(a, v, m, n, ncols);
            finish4(a, v + 4, m, n + 4, ncols);
        }
    }
    if (a.out_type != 3) return;
    float x = 0.f;
    if (n < ncols) {
#pragma unroll
        for (int i = 0; i < 8; ++i) x = fmaxf(x, fp8_finite_abs(v[i]));
    }
    x = row16_max(x);
    uint32_t o[2], code;
    float s;
    fp8_quantize_pack<8>(v, x, kind, o, code, s);
    if (n >= ncols) return;
    *reinterpret_cast<uint2*>((uint8_t*)a.out + (int64_t)m * a.ldo + n) = make_uint2(o[0], o[1]);
    if ((n & 127) == 0) {
        if (kind == 0) ((uint8_t*)a.out_scale)[(int64_t)m * a.ldos + n / FP8_G] = (uint8_t)code;
        else ((float*)a.out_scale)[(int64_t)m * a.ldos + n / FP8_G] = s;
    }
}

// ---- host ---------------------------------------------------------------------------------------------------------------------------------------
constexpr int CUS = 256;

struct Plan {
    int rows;                                                          // 16-row tiles of k_fp8_gemm_rows; 0: tile kernel, -1: big kernel
    int bm, bn, tiles_m, tiles_n, splits;
    int64_t ldws, ws_bytes;
};

// wide: rows of out and residual start on 16 bytes, and EXACT is not asked for (the large kernel has no such form).  (64-bit sizes: M, N up to 2^31 - 1 are rounded up to tiles here)
Plan plan_of(int64_t M, int64_t N, int64_t K, bool swi, int out_type, int kind, bool wide) {
    Plan p{};
    const int64_t KB = (K + FP8_G - 1) / FP8_G, ncols = swi ? N / 2 : N;
    p.ldws = swi ? 2 * ((ncols + 7) / 8 * 8) : (ncols + 7) / 8 * 8;
    // Few rows: the weights stream once (device time at K = 3072, N = 9216, us, against the tile kernel: M = 17 9.4 : 15.1, 32 10.4 : 16.0, 64 13.3 : 18.0;
    // K = 8192, N = 3072: 32 12.3 : 18.7, 64 16.5 : 20.1).  Behind 32 rows x is most of what a workgroup of a wide product reads: N = 32064 at 64 rows
    // 40.1 : 34.0.
    if (M <= 32 || (M <= 64 && ncols <= 64 * CUS)) {
        p.rows = M <= 16 ? 1 : M <= 32 ? 2 : 4;
        p.splits = 1;
        p.ws_bytes = out_type == 3 ? M * p.ldws * 4 : 0;
        return p;
    }
    p.bm = swi ? 64 : 128;
    p.bn = 128;                                                        // columns of the result per tile (SwiGLU: 256 rows of w)
    p.tiles_m = (int)((M + p.bm - 1) / p.bm);
    p.tiles_n = (int)((ncols + p.bn - 1) / p.bn);
    const int64_t tiles = (int64_t)p.tiles_m * p.tiles_n;
    // A round of small tiles (two workgroups per CU) takes as long as one of big tiles (one workgroup), which does twice as much.  us, small : big:
    // 9216 x 3072, M = 256 27.0 : 39.8, 823 (504 tiles) 34.4 : 40.3, 1024 (576) 61.1 : 40.3; 300 x 32064 (753) 61.5 : 46.2; SwiGLU 2 x 8192 x 3072, M = 256
    // 42.1 : 45.8, 512 (512) 50.6 : 46.0.
    if (kind == 0 && KB >= 2 && out_type != 2 && tiles >= 2 * CUS && wide && ncols % 8 == 0) {
        p.rows = -1;
        p.tiles_m = (int)((M + 255) / 256);
        p.tiles_n = (int)((ncols + (swi ? 127 : 255)) / (swi ? 128 : 256));
        p.splits = 1;
        // A sparse last round stays as it is: alone on the card its K tiles take 0.97 us, in a full round 1.7 (power and memory are shared).  6568 x 3072 x 8192, 252 + 60
        // tiles, 171.0 us; those 60 as small tiles with K cut 171.8, as big ones with K in four slices 171.0; 2560 x 9216 x 3072 79.7 against 96.8 in slices.
        return p;
    }
    // Fewer tiles than one round of two workgroups per CU: cut K so that a round is filled, at least 4 K tiles per slice.  (us with at least 4 : 3 : 2, 77 x 1003 x 1040
    // 10.6 : 9.5 : 9.9, 100 x 3072 x 3072 15.5 : 16.3 : 20.0, 128 x 3072 x 8192 22.7 : 26.2 : 26.4, 100 x 9216 x 3072 20.1 : 22.4 : 22.4.)
    p.splits = (int)std::max<int64_t>(1, std::min<int64_t>(2 * CUS / tiles, KB / 4));
    p.ws_bytes = p.splits > 1 ? p.splits * M * p.ldws * 4 : 0;
    return p;
}

int32_t bad(const char* msg) {
    d3d_set_error_(msg);
    return D3D_EINVAL;
}

// more than 64 KiB of dynamic LDS is asked for once per kernel and device
int32_t allow_lds(const void* kernel, size_t bytes, std::atomic<uint64_t>& done) {
    int dev = 0;
    D3D_HIP(hipGetDevice(&dev));
    const uint64_t bit = 1ull << (dev & 63);
    if (!(done.load(std::memory_order_relaxed) & bit)) {
        D3D_HIP(hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
        done.fetch_or(bit, std::memory_order_relaxed);
    }
    return D3D_OK;
}

template <int KIND, bool SWI, bool EXACT>
int32_t launch_tile(const GemmArgs& a, hipStream_t s) {
    constexpr int BM = SWI ? 64 : 128, BN = SWI ? 256 : 128;
    const size_t sh = 2 * (BM + BN) * FP8_G + (SWI ? 0 : 2 * 1024);
    static std::atomic<uint64_t> done{0};
    const int32_t rc = allow_lds(reinterpret_cast<const void*>(&k_fp8_gemm_tile<KIND, SWI, EXACT, BM, BN>), sh, done);
    if (rc != D3D_OK) return rc;
    hipLaunchKernelGGL((k_fp8_gemm_tile<KIND, SWI, EXACT, BM, BN>), dim3((uint32_t)(a.tiles_m * a.tiles_n * a.splits)), dim3(256), sh, s, a);
    D3D_LAUNCH_CHECK();
}

template <int KIND, bool SWI, bool EXACT, int MT, int NJ>
int32_t launch_rows_of(const GemmArgs& a, int R, hipStream_t s) {
    constexpr int NW = NJ * (SWI ? 2 : 1), T = MT * NW, U = 4 / MT, WAVES = SWI || MT == 4 ? 8 : 16, SLOT = (NW + MT) * 2048, LDS = 160 * 1024;
    const int64_t grid = ((int64_t)(SWI ? a.I : a.N) + R - 1) / R;
    const int per = (a.KB + WAVES - 1) / WAVES, nw = (a.KB + per - 1) / per;                    // K blocks of a wave; the waves that takes
    // more workgroups than CUs: two of them per CU, so that one loads while the other adds up (16384 x 3072 at 8 rows: 12.2 us; one, with twice
    // the blocks in flight: 14.2)
    const int nb = std::min({U, per, std::max(1, (grid > CUS ? LDS / 2 : LDS) / (nw * SLOT))});
    const size_t sh = (size_t)nw * std::max(nb * SLOT, T * 1024);
    if (grid * nw * 64 >= (int64_t)1 << 32) return bad("d3d_fp8_gemm: too many columns for one launch");
    static_assert(WAVES * (SLOT > T * 1024 ? SLOT : T * 1024) <= LDS, "one block per wave fits");
    static std::atomic<uint64_t> done{0};
    const int32_t rc = allow_lds(reinterpret_cast<const void*>(&k_fp8_gemm_rows<KIND, SWI, EXACT, MT, NJ, U, WAVES>), LDS, done);
    if (rc != D3D_OK) return rc;
    hipLaunchKernelGGL((k_fp8_gemm_rows<KIND, SWI, EXACT, MT, NJ, U, WAVES>), dim3((uint32_t)grid), dim3(nw * 64), sh, s, a, R, nb);
    D3D_LAUNCH_CHECK();
}
template <int KIND, bool SWI, bool EXACT, int MT>
int32_t launch_rows(const GemmArgs& a, hipStream_t s) {
    // R: one workgroup per CU up to 48 rows (SwiGLU: 16), else a whole number of them of up to 32
    constexpr int MOST = SWI ? 16 : 48, MANY = SWI ? 16 : 32;
    const int64_t ncols = SWI ? a.I : a.N, per_cu = ncols <= CUS * MOST ? 1 : (ncols + CUS * MANY - 1) / (CUS * MANY);
    const int R = std::max(8, (int)((ncols + CUS * per_cu - 1) / (CUS * per_cu) + 3) / 4 * 4);
    if constexpr (MOST > 16) {
        if (R > 32) return launch_rows_of<KIND, SWI, EXACT, MT, 3>(a, R, s);
        if (R > 16) return launch_rows_of<KIND, SWI, EXACT, MT, 2>(a, R, s);
    }
    return launch_rows_of<KIND, SWI, EXACT, MT, 1>(a, R, s);
}
template <bool SWI, int DT>
int32_t launch_big_of(const GemmArgs& a, hipStream_t s) {
    const size_t sh = 2 * 512 * FP8_G + 2 * 2048;
    static std::atomic<uint64_t> done{0};
    const int32_t rc = allow_lds(reinterpret_cast<const void*>(&k_fp8_gemm_big<SWI, DT>), sh, done);
    if (rc != D3D_OK) return rc;
    hipLaunchKernelGGL((k_fp8_gemm_big<SWI, DT>), dim3((uint32_t)(a.tiles_m * a.tiles_n)), dim3(256), sh, s, a);
    D3D_LAUNCH_CHECK();
}
template <bool SWI>
int32_t launch_big(const GemmArgs& a, hipStream_t s) {
    if constexpr (SWI) {
        if (a.out_type == 3) return launch_big_of<SWI, 3>(a, s);
    }
    return a.out_type == 0 ? launch_big_of<SWI, 0>(a, s) : launch_big_of<SWI, 1>(a, s);
}
template <int KIND, bool SWI>
int32_t launch(const GemmArgs& a, int rows, hipStream_t s) {
    // a result that is quantised again is EXACT too while that is free (8 rows of 8192 x 3072: 15.7 us; at 64 rows 32.4 against 25.6)
    const bool exact = a.out_type == 2 || a.exact || (a.out_type == 3 && rows <= 2);
    if constexpr (KIND == 0) {
        if (rows < 0) return launch_big<SWI>(a, s);
    }
    if (rows == 1) return exact ? launch_rows<KIND, SWI, true, 1>(a, s) : launch_rows<KIND, SWI, false, 1>(a, s);
    if (rows == 2) return exact ? launch_rows<KIND, SWI, true, 2>(a, s) : launch_rows<KIND, SWI, false, 2>(a, s);
    if (rows == 4) return exact ? launch_rows<KIND, SWI, true, 4>(a, s) : launch_rows<KIND, SWI, false, 4>(a, s);
    return a.out_type == 2 || a.exact ? launch_tile<KIND, SWI, true>(a, s) : launch_tile<KIND, SWI, false>(a, s);
}

}  // namespace

extern "C" {

int64_t d3d_fp8_gemm_workspace(int32_t M, int32_t N, int32_t K, int32_t swiglu, int32_t out_type, int32_t scale_kind) {
    if (M <= 0 || N <= 0 || K <= 0) return 0;
    // (which kernel is taken depends on where rows start and on `exact`, too: enough for both)
    return std::max(plan_of(M, N, K, swiglu != 0, out_type, scale_kind, true).ws_bytes, plan_of(M, N, K, swiglu != 0, out_type, scale_kind, false).ws_bytes);
}

int32_t d3d_fp8_gemm(const d3d_fp8_gemm_args* g) {
    if (!g || g->M < 0 || g->N < 0 || g->K < 0 || g->scale_kind < 0 || g->scale_kind > 1 || g->out_type < 0 || g->out_type > 3)
        return bad("d3d_fp8_gemm: bad sizes or types");
    const bool swi = g->swiglu != 0;
    const int ncols = swi ? g->N / 2 : g->N;
    if (g->M == 0 || ncols == 0) return D3D_OK;
    if (g->K == 0 || g->K % 16) return bad("d3d_fp8_gemm: K must be a positive multiple of 16");
    if (swi && (g->N % 32 || g->bias || g->residual)) return bad("d3d_fp8_gemm: SwiGLU takes 2 x (a multiple of 16) rows of w and neither bias nor residual");
    if (!swi && g->out_type == 3) return bad("d3d_fp8_gemm: only SwiGLU quantises its result");
    if (!g->x || !g->w || !g->sx || !g->sw || !g->out || (g->out_type == 3 && !g->out_scale)) return bad("d3d_fp8_gemm: null operand");
    if (((uintptr_t)g->x & 15) || ((uintptr_t)g->w & 15) || g->ldx % 16 || g->ldw % 16 || g->ldx < 0 || g->ldw < 0)
        return bad("d3d_fp8_gemm: rows of x and w must start on 16 bytes");
    if (g->out_type == 3 && (((uintptr_t)g->out & 15) || g->ldo % 16)) return bad("d3d_fp8_gemm: rows of a quantised result must start on 16 bytes");
    if (g->K >= 1 << 24) return bad("d3d_fp8_gemm: K of 2^24 and more");
    if (g->ldx >= (int64_t)1 << 24 || g->ldw >= (int64_t)1 << 24) return bad("d3d_fp8_gemm: rows further than 16 MiB apart");
    if (g->ldsx < 0 || g->ldsw < 0 || g->ldsx >= 1 << 20 || (int64_t)(g->N / FP8_G + 1) * g->ldsw >= 1 << 29) return bad("d3d_fp8_gemm: scale rows too far apart");
    if (swi && (int64_t)g->N * g->ldw >= (int64_t)1 << 32) return bad("d3d_fp8_gemm: SwiGLU weights of 4 GiB and more");
    if (g->ldr < 0) return bad("d3d_fp8_gemm: residual rows in descending order");
    if (g->ldo < 0 || (g->M > 1 && (g->ldo < ncols || (g->out_type == 3 && g->ldos < (ncols + FP8_G - 1) / FP8_G))))
        return bad("d3d_fp8_gemm: rows of the result would lie over one another");
    const bool wide = !g->exact && ((uintptr_t)g->out & 15) == 0 && g->ldo % 8 == 0 && g->ldo < 1 << 22 && g->ldr < 1 << 22 && (!g->residual || (((uintptr_t)g->residual & 15) == 0 && g->ldr % 8 == 0)) && ((uintptr_t)g->bias & 15) == 0;
    const Plan p = plan_of(g->M, g->N, g->K, swi, g->out_type, g->scale_kind, wide);
    const int64_t c8 = ((int64_t)ncols + 127) / 128 * 16;              // threads per row of k_fp8_gemm_finish
    if (p.ws_bytes && g->M * c8 >= ((int64_t)1 << 32) - 256) return bad("d3d_fp8_gemm: too many columns for one launch");
    if (p.rows <= 0 && (int64_t)p.tiles_m * p.tiles_n * p.splits >= (int64_t)1 << 24) return bad("d3d_fp8_gemm: too many tiles for one launch");
    if (p.ws_bytes > g->workspace_bytes || (p.ws_bytes && (!g->workspace || ((uintptr_t)g->workspace & 15))))
        return bad("d3d_fp8_gemm: workspace smaller than d3d_fp8_gemm_workspace() or not on 16 bytes");
    GemmArgs a{};
    a.x = (const uint8_t*)g->x; a.w = (const uint8_t*)g->w; a.sx = g->sx; a.sw = g->sw; a.bias = g->bias; a.res = g->residual;
    a.out = g->out; a.out_scale = g->out_scale; a.ws = (float*)g->workspace;
    a.ldx = g->ldx; a.ldw = g->ldw; a.ldsx = g->ldsx; a.ldsw = g->ldsw; a.ldr = g->ldr; a.ldo = g->ldo; a.ldos = g->ldos; a.ldws = p.ldws;
    a.M = g->M; a.N = g->N; a.K = g->K; a.KB = (g->K + FP8_G - 1) / FP8_G; a.I = ncols;
    a.tiles_m = p.tiles_m; a.tiles_n = p.tiles_n; a.splits = p.splits; a.out_type = g->out_type; a.exact = g->exact != 0;
    const int eb = g->out_type == 2 ? 16 : 8;                          // bytes of four columns
    const int es = eb / 4;
    a.vec = g->out_type == 3 || (((uintptr_t)g->out % eb) == 0 && (g->ldo * es) % eb == 0 &&
                                 (!g->residual || (((uintptr_t)g->residual % eb) == 0 && (g->ldr * es) % eb == 0)));
    hipStream_t s = (hipStream_t)g->stream;
    const int32_t rc = swi ? (g->scale_kind == 0 ? launch<0, true>(a, p.rows, s) : launch<1, true>(a, p.rows, s))
                           : (g->scale_kind == 0 ? launch<0, false>(a, p.rows, s) : launch<1, false>(a, p.rows, s));
    if (rc != D3D_OK || !p.ws_bytes) return rc;
    const int64_t nb = (a.M * c8 + 255) / 256;
    hipLaunchKernelGGL(k_fp8_gemm_finish, dim3((uint32_t)nb), dim3(256), 0, s, a, swi ? 1 : 0, (int)c8, g->scale_kind);
    D3D_LAUNCH_CHECK();
}

}  // extern "C"
