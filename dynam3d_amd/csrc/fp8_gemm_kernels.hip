// fp8_gemm_kernels.hip -- the 8-bit "NT" matrix product of the language model's linears on gfx950:
//
//   y[m, n] = sum_b sx[m, b] sw[n / 128, b] sum_{k in block b} xq[m, k] wq[n, k]     (+ bias[n] + residual[m, n], or SwiGLU over two halves)
//
// xq (M, K), wq (N, K) E4M3, one scale per row and 128 columns of x and per 128 x 128 block of w (fp8_common.h: E8M0 or float32).  Sums are
// float32; the result is rounded once, to bf16 / fp16 / float32 -- or, behind SwiGLU, quantised again for the product that follows.
//
// What the 8-bit matrix instructions round (measured, all shapes alike): 8 neighbouring products are aligned to the largest of them and cut 13
// bits below it, then added to the float32 accumulator.  A product loses less than 2^-13 of the largest beside it, at most 7 * 2^-13 sum |x w| in
// all and ~2^-14 of a result of random signs: far inside half a step of bf16 (2^-9), below one of fp16 (2^-12), but not of float32.  A
// float32 result is therefore computed EXACTly: E4M3 converted to bf16 in registers (exact), products on the bf16 matrix instruction (exact,
// aligned to 24 bits), half the rate.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <atomic>

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
    int vec;                         // rows of out / res allow 4-column vector accesses
};

__device__ uint4 g_zero16;           // what the lanes behind the end of a ragged K read: an E4M3 zero can meet no NaN

// One 1 KiB piece (8 rows x 128 B) of an operand tile into LDS, 16 bytes per lane, no registers in between.  In asm so that the compiler does
// not drain it in front of every LDS read (it counts the builtin as a pending LDS write); the K loops wait for it explicitly.
__device__ __forceinline__ void dma_piece(uint32_t voff, const uint8_t* base, uint32_t dst) {
    const uint32_t d = __builtin_amdgcn_readfirstlane(dst);
    uint32_t keep;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %3\n\ts_mov_b32 m0, %0"
                 : "=&s"(keep) : "v"(voff), "s"(d), "s"(base) : "memory");
}
__device__ __forceinline__ void dma_piece_at(const uint8_t* addr, uint32_t dst) {
    const uint32_t d = __builtin_amdgcn_readfirstlane(dst);
    uint32_t keep;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off\n\ts_mov_b32 m0, %0"
                 : "=&s"(keep) : "v"(addr), "s"(d) : "memory");
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

__device__ __forceinline__ float silu(float x) { return x / (1.f + __expf(-x)); }

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
//   * E8M0: the scales ride in the instruction.  float32 scales, and EXACT: each K tile's product is multiplied by sx * sw and added.
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

    // scales of this lane's rows: x row per i, w row (E8M0: of the lane's operand row; float32: of its 4 result columns, one block) per j
    const uint8_t* sxb = (const uint8_t*)a.sx + (int64_t)row0 * a.ldsx * ESZ;
    uint32_t sxo[4], swo[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        sxo[i] = (uint32_t)(min(wr * 64 + i * 16 + fi, a.M - 1 - row0) * (int)a.ldsx * ESZ);
        swo[i] = (uint32_t)((wrow(wc * 64 + i * 16 + fi) >> 7) * (int)a.ldsw * ESZ);
    }
    uint32_t sx[4], sw[4], nsx[4], nsw[4];
    auto load_scales = [&](int kt) {
        const uint8_t *px = sxb + kt * ESZ, *pw = (const uint8_t*)a.sw + kt * ESZ;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            nsx[i] = KIND == 0 ? (uint32_t)px[sxo[i]] : *(const uint32_t*)(px + sxo[i]);
            nsw[i] = KIND == 0 ? (uint32_t)pw[swo[i]] : *(const uint32_t*)(pw + swo[i]);
        }
    };

    v4f acc[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = v4f{0.f, 0.f, 0.f, 0.f};

    if (order.n > 0) {
        load_scales(order.tile(0));
        stage(0);
    }
    for (int p = 0; p < order.n; ++p) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();                                 // tile p has landed everywhere, tile p - 1 has been read everywhere
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            sx[i] = nsx[i];
            sw[i] = nsw[i];
            asm volatile("" : "+v"(sx[i]), "+v"(sw[i]));              // the compiler's own wait for the scales belongs HERE, not behind the next DMA
        }
        if (p + 1 < order.n) {
            load_scales(order.tile(p + 1));
            stage(p + 1);
        }
        const uint8_t* la = smem + (p & 1) * STAGE;
        const uint8_t* lb = la + BM * FP8_G;
        if constexpr (EXACT) {
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
                        const float s = scale_value(sx[i], KIND) * scale_value(sw[jh + j], KIND);
#pragma unroll
                        for (int r = 0; r < 4; ++r) acc[i][jh + j][r] = __builtin_fmaf(d[i][j][r], s, acc[i][jh + j][r]);
                    }
            }
        } else {
            v8i af[4], bf[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int rb = wc * 64 + i * 16 + fi, ra = wr * 64 + i * 16 + fi, s = fi & 7;
                bf[i] = frag(lb + rb * FP8_G + ((fg ^ s) << 4), lb + rb * FP8_G + (((fg + 4) ^ s) << 4));
                af[i] = frag(la + ra * FP8_G + ((fg ^ s) << 4), la + ra * FP8_G + (((fg + 4) ^ s) << 4));
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if constexpr (KIND == 0) {
                        acc[i][j] = mma_scaled(bf[j], af[i], acc[i][j], sw[j], sx[i]);
                    } else {
                        const v4f d = mma_plain(bf[j], af[i], v4f{0.f, 0.f, 0.f, 0.f});
                        const float s = __uint_as_float(sx[i]) * __uint_as_float(sw[j]);
#pragma unroll
                        for (int r = 0; r < 4; ++r) acc[i][j][r] = __builtin_fmaf(d[r], s, acc[i][j][r]);
                    }
                }
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
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
                for (int r = 0; r < 4; ++r) v[i][j * 4 + r] = acc[i][2 * j + 1][r] * silu(acc[i][2 * j][r]);
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

// ---- split K: the slices' float32 sums, added in slice order, and the epilogue ---------------------------------------------------------------
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
            for (int i = 0; i < 8; ++i) v[i] = u[i] * silu(v[i]);
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
    int bm, bn, tiles_m, tiles_n, splits;
    int64_t ldws, ws_bytes;
};

Plan plan_of(int M, int N, int K, bool swi) {
    Plan p{};
    const int KB = (K + FP8_G - 1) / FP8_G, ncols = swi ? N / 2 : N;
    p.bm = swi ? 64 : 128;
    p.bn = 128;                                                        // columns of the result per tile (SwiGLU: 256 rows of w)
    p.tiles_m = (M + p.bm - 1) / p.bm;
    p.tiles_n = (ncols + p.bn - 1) / p.bn;
    const int64_t tiles = (int64_t)p.tiles_m * p.tiles_n;
    // fewer tiles than one round of two workgroups per CU: cut K so that a round is filled, at least 4 K tiles per slice
    p.splits = (int)std::max<int64_t>(1, std::min<int64_t>(2 * CUS / tiles, KB / 4));
    p.ldws = swi ? 2 * ((ncols + 7) / 8 * 8) : (ncols + 7) / 8 * 8;
    p.ws_bytes = p.splits > 1 ? (int64_t)p.splits * M * p.ldws * 4 : 0;
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
    const size_t sh = 2 * (BM + BN) * FP8_G;
    static std::atomic<uint64_t> done{0};
    const int32_t rc = allow_lds(reinterpret_cast<const void*>(&k_fp8_gemm_tile<KIND, SWI, EXACT, BM, BN>), sh, done);
    if (rc != D3D_OK) return rc;
    hipLaunchKernelGGL((k_fp8_gemm_tile<KIND, SWI, EXACT, BM, BN>), dim3((uint32_t)(a.tiles_m * a.tiles_n * a.splits)), dim3(256), sh, s, a);
    D3D_LAUNCH_CHECK();
}

}  // namespace

extern "C" {

int64_t d3d_fp8_gemm_workspace(int32_t M, int32_t N, int32_t K, int32_t swiglu) {
    if (M <= 0 || N <= 0 || K <= 0) return 0;
    return plan_of(M, N, K, swiglu != 0).ws_bytes;
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
    if (g->ldx >= (int64_t)1 << 24 || g->ldw >= (int64_t)1 << 24) return bad("d3d_fp8_gemm: rows further than 16 MiB apart");
    if (g->ldsx < 0 || g->ldsw < 0 || g->ldsx >= 1 << 20 || (int64_t)(g->N / FP8_G + 1) * g->ldsw >= 1 << 29) return bad("d3d_fp8_gemm: scale rows too far apart");
    if (swi && (int64_t)g->N * g->ldw >= (int64_t)1 << 32) return bad("d3d_fp8_gemm: SwiGLU weights of 4 GiB and more");
    const Plan p = plan_of(g->M, g->N, g->K, swi);
    if ((int64_t)p.tiles_m * p.tiles_n * p.splits >= (int64_t)1 << 31) return bad("d3d_fp8_gemm: too many tiles for one launch");
    if (p.ws_bytes > g->workspace_bytes || (p.ws_bytes && (!g->workspace || ((uintptr_t)g->workspace & 15))))
        return bad("d3d_fp8_gemm: workspace smaller than d3d_fp8_gemm_workspace() or not on 16 bytes");
    GemmArgs a{};
    a.x = (const uint8_t*)g->x; a.w = (const uint8_t*)g->w; a.sx = g->sx; a.sw = g->sw; a.bias = g->bias; a.res = g->residual;
    a.out = g->out; a.out_scale = g->out_scale; a.ws = (float*)g->workspace;
    a.ldx = g->ldx; a.ldw = g->ldw; a.ldsx = g->ldsx; a.ldsw = g->ldsw; a.ldr = g->ldr; a.ldo = g->ldo; a.ldos = g->ldos; a.ldws = p.ldws;
    a.M = g->M; a.N = g->N; a.K = g->K; a.KB = (g->K + FP8_G - 1) / FP8_G; a.I = ncols;
    a.tiles_m = p.tiles_m; a.tiles_n = p.tiles_n; a.splits = p.splits; a.out_type = g->out_type;
    const int eb = g->out_type == 2 ? 16 : 8;                          // bytes of four columns
    const int es = eb / 4;
    a.vec = g->out_type == 3 || (((uintptr_t)g->out % eb) == 0 && (g->ldo * es) % eb == 0 &&
                                 (!g->residual || (((uintptr_t)g->residual % eb) == 0 && (g->ldr * es) % eb == 0)));
    hipStream_t s = (hipStream_t)g->stream;
    const int32_t rc = g->out_type == 2
                           ? (swi ? (g->scale_kind == 0 ? launch_tile<0, true, true>(a, s) : launch_tile<1, true, true>(a, s))
                                  : (g->scale_kind == 0 ? launch_tile<0, false, true>(a, s) : launch_tile<1, false, true>(a, s)))
                           : (swi ? (g->scale_kind == 0 ? launch_tile<0, true, false>(a, s) : launch_tile<1, true, false>(a, s))
                                  : (g->scale_kind == 0 ? launch_tile<0, false, false>(a, s) : launch_tile<1, false, false>(a, s)));
    if (rc != D3D_OK || p.splits == 1) return rc;
    const int c8 = (ncols + 127) / 128 * 16;
    const int64_t nb = ((int64_t)a.M * c8 + 255) / 256;
    hipLaunchKernelGGL(k_fp8_gemm_finish, dim3((uint32_t)nb), dim3(256), 0, s, a, swi ? 1 : 0, c8, g->scale_kind);
    D3D_LAUNCH_CHECK();
}

}  // extern "C"
