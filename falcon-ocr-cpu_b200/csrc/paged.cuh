// paged.cuh -- device helpers shared by the rotary kernels and the paged
// 8-bit KV cache (rope.cu, paged_append.cu, paged_attention.cu): rows of
// heads in FP32 or BF16, a batch's sequences, and the 8-bit codes.
#pragma once

#include <float.h>

#include "fo_common.cuh"
#include "fo_kernels.h"

namespace fo {

// ------------------------------------------------------------------ launches
// The kernels here follow one another closely (a decode step is an append and
// an attention, of some microseconds each): each lets the next one be set up as
// soon as all its own blocks run, and waits for the one before it to be over
// before it touches memory.  What that one writes (scales, lengths, a rotation
// table) changes in this one's lifetime, so nothing here is loaded through the
// read-only path, which is for memory that does not; and the wait is a barrier to
// the compiler for ordinary loads.
__device__ __forceinline__ void wait_for_prior_kernel() {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
}
template <typename... Params, typename... Args>
cudaError_t launch(void (*kernel)(Params...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// ------------------------------------------------------------- row elements
// Ordinary loads: fo_rope may write the rows that it reads.
template <typename T>
__device__ __forceinline__ float load1(const T *p);
template <>
__device__ __forceinline__ float load1<float>(const float *p) { return *p; }
template <>
__device__ __forceinline__ float load1<uint16_t>(const uint16_t *p) { return bf16_f32(*p); }

// Eight adjacent elements as they lie in memory (16 bytes of BF16, 32 of
// FP32), 16-byte aligned, and as floats.
template <typename T>
struct Raw8 {
    uint4 w[sizeof(T) / 2];
};
template <typename T>
__device__ __forceinline__ Raw8<T> load_raw8(const T *p) {
    Raw8<T> r;
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; i++) r.w[i] = reinterpret_cast<const uint4 *>(p)[i];
    return r;
}
__device__ __forceinline__ void unpack8(const Raw8<float> &r, float *x) {
    const uint32_t w[8] = {r.w[0].x, r.w[0].y, r.w[0].z, r.w[0].w, r.w[1].x, r.w[1].y, r.w[1].z, r.w[1].w};
#pragma unroll
    for (int i = 0; i < 8; i++) x[i] = __uint_as_float(w[i]);
}
__device__ __forceinline__ void unpack8(const Raw8<uint16_t> &r, float *x) {
    const uint32_t w[4] = {r.w[0].x, r.w[0].y, r.w[0].z, r.w[0].w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        x[2 * i] = __uint_as_float(w[i] << 16);
        x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    }
}
template <typename T>
__device__ __forceinline__ void load8(const T *p, float *x) {
    unpack8(load_raw8(p), x);
}

// Two floats as a BF16 pair, each rounded to nearest even (NaN stays NaN).
__device__ __forceinline__ uint32_t bf16_pair(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

__device__ __forceinline__ void store1(float *p, float x) { *p = x; }
__device__ __forceinline__ void store1(uint16_t *p, float x) { *p = (uint16_t)bf16_pair(x, 0.0f); }
__device__ __forceinline__ void store8(float *p, const float *x) {
    reinterpret_cast<float4 *>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
    reinterpret_cast<float4 *>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
}
__device__ __forceinline__ void store8(uint16_t *p, const float *x) {
    *reinterpret_cast<uint4 *>(p) =
        make_uint4(bf16_pair(x[0], x[1]), bf16_pair(x[2], x[3]), bf16_pair(x[4], x[5]), bf16_pair(x[6], x[7]));
}

// ---------------------------------------------------------------- rotation
// An entry of the rotation's table.  (A load that is as coherent as any, behind the
// wait for the prior kernel like all volatile ones, but that the compiler need
// not keep in order with the rows' loads and stores: C++'s takes 18.0 us for 6,544
// FP32 rows of 24 heads of 64, this one 16.5.)
__device__ __forceinline__ float2 load_entry(const float2 *p) {
    float2 cs;
    asm volatile("ld.global.v2.f32 {%0, %1}, [%2];" : "=f"(cs.x), "=f"(cs.y) : "l"(p));
    return cs;
}
// A pair's two results, every product and sum rounded on its own.
__device__ __forceinline__ float rot_first(float a, float b, float2 cs) {
    return __fsub_rn(__fmul_rn(a, cs.x), __fmul_rn(b, cs.y));
}
__device__ __forceinline__ float rot_second(float a, float b, float2 cs) {
    return __fadd_rn(__fmul_rn(b, cs.x), __fmul_rn(a, cs.y));
}

// ---------------------------------------------------------------- sequences
// Sequence b of a batch: its rows [first, first + n) and its positions.  What
// does not fit its buffers (rows out of order or beyond total_rows, more than
// max_rows; a length beyond the page table) raises FO_DEVERR_PAGED and leaves
// the sequence without rows, or without positions.
struct Sequence {
    int first, len, n;
};
__device__ __forceinline__ Sequence load_sequence(const fo_paged_batch &b, int page_size, int seq, unsigned *err) {
    // Rows and a table's positions are below 2^31 (checked on the host).
    Sequence s;
    s.len = b.lens[seq];
    if (b.row_start) {
        const int r0 = b.row_start[seq], r1 = b.row_start[seq + 1];
        s.first = r0;
        s.n = r1 - r0;
        if (r0 < 0 || r1 < r0 || r1 > (int)b.total_rows || s.n > (int)b.max_rows) {
            atomicOr(err, FO_DEVERR_PAGED);
            s.first = 0;
            s.n = 0;
        }
    } else {
        s.first = seq * (int)b.max_rows;
        s.n = (int)b.max_rows;
    }
    if (s.len > (int)b.table_stride * page_size) {
        atomicOr(err, FO_DEVERR_PAGED);
        s.len = 0;
    }
    s.len = max(s.len, 0);
    return s;
}

// The pool's page number for a sequence's page j (0 and the error word for
// one outside the pool).
__device__ __forceinline__ int64_t page_of(const fo_paged_batch &b, int64_t n_pages, int64_t seq, int64_t j,
                                           unsigned *err, bool &valid) {
    const int64_t p = b.page_table[seq * b.table_stride + j];
    valid = p >= 0 && p < n_pages;
    if (!valid) atomicOr(err, FO_DEVERR_PAGED);
    return valid ? p : 0;
}

// -------------------------------------------------------------------- codes
__device__ __forceinline__ float code_max(int format) { return format == FO_PAGED_I8 ? 127.0f : 448.0f; }

// A value against its block's scale, x / scale rounded once, saturated to the
// largest code (so is an infinity); NaN, and anything in a block of scale 0,
// gives 0.
__device__ __forceinline__ float scaled(float x, float scale, float top) {
    const float y = __fdiv_rn(x, scale);
    return scale > 0.0f && x == x ? fminf(fmaxf(y, -top), top) : 0.0f;
}

// Four codes from four values within the codes' range, rounded to nearest
// even.  1.5 * 2^23 + x has the integer nearest x in its low bits.
template <int FORMAT>
__device__ __forceinline__ uint32_t encode4(float a, float b, float c, float d) {
    if constexpr (FORMAT == FO_PAGED_I8) {
        const uint32_t x = __float_as_uint(a + 12582912.0f), y = __float_as_uint(b + 12582912.0f);
        const uint32_t z = __float_as_uint(c + 12582912.0f), w = __float_as_uint(d + 12582912.0f);
        return __byte_perm(__byte_perm(x, y, 0x0040), __byte_perm(z, w, 0x0040), 0x5410);
    } else {
        uint32_t r;
        asm("{\n\t.reg .b16 lo, hi;\n\t"
            "cvt.rn.satfinite.e4m3x2.f32 lo, %2, %1;\n\t"
            "cvt.rn.satfinite.e4m3x2.f32 hi, %4, %3;\n\t"
            "mov.b32 %0, {lo, hi};\n\t}"
            : "=r"(r)
            : "f"(a), "f"(b), "f"(c), "f"(d));
        return r;
    }
}

// Eight values x as codes of x / scale (scaled(), then encode4()).  Nearly always
// x times the scale's reciprocal, off from the quotient by 2^-23 of it at most,
// rounds to the same code, and only where one of the eight comes near a tie
// between two codes (or is one of FP8's subnormal codes, or the reciprocal is no
// normal number, or a value is not finite) are the divisions done: a third of
// their instructions.
template <int FORMAT>
__device__ __forceinline__ uint2 encode8(const float *x, float scale, float inverse, bool exact) {
    if constexpr (FORMAT == FO_PAGED_I8) {
        // 1.5 * 2^23 + y has the integer nearest y in its low bits.
        uint32_t z[8];
        float most = 0.0f;  // distance from an integer
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const float y = x[e] * inverse, m = y + 12582912.0f;
            z[e] = __float_as_uint(m);
            most = fmaxf(most, fabsf(y - (m - 12582912.0f)));
        }
        if (!(most < 0.4999f) || exact) {
            float y[8];
#pragma unroll
            for (int e = 0; e < 8; e++) y[e] = scaled(x[e], scale, code_max(FORMAT));
            return make_uint2(encode4<FORMAT>(y[0], y[1], y[2], y[3]), encode4<FORMAT>(y[4], y[5], y[6], y[7]));
        }
        return make_uint2(
            __byte_perm(__byte_perm(z[0], z[1], 0x0040), __byte_perm(z[2], z[3], 0x0040), 0x5410),
            __byte_perm(__byte_perm(z[4], z[5], 0x0040), __byte_perm(z[6], z[7], 0x0040), 0x5410));
    } else {
        // A normal code has 20 bits fewer than FP32; a tie is a half of their range.
        float y[8];
        uint32_t near = 0xFFFFFu;
        float least = 1.0f;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            y[e] = x[e] * inverse;
            near = min(near, (__float_as_uint(y[e]) + 0x80010u) & 0xFFFFFu);
            least = fminf(least, fabsf(y[e]));
        }
        if (near < 0x20u || least < 0.015625f || exact) {
#pragma unroll
            for (int e = 0; e < 8; e++) y[e] = scaled(x[e], scale, code_max(FORMAT));
        }
        return make_uint2(encode4<FORMAT>(y[0], y[1], y[2], y[3]), encode4<FORMAT>(y[4], y[5], y[6], y[7]));
    }
}

// Two FP8 codes as an FP16 pair (exact); the low byte's in the low half.
__device__ __forceinline__ uint32_t e4m3x2_f16x2(uint32_t pair) {
    uint32_t r;
    asm("{\n\t.reg .b16 lo;\n\tcvt.u16.u32 lo, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\t}" : "=r"(r) : "r"(pair));
    return r;
}
__device__ __forceinline__ float2 f16x2_f32x2(uint32_t h) {
    float2 f;
    asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %2;\n\tcvt.f32.f16 %0, lo;\n\tcvt.f32.f16 %1, hi;\n\t}"
        : "=f"(f.x), "=f"(f.y)
        : "r"(h));
    return f;
}

// Four codes as floats (exact).
template <int FORMAT>
__device__ __forceinline__ void decode4(uint32_t w, float *f) {
    if constexpr (FORMAT == FO_PAGED_I8) {
        s8x4_f32(w, f);
    } else {
        const float2 lo = f16x2_f32x2(e4m3x2_f16x2(w & 0xFFFFu)), hi = f16x2_f32x2(e4m3x2_f16x2(w >> 16));
        f[0] = lo.x, f[1] = lo.y, f[2] = hi.x, f[3] = hi.y;
    }
}

}  // namespace fo
