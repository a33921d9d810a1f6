// Device-side pieces shared by the readout operators: 16-byte units of a row
// at any alignment, e4m3 blocks of 128, element types.
//
// A block of 128 entries z with A = max |z| is stored as the codes
// e4m3(z / scale) with the float32 scale A / 448; a block with A < 2^-100 as
// zero codes with scale 0.  A NaN in a block makes A and so the whole block
// NaN; an infinite A leaves zeros for the finite entries and NaN for the rest.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <cstdint>

namespace mdsoap {
namespace readout {

constexpr int kBlock = 128;
constexpr float kTop = 448.0f;      // largest e4m3 value
constexpr float kTiny = 0x1p-100f;  // blocks below it are zeros: 448 / A stays far inside float32

inline int64_t blocks_of(int64_t n) { return (n + kBlock - 1) / kBlock; }

// ------------------------------------------------------------ element types

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }

template <class T>
__device__ __forceinline__ T from_float(float x);
template <>
__device__ __forceinline__ float from_float<float>(float x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <>
__device__ __forceinline__ __half from_float<__half>(float x) { return __float2half_rn(x); }

// ------------------------------------------------------------ 16-byte units

// Elements of T in one 16-byte unit.
template <class T>
constexpr int kUnit = 16 / (int)sizeof(T);

// The two 16-bit elements of a word, and back (each rounded to nearest).
template <class T>
__device__ __forceinline__ float2 unpack2(uint32_t w);
template <>
__device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t w) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <>
__device__ __forceinline__ float2 unpack2<__half>(uint32_t w) {
    return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
template <class T>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
    const __nv_bfloat162 t = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&t);
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
    const __half2 t = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&t);
}

template <class T>
__device__ __forceinline__ void unpack(const uint4& u, float (&f)[kUnit<T>]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (sizeof(T) == 4) {
            f[i] = __uint_as_float(w[i]);
        } else {
            const float2 t = unpack2<T>(w[i]);
            f[2 * i] = t.x, f[2 * i + 1] = t.y;
        }
    }
}

template <class T>
__device__ __forceinline__ uint4 pack(const float (&f)[kUnit<T>]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (sizeof(T) == 4) w[i] = __float_as_uint(f[i]);
        else w[i] = pack2<T>(f[2 * i], f[2 * i + 1]);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// Bytes [shift, shift + 16) of the 32 bytes a, b; 0 < shift < 16, the same in
// all lanes of a warp.
__device__ __forceinline__ uint4 splice(const uint4& a, const uint4& b, int shift) {
    uint32_t w0, w1, w2, w3, w4;
    switch (shift >> 2) {
        case 0: w0 = a.x, w1 = a.y, w2 = a.z, w3 = a.w, w4 = b.x; break;
        case 1: w0 = a.y, w1 = a.z, w2 = a.w, w3 = b.x, w4 = b.y; break;
        case 2: w0 = a.z, w1 = a.w, w2 = b.x, w3 = b.y, w4 = b.z; break;
        default: w0 = a.w, w1 = b.x, w2 = b.y, w3 = b.z, w4 = b.w; break;
    }
    const int r = (shift & 3) * 8;
    return make_uint4(__funnelshift_r(w0, w1, r), __funnelshift_r(w1, w2, r), __funnelshift_r(w2, w3, r),
                      __funnelshift_r(w3, w4, r));
}

// A read-only matrix with unit column stride.  [begin, end) is the byte range
// its elements span: the two aligned words that hold a misaligned unit are
// only read where both lie inside it.
template <class T>
struct MatrixIn {
    const T* data;
    int64_t rows, width, stride;

    __device__ __forceinline__ uint4 unit(int64_t row, int64_t col) const {
        if (col >= width) return make_uint4(0, 0, 0, 0);
        const T* p = data + row * stride + col;
        if (col + kUnit<T> <= width) {
            const uintptr_t at = reinterpret_cast<uintptr_t>(p);
            const int shift = (int)(at & 15);
            if (shift == 0) return __ldg(reinterpret_cast<const uint4*>(p));
            const uintptr_t begin = reinterpret_cast<uintptr_t>(data);
            const uintptr_t end = reinterpret_cast<uintptr_t>(data + (rows - 1) * stride + width);
            const uintptr_t word = at - shift;
            if (word >= begin && word + 32 <= end) {
                const uint4* w = reinterpret_cast<const uint4*>(word);
                return splice(__ldg(w), __ldg(w + 1), shift);
            }
        }
        uint4 u = make_uint4(0, 0, 0, 0);
        T* t = reinterpret_cast<T*>(&u);
#pragma unroll
        for (int i = 0; i < kUnit<T>; ++i)
            if (col + i < width) t[i] = p[i];
        return u;
    }
};

// A row store of one unit per lane; the lanes of a warp hold consecutive units
// (lane l the elements col .. col + kUnit).  All 32 lanes call it together.
// Where the row is not 16-byte aligned, each lane joins its unit's head to its
// lower neighbour's tail and stores that aligned word; the two ends of the
// warp's stretch go out element by element.
template <class T>
__device__ __forceinline__ void store_unit(T* row, int64_t col, int64_t width, const uint4& u) {
    T* p = row + col;
    const int shift = (int)(reinterpret_cast<uintptr_t>(row) & 15);  // uniform: col is a multiple of the unit
    const T* t = reinterpret_cast<const T*>(&u);
    const bool full = col + kUnit<T> <= width;
    if (shift == 0) {
        if (full) {
            *reinterpret_cast<uint4*>(p) = u;
        } else {
#pragma unroll
            for (int i = 0; i < kUnit<T>; ++i)
                if (col + i < width) p[i] = t[i];
        }
        return;
    }
    uint4 below;
    below.x = __shfl_up_sync(0xffffffffu, u.x, 1);
    below.y = __shfl_up_sync(0xffffffffu, u.y, 1);
    below.z = __shfl_up_sync(0xffffffffu, u.z, 1);
    below.w = __shfl_up_sync(0xffffffffu, u.w, 1);
    const int lane = threadIdx.x & 31;
    const int head = (16 - shift) / (int)sizeof(T);  // elements of a unit below the next aligned word
    if (lane > 0 && col + head <= width) {
        // the aligned word ends `head` elements into this lane's unit
        *reinterpret_cast<uint4*>(p + head - kUnit<T>) = splice(below, u, 16 - shift);
    } else {
#pragma unroll
        for (int i = 0; i < kUnit<T>; ++i) {
            // head of this unit, and (when the word was cut off) the neighbour's tail
            if (i < head && col + i < width) p[i] = t[i];
        }
        if (lane > 0) {
            const T* b = reinterpret_cast<const T*>(&below);
#pragma unroll
            for (int i = 0; i < kUnit<T>; ++i)
                if (i >= head && col - kUnit<T> + i < width) p[i - kUnit<T>] = b[i];
        }
    }
    if (lane == 31) {
#pragma unroll
        for (int i = 0; i < kUnit<T>; ++i)
            if (i >= head && col + i < width) p[i] = t[i];
    }
}

// ------------------------------------------------------------ quads
//
// Four neighbouring elements a lane: a warp holds one block of 128 of a row.

template <class T>
struct Quad;  // the word that four elements fill
template <>
struct Quad<float> { using Word = uint4; };
template <>
struct Quad<__nv_bfloat16> { using Word = uint2; };
template <>
struct Quad<__half> { using Word = uint2; };

template <class T>
__device__ __forceinline__ float4 unpack4(const typename Quad<T>::Word& w) {
    if constexpr (sizeof(T) == 4) {
        return make_float4(__uint_as_float(w.x), __uint_as_float(w.y), __uint_as_float(w.z), __uint_as_float(w.w));
    } else {
        const float2 a = unpack2<T>(w.x), b = unpack2<T>(w.y);
        return make_float4(a.x, a.y, b.x, b.y);
    }
}

template <class T>
__device__ __forceinline__ typename Quad<T>::Word pack4(const float4& f) {
    if constexpr (sizeof(T) == 4)
        return make_uint4(__float_as_uint(f.x), __float_as_uint(f.y), __float_as_uint(f.z), __float_as_uint(f.w));
    else
        return make_uint2(pack2<T>(f.x, f.y), pack2<T>(f.z, f.w));
}

__device__ __forceinline__ uint2 splice(const uint2& a, const uint2& b, int shift) {
    const uint32_t w0 = shift < 4 ? a.x : a.y, w1 = shift < 4 ? a.y : b.x, w2 = shift < 4 ? b.x : b.y;
    const int r = (shift & 3) * 8;
    return make_uint2(__funnelshift_r(w0, w1, r), __funnelshift_r(w1, w2, r));
}

// Whether a row's quads can be read and written as words.
template <class T>
__device__ __forceinline__ bool quads_aligned(const T* row) {
    return reinterpret_cast<uintptr_t>(row) % sizeof(typename Quad<T>::Word) == 0;
}

// Elements col .. col + 3 of a row of any alignment, zero past `width`.
// [begin, end) is the byte range of the whole matrix: the two aligned words
// that hold a misaligned quad are only read where both lie inside it.
template <class T>
__device__ __forceinline__ typename Quad<T>::Word load_quad(const T* row, int64_t col, int64_t width, uintptr_t begin,
                                                            uintptr_t end) {
    using Word = typename Quad<T>::Word;
    const T* p = row + col;
    Word w{};
    if (col + 4 <= width) {
        const uintptr_t at = reinterpret_cast<uintptr_t>(p);
        const int shift = (int)(at % sizeof(Word));
        if (shift == 0) return __ldg(reinterpret_cast<const Word*>(p));
        const uintptr_t word = at - shift;
        if (word >= begin && word + 2 * sizeof(Word) <= end) {
            const Word* q = reinterpret_cast<const Word*>(word);
            return splice(__ldg(q), __ldg(q + 1), shift);
        }
    }
    T* t = reinterpret_cast<T*>(&w);
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (col + i < width) t[i] = p[i];
    return w;
}

// A misaligned quad whose two aligned words may be read.
template <class T>
__device__ __forceinline__ typename Quad<T>::Word load_split(const T* p) {
    using Word = typename Quad<T>::Word;
    const uintptr_t at = reinterpret_cast<uintptr_t>(p);
    const int shift = (int)(at % sizeof(Word));
    const Word* q = reinterpret_cast<const Word*>(at - shift);
    return shift == 0 ? __ldg(q) : splice(__ldg(q), __ldg(q + 1), shift);
}

__device__ __forceinline__ uint2 shuffle_up(const uint2& w) {
    return make_uint2(__shfl_up_sync(0xffffffffu, w.x, 1), __shfl_up_sync(0xffffffffu, w.y, 1));
}
__device__ __forceinline__ uint4 shuffle_up(const uint4& w) {
    return make_uint4(__shfl_up_sync(0xffffffffu, w.x, 1), __shfl_up_sync(0xffffffffu, w.y, 1),
                      __shfl_up_sync(0xffffffffu, w.z, 1), __shfl_up_sync(0xffffffffu, w.w, 1));
}

// One quad per lane of a row of any alignment; all 32 lanes, holding
// consecutive quads, call it together.  Where the row is not aligned to words,
// each lane joins its quad's head to its lower neighbour's tail and stores that
// aligned word; the two ends of the warp's stretch go out element by element.
template <class T>
__device__ __forceinline__ void store_quad(T* row, int64_t col, int64_t width, const typename Quad<T>::Word& w) {
    using Word = typename Quad<T>::Word;
    T* p = row + col;
    const int shift = (int)(reinterpret_cast<uintptr_t>(row) % sizeof(Word));  // col is a multiple of four
    const T* t = reinterpret_cast<const T*>(&w);
    if (shift == 0) {
        if (col + 4 <= width) {
            *reinterpret_cast<Word*>(p) = w;
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (col + i < width) p[i] = t[i];
        }
        return;
    }
    const Word below = shuffle_up(w);
    const int lane = threadIdx.x & 31;
    const int head = ((int)sizeof(Word) - shift) / (int)sizeof(T);  // elements of a quad below the next aligned word
    if (lane > 0 && col + head <= width) {
        *reinterpret_cast<Word*>(p + head - 4) = splice(below, w, (int)sizeof(Word) - shift);
    } else {
        const T* b = reinterpret_cast<const T*>(&below);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (i < head && col + i < width) p[i] = t[i];
            if (lane > 0 && i >= head && col - 4 + i < width) p[i - 4] = b[i];
        }
    }
    if (lane == 31) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (i >= head && col + i < width) p[i] = t[i];
    }
}

// kUnit<T> float32 values of a vector from `col` on; zero past `width`.
template <int N>
__device__ __forceinline__ void load_vector(const float* v, int64_t col, int64_t width, float (&f)[N]) {
    const float* p = v + col;
    if (col + N <= width && (reinterpret_cast<uintptr_t>(p) & 15) == 0) {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const float4 q = __ldg(reinterpret_cast<const float4*>(p + i));
            f[i] = q.x, f[i + 1] = q.y, f[i + 2] = q.z, f[i + 3] = q.w;
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = col + i < width ? __ldg(p + i) : 0.0f;
}

// ------------------------------------------------------------ blocks of 128

// |x| as an unsigned whose order is the magnitudes' with NaN on top.
__device__ __forceinline__ uint32_t magnitude(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// The larger magnitude; NaN if one is.
__device__ __forceinline__ float larger(float most, float x) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(most), "f"(fabsf(x)));
    return r;
}
__device__ __forceinline__ float larger(float a, float b, float c) {
    float r;
    asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
// The largest of the warp's magnitudes.
__device__ __forceinline__ float warp_larger(float most) {
    float r;
    asm("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(most));
    return r;
}

__device__ __forceinline__ float reciprocal(float x) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// A block's scale; the constant is the rounded reciprocal of 448.
__device__ __forceinline__ float scale_of(float top) { return top < kTiny ? 0.0f : __fmul_rn(top, 1.0f / kTop); }

// z / scale for the entries of a block with the maximum `top`: the quick
// reciprocal's product with one correction by its exact remainder, which leaves
// the correctly rounded quotient but for about one entry in a million.  Zero in
// a block that is stored as zeros, and for the finite entries beside an
// infinite one.
struct Factor {
    float inverse, scale;
    __device__ __forceinline__ explicit Factor(float top) {
        scale = scale_of(top);
        inverse = reciprocal(scale);
        if (top < kTiny || top == INFINITY) inverse = scale = 0.0f;
    }
    __device__ __forceinline__ float operator()(float z) const {
        const float q = z * inverse;
        return fmaf(fmaf(-q, scale, z), inverse, q);
    }
    // the same for x f and y f' (the factors as a pair), in packed arithmetic
    __device__ __forceinline__ void pair(float x, float y, uint64_t f, float& q, float& r) const {
        asm("{\n\t.reg .b64 z, n, i, q;\n\t"
            "mov.b64 z, {%2, %3};\n\tmov.b64 i, {%5, %5};\n\tmov.b64 n, {%6, %6};\n\t"
            "mul.rn.f32x2 z, z, %4;\n\t"
            "mul.rn.f32x2 q, z, i;\n\t"
            "fma.rn.f32x2 z, q, n, z;\n\t"
            "fma.rn.f32x2 q, z, i, q;\n\t"
            "mov.b64 {%0, %1}, q;\n\t}"
            : "=f"(q), "=f"(r)
            : "f"(x), "f"(y), "l"(f), "f"(inverse), "f"(-scale));
    }
};

// Two e4m3 codes, `a` in the low byte.
__device__ __forceinline__ uint32_t codes2(float a, float b) {
    return __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
}

__device__ __forceinline__ uint32_t codes4(float a, float b, float c, float d) {
    return codes2(a, b) | codes2(c, d) << 16;
}

__device__ __forceinline__ float warp_sum(float x) {
#pragma unroll
    for (int d = 16; d; d >>= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
    return x;
}

}  // namespace readout
}  // namespace mdsoap
