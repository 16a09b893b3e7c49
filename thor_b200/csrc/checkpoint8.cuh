// 8-bit activation checkpoints: the device side of their format, shared by every kernel that writes or reads one.
//
// A block is 32 neighbouring columns of one row.  Its scale is the smallest power of two s with max|x| <= s * M, M the
// largest code (448 for e4m3, 57344 for e5m2, 127 for int8), stored as the byte log2(s) + 127 (e8m0); a code is x / s
// rounded to nearest even.  Division and multiplication by a power of two are exact, so pack / unpack have exactly one rounding, and a block that is
// packed again from its own unpacked form stands for the same values (maybe by other codes: 450 packs as 224 with s = 2, and the 448 it unpacks to as 448
// with s = 1).  s is clamped at 2^-127 from below (an
// all-zero block has that scale).  A block that holds an infinity or a NaN has the scale byte 255 and codes zero, and
// unpacks as NaN throughout: an overflow stays visible in the backward pass.
//
// A thread holds sixteen neighbouring columns (32 bytes of a 16-bit tensor, one 16-byte word of codes), so two neighbouring lanes
// hold a block.
#pragma once

#include <type_traits>

#include "common.cuh"

namespace tb {
namespace ck8 {

constexpr int kBlock = 32;  // columns of a block
constexpr int kVec = 16;    // columns of a thread

__host__ __device__ inline uint64_t codePitch(uint64_t cols) { return (cols + 15) / 16 * 16; }
__host__ __device__ inline uint64_t scalePitch(uint64_t cols) { return (cols + kBlock - 1) / kBlock; }

inline bool codeDtypeOk(int dt) { return dt == THOR_B200_FP8_E4M3 || dt == THOR_B200_FP8_E5M2 || dt == THOR_B200_INT8; }
inline bool valueDtypeOk(int dt) { return dt == THOR_B200_FP32 || dt == THOR_B200_FP16 || dt == THOR_B200_BF16; }

// ---- two fp32 values in one instruction ------------------------------------------------------------------
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 r;
    asm("{\n\t.reg .b64 a, b, c;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\tfma.rn.f32x2 a, a, b, c;\n\tmov.b64 {%0, %1}, a;\n\t}"
        : "=f"(r.x), "=f"(r.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return r;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 r;
    asm("{\n\t.reg .b64 a, b;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmul.rn.f32x2 a, a, b;\n\tmov.b64 {%0, %1}, a;\n\t}"
        : "=f"(r.x), "=f"(r.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return r;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 r;
    asm("{\n\t.reg .b64 a, b;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tadd.rn.f32x2 a, a, b;\n\tmov.b64 {%0, %1}, a;\n\t}"
        : "=f"(r.x), "=f"(r.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return r;
}
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }
__device__ __forceinline__ float exp2Approx(float v) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
__device__ __forceinline__ float reciprocalApprox(float v) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}

// ---- scales and codes ---------------------------------------------------------------------------------------
// max(m, |a|, |b|), NaN if one of them is NaN
__device__ __forceinline__ float maxAbs3(float m, float a, float b) {
    float r;
    asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(m), "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float maxAbs16(const float2 (&v)[8]) {
    float m = maxAbs3(0.0f, v[0].x, v[0].y), n = maxAbs3(0.0f, v[4].x, v[4].y);
#pragma unroll
    for (int i = 1; i < 4; ++i) {
        m = maxAbs3(m, v[i].x, v[i].y);
        n = maxAbs3(n, v[i + 4].x, v[i + 4].y);
    }
    return maxAbs3(0.0f, m, n);
}
// over the two lanes of a block; all 32 lanes take part
__device__ __forceinline__ float blockMax(float m) { return maxAbs3(0.0f, m, __shfl_xor_sync(0xffffffffu, m, 1)); }

// Scale byte of a block with largest magnitude `amax`: the exponent field, plus one where the significand is above that of
// M (the addition carries exactly then), less the exponent of M.
__device__ __forceinline__ uint32_t scaleByte(float amax, int code) {
    const uint32_t bits = __float_as_uint(amax);
    const uint32_t carry = code == THOR_B200_INT8 ? 0x7fffffu - 0x7e0000u : 0x7fffffu - 0x600000u;  // 127 = 1.984375 * 2^6, 448 and 57344 = 1.75 * 2^n
    const int exponent = code == THOR_B200_INT8 ? 6 : (code == THOR_B200_FP8_E4M3 ? 8 : 15);
    const int byte = max(static_cast<int>((bits + carry) >> 23) - exponent, 0);
    return bits >= 0x7f800000u ? 255u : static_cast<uint32_t>(byte);
}
// FINITE, for gradients: a magnitude within half a step of 2^128 (a type's lowest number, as masks write it) has the code of 2^128, an infinity in fp32, and an
// infinity times a slope or a gradient of zero would be NaN.  Scales that reach so far (from 2^113 on) are one unit in the last place smaller there, so
// that 2^128 becomes the largest number.
template <bool FINITE = false>
__device__ __forceinline__ float scaleValue(uint32_t byte) {
    const uint32_t power = FINITE ? (byte << 23) - (byte >= 240u ? 1u : 0u) : byte << 23;
    return __uint_as_float(byte == 0 ? 0x00400000u : (byte == 255u ? 0x7fc00000u : power));
}

template <int CODE>
__device__ __forceinline__ uint32_t pack4(float2 a, float2 b) {
    if constexpr (CODE == THOR_B200_INT8) {
        // adding 1.5 * 2^23 rounds to an integer (to nearest even) and leaves it in the low bits in two's complement
        const float2 magic = both(12582912.0f);
        a = add2(a, magic);
        b = add2(b, magic);
        return __byte_perm(__byte_perm(__float_as_uint(a.x), __float_as_uint(a.y), 0x0040), __byte_perm(__float_as_uint(b.x), __float_as_uint(b.y), 0x0040), 0x5410);
    } else {
        uint16_t lo, hi;
        if constexpr (CODE == THOR_B200_FP8_E4M3) {
            asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(a.y), "f"(a.x));
            asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(b.y), "f"(b.x));
        } else {
            asm("cvt.rn.satfinite.e5m2x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(a.y), "f"(a.x));
            asm("cvt.rn.satfinite.e5m2x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(b.y), "f"(b.x));
        }
        return static_cast<uint32_t>(lo) | (static_cast<uint32_t>(hi) << 16);
    }
}
template <int CODE>
__device__ __forceinline__ uint4 encodeAs(const float2 (&v)[8], float2 inv) {
    return make_uint4(pack4<CODE>(mul2(v[0], inv), mul2(v[1], inv)), pack4<CODE>(mul2(v[2], inv), mul2(v[3], inv)), pack4<CODE>(mul2(v[4], inv), mul2(v[5], inv)),
                      pack4<CODE>(mul2(v[6], inv), mul2(v[7], inv)));
}
// Codes of sixteen values of a block with scale byte `byte`.
__device__ __forceinline__ uint4 encode16(const float2 (&v)[8], uint32_t byte, int code) {
    if (byte == 255u) return make_uint4(0u, 0u, 0u, 0u);
    const float2 inv = both(__uint_as_float((254u - byte) << 23));  // 2^(127 - byte); byte <= 249 here
    if (code == THOR_B200_FP8_E4M3) return encodeAs<THOR_B200_FP8_E4M3>(v, inv);
    return code == THOR_B200_INT8 ? encodeAs<THOR_B200_INT8>(v, inv) : encodeAs<THOR_B200_FP8_E5M2>(v, inv);
}

template <int CODE>
__device__ __forceinline__ void unpack4(uint32_t c, float2& a, float2& b) {
    if constexpr (CODE == THOR_B200_INT8) {
        // byte + 128 in the low bits of 2^23 is the float 2^23 + 128 + value; both steps are exact
        const uint32_t u = c ^ 0x80808080u;
        const float2 off = both(-8388736.0f);
        a = make_float2(__uint_as_float(__byte_perm(u, 0x4b000000u, 0x7440)), __uint_as_float(__byte_perm(u, 0x4b000000u, 0x7441)));
        b = make_float2(__uint_as_float(__byte_perm(u, 0x4b000000u, 0x7442)), __uint_as_float(__byte_perm(u, 0x4b000000u, 0x7443)));
        a = add2(a, off);
        b = add2(b, off);
    } else {
        uint32_t lo, hi;
        if constexpr (CODE == THOR_B200_FP8_E4M3) {
            asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(lo) : "h"(static_cast<uint16_t>(c)));
            asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(hi) : "h"(static_cast<uint16_t>(c >> 16)));
        } else {  // an e5m2 code is the upper byte of the fp16 number of the same value
            lo = __byte_perm(c, 0u, 0x1404);
            hi = __byte_perm(c, 0u, 0x3424);
        }
        a = __half22float2(*reinterpret_cast<const __half2*>(&lo));
        b = __half22float2(*reinterpret_cast<const __half2*>(&hi));
    }
}
template <int CODE>
__device__ __forceinline__ void numbersAs(uint4 c, float2 (&v)[8]) {
    unpack4<CODE>(c.x, v[0], v[1]);
    unpack4<CODE>(c.y, v[2], v[3]);
    unpack4<CODE>(c.z, v[4], v[5]);
    unpack4<CODE>(c.w, v[6], v[7]);
}
// The numbers that codes stand for before they are scaled.
__device__ __forceinline__ void numbers16(uint4 c, int code, float2 (&v)[8]) {
    if (code == THOR_B200_FP8_E4M3) numbersAs<THOR_B200_FP8_E4M3>(c, v);
    else if (code == THOR_B200_INT8) numbersAs<THOR_B200_INT8>(c, v);
    else numbersAs<THOR_B200_FP8_E5M2>(c, v);
}
template <bool FINITE>
__device__ __forceinline__ void decode16(uint4 c, uint32_t byte, int code, float2 (&v)[8]) {
    const float2 s = both(scaleValue<FINITE>(byte));
    numbers16(c, code, v);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = mul2(v[i], s);
}

// ---- sixteen neighbouring elements of a row ---------------------------------------------------------------
__device__ __forceinline__ float2 widen(uint32_t w, __half) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
// a bf16 number is the upper half of the fp32 number of the same value
__device__ __forceinline__ float2 widen(uint32_t w, __nv_bfloat16) { return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)); }
__device__ __forceinline__ uint32_t narrow(float2 v, __half) {
    const __half2 h = __floats2half2_rn(v.x, v.y);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t narrow(float2 v, __nv_bfloat16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(v.x, v.y);
    return *reinterpret_cast<const uint32_t*>(&h);
}
// Sixteen elements as 32-bit words: 8 of a 16-bit type, 16 of fp32.
template <class T>
constexpr int kRegs = 4 * static_cast<int>(sizeof(T));
template <class T>
__device__ __forceinline__ void widen16(const uint32_t (&w)[kRegs<T>], float2 (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        if constexpr (sizeof(T) == 4) v[i] = make_float2(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
        else v[i] = widen(w[i], T{});
    }
}
template <class T>
__device__ __forceinline__ void narrow16(const float2 (&v)[8], uint32_t (&w)[kRegs<T>]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        if constexpr (sizeof(T) == 4) {
            w[2 * i] = __float_as_uint(v[i].x);
            w[2 * i + 1] = __float_as_uint(v[i].y);
        } else {
            w[i] = narrow(v[i], T{});
        }
    }
}

// Where a row starts: the product passes 32 bits, its factors do not.
__device__ __forceinline__ uint64_t rowStart(uint32_t row, uint32_t stride) { return static_cast<uint64_t>(row) * stride; }

// Rows of a tensor that is read.
template <class T>
struct Rows {
    const T* p;
    uint32_t stride;  // elements between rows
    const void* end;  // one past the last element
};

// What a thread has loaded of a row.  ALIGNED: rows start on 32 bytes and have a multiple of 16 columns, so sixteen columns are whole or absent
// and are the words themselves.  Otherwise: the words of eight elements that contain the sixteen elements, one more than they fill.
template <class T, bool ALIGNED>
struct Raw {
    uint32_t w[ALIGNED ? kRegs<T> : kRegs<T> / 2 * 3];
};

// A word that reaches over the tensor's first or last byte, element by element.
template <class T>
__device__ __noinline__ uint4 edgeWord(const char* word, const void* begin, const void* end) {
    constexpr int per = 4 / sizeof(T);
    uint32_t r[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        r[i] = 0;
#pragma unroll
        for (int j = 0; j < per; ++j) {
            const char* e = word + 4 * i + j * sizeof(T);
            if (e >= begin && e < end) {
                if constexpr (per == 1) r[i] = *reinterpret_cast<const uint32_t*>(e);
                else r[i] |= static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(e)) << (16 * j);
            }
        }
    }
    return make_uint4(r[0], r[1], r[2], r[3]);
}

// Columns col .. col + 15 of a row of `cols`; p points at the first of them.
template <class T, bool ALIGNED>
__device__ __forceinline__ void fetch16(const Rows<T>& in, const T* p, uint32_t col, uint32_t cols, Raw<T, ALIGNED>& raw) {
    constexpr int W = kRegs<T> / 2, words = ALIGNED ? 2 : 3;  // registers of a word of eight elements, words
#pragma unroll
    for (int i = 0; i < W * words; ++i) raw.w[i] = 0;
    if (col >= cols) return;
    auto put = [&](int i, const uint4& q) { raw.w[i] = q.x, raw.w[i + 1] = q.y, raw.w[i + 2] = q.z, raw.w[i + 3] = q.w; };
    if constexpr (ALIGNED) {
#pragma unroll
        for (int i = 0; i < W * words; i += 8) {
            uint4 lo, hi;
            load256(lo, hi, reinterpret_cast<const uint32_t*>(p) + i);
            put(i, lo);
            put(i + 4, hi);
        }
    } else {
        constexpr int bytes = 4 * W;
        const char* const word0 = reinterpret_cast<const char*>(reinterpret_cast<uintptr_t>(p) & ~static_cast<uintptr_t>(bytes - 1));
        const char* const last = reinterpret_cast<const char*>(p + min(16u, cols - col));
        if (word0 >= reinterpret_cast<const char*>(in.p) && word0 + bytes * words <= in.end) {
#pragma unroll
            for (int i = 0; i < words; ++i) {
                if (i + 1 < words || word0 + bytes * i < last) {  // the last word is the neighbouring lane's first: L1 keeps it
                    if constexpr (W == 4) {
                        put(4 * i, __ldg(reinterpret_cast<const uint4*>(word0) + i));
                    } else {
                        uint4 lo, hi;
                        asm volatile("ld.global.nc.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                                     : "=r"(lo.x), "=r"(lo.y), "=r"(lo.z), "=r"(lo.w), "=r"(hi.x), "=r"(hi.y), "=r"(hi.z), "=r"(hi.w)
                                     : "l"(word0 + bytes * i));
                        put(8 * i, lo);
                        put(8 * i + 4, hi);
                    }
                }
            }
        } else {  // at the tensor's first or last byte
#pragma unroll
            for (int i = 0; i < W * words; i += 4)
                if (word0 + 4 * i < last) put(i, edgeWord<T>(word0 + 4 * i, in.p, in.end));
        }
    }
}

// Calls f with m as an integral constant, m elements past a word of eight elements.  Every row has one m, so a warp of one or two rows takes one or two of the
// branches, and each of them moves whole registers (and shifts pairs by half a register where m is odd) instead of selecting by m.  Rows of fewer than 256 columns put 3 to
// 16 rows into a warp, which then takes up to eight branches: bf16 [1000000, 33] pack 44 us, unpack 89, GELU 126 each way, LayerNorm 147 and 174, 0.15 to 0.35 of the
// copy rate; [262144, 97] 0.28 to 0.55; [60000, 333] 0.32 to 0.67.
template <class T, class F>
__device__ __forceinline__ void byOffset(const void* p, F&& f) {
    switch ((static_cast<uint32_t>(reinterpret_cast<uintptr_t>(p)) / sizeof(T)) % 8) {
        case 0: f(std::integral_constant<int, 0>{}); break;
        case 1: f(std::integral_constant<int, 1>{}); break;
        case 2: f(std::integral_constant<int, 2>{}); break;
        case 3: f(std::integral_constant<int, 3>{}); break;
        case 4: f(std::integral_constant<int, 4>{}); break;
        case 5: f(std::integral_constant<int, 5>{}); break;
        case 6: f(std::integral_constant<int, 6>{}); break;
        default: f(std::integral_constant<int, 7>{});
    }
}
// 32-bit word that starts at element `e` of a run of words
template <class T, int N>
__device__ __forceinline__ uint32_t wordAt(const uint32_t (&r)[N], int e) {
    if constexpr (sizeof(T) == 4) return r[e];
    else return e % 2 == 0 ? r[e / 2] : __funnelshift_r(r[e / 2], r[e / 2 + 1], 16);
}

// Calls f with m as an integral constant below N; where m is the same for a whole warp it takes one branch.
template <int N, class F>
__device__ __forceinline__ void byConstant(uint32_t m, F&& f) {
    if constexpr (N == 1) {
        f(std::integral_constant<int, 0>{});
    } else {
        if (m < N / 2) byConstant<N / 2>(m, f);
        else byConstant<N - N / 2>(m - N / 2, [&](auto i) { f(std::integral_constant<int, decltype(i)::value + N / 2>{}); });
    }
}
// Zeroes the columns past the row's end, in the lane that holds it; its place is the same in every row, so by constants (LayerNorm forward [20000, 333] bf16
// 16.5 -> 14.5 us against comparing each column).
__device__ __forceinline__ void cutRow(uint32_t col, uint32_t cols, float2 (&v)[8]) {
    if (col < cols && col + 16 > cols) {
        byConstant<16>(cols - col, [&](auto n) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if (2 * i >= decltype(n)::value) v[i].x = 0.0f;
                if (2 * i + 1 >= decltype(n)::value) v[i].y = 0.0f;
            }
        });
    }
}

// The words from element m on, by selection: for warps whose lanes hold many rows, each with an m of its own.
template <class T>
__device__ __forceinline__ void selectWords(const uint32_t (&raw)[kRegs<T> / 2 * 3], uint32_t m, uint32_t (&w)[kRegs<T>]) {
    constexpr int W = kRegs<T> / 2, N = kRegs<T>;
    uint32_t r[W * 3];
#pragma unroll
    for (int i = 0; i < W * 3; ++i) r[i] = raw[i];
#pragma unroll
    for (int s = W / 2; s >= 1; s /= 2) {  // shift by s registers where m asks for it; what a later shift needs is kept
#pragma unroll
        for (int i = 0; i + s < W * 3; ++i) r[i] = (m * sizeof(T) / 4) & s ? r[i + s] : r[i];
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
        if constexpr (sizeof(T) == 4) w[i] = r[i];
        else w[i] = __funnelshift_r(r[i], r[i + 1], (m % 2) * 16);
    }
}

// The sixteen values that fetch16 of the same arguments has loaded; zero past the row's end.  MIXED: the lanes of a warp hold many rows.
template <class T, bool ALIGNED, bool MIXED = false>
__device__ __forceinline__ void expand16(const T* p, uint32_t col, uint32_t cols, const Raw<T, ALIGNED>& raw, float2 (&v)[8]) {
    if constexpr (ALIGNED) {
        widen16<T>(raw.w, v);
    } else {
        uint32_t w[kRegs<T>];
        if constexpr (MIXED) {
            selectWords<T>(raw.w, (static_cast<uint32_t>(reinterpret_cast<uintptr_t>(p)) / sizeof(T)) % 8, w);
        } else {
            byOffset<T>(p, [&](auto m) {
#pragma unroll
                for (int i = 0; i < kRegs<T>; ++i) w[i] = wordAt<T>(raw.w, decltype(m)::value + i * static_cast<int>(4 / sizeof(T)));
            });
        }
        widen16<T>(w, v);
        cutRow(col, cols, v);
    }
}
template <bool ALIGNED, class T>
__device__ __forceinline__ void load16(const Rows<T>& in, const T* p, uint32_t col, uint32_t cols, float2 (&v)[8]) {
    Raw<T, ALIGNED> raw;
    fetch16(in, p, col, cols, raw);
    expand16(p, col, cols, raw, v);
}

__device__ __forceinline__ void store256(void* to, const uint32_t* w) {
    asm volatile("st.global.cs.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(to), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7]) : "memory");
}

// Writes sixteen values to columns col .. of a row of `cols`, from p on; a lane with cols = 0 writes nothing.  All 32 lanes call it.
// Not ALIGNED: a lane writes the words of eight elements (32 bytes of fp32, 16 of a 16-bit type) that start in its range, the first of them with the
// last elements of the lane before it; `before` / `after`: that lane / the lane behind holds the sixteen columns before / behind these.  Where a
// neighbour is missing its part is left out, and what is left is written in smaller pieces; words that reach over the row's end are
// written element by element.  (32-byte words of 16-bit types take twice the exchanges and cases: unpack [8192, 8191] bf16, when it stored its rows this way, 46.6 us
// against 42; 16-byte words of fp32 leave half a sector to every store: unpack [4096, 2999] 15.3 us against 9.5.)
template <bool ALIGNED, class T>
__device__ __forceinline__ void store16(T* p, uint32_t col, uint32_t cols, const float2 (&v)[8], bool before, bool after) {
    constexpr int N = kRegs<T>;
    uint32_t own[N];
    narrow16<T>(v, own);
    if constexpr (ALIGNED) {
        if (col >= cols) return;
#pragma unroll
        for (int i = 0; i < N; i += 8) store256(reinterpret_cast<uint32_t*>(p) + i, own + i);
    } else {
        constexpr int E = 8, PER = 4 / sizeof(T), W = E / PER;  // elements of a word, elements of a register, registers of a word
        uint32_t run[W + N];                                    // the lane before's last word and these
#pragma unroll
        for (int i = 0; i < W; ++i) run[i] = __shfl_up_sync(0xffffffffu, own[N - W + i], 1);
#pragma unroll
        for (int i = 0; i < N; ++i) run[W + i] = own[i];
        if (col >= cols) return;
        const int left = static_cast<int>(min(cols - col, 1u << 20));  // elements up to the row's end
        byOffset<T>(p, [&](auto offset) {
            constexpr int m = decltype(offset)::value;  // elements of the first word that belong to the lane before
            auto element = [&](int e, uint32_t w) {     // e counted from p; the element is the low part of w
                if constexpr (sizeof(T) == 4) reinterpret_cast<uint32_t*>(p)[e] = w;
                else reinterpret_cast<uint16_t*>(p)[e] = static_cast<uint16_t>(w);
            };
#pragma unroll
            for (int k = 0; k < N / W; ++k) {
                const int first = k * E - m;  // of the word
                uint32_t r[W];
#pragma unroll
                for (int j = 0; j < W; ++j) r[j] = wordAt<T>(run, E + first + j * PER);
                if (first + E > left) {
#pragma unroll
                    for (int e = 0; e < E; ++e)
                        if (first + e < left && (first + e >= 0 || before)) element(first + e, PER == 1 ? r[e % W] : r[e / 2] >> (16 * (e % 2)));
                } else if (k > 0 || m == 0 || before) {
                    if constexpr (W == 8) store256(p + first, r);
                    else __stcs(reinterpret_cast<uint4*>(p + first), make_uint4(r[0], r[1], r[2], r[3]));
                } else {  // from element m of the word on
                    if constexpr (PER == 2 && m % 2 == 1) element(0, r[m / 2] >> 16);
                    constexpr int one = (m + PER - 1) / PER, two = (one + 1) / 2 * 2, four = (two + 3) / 4 * 4;  // first whole register, pair, four
                    uint32_t* const to = reinterpret_cast<uint32_t*>(p + first);
                    if constexpr (one % 2 == 1) to[one] = r[one];
                    if constexpr (two % 4 == 2) *reinterpret_cast<uint2*>(to + two) = make_uint2(r[two], r[two + 1]);
                    if constexpr (four + 4 <= W) *reinterpret_cast<uint4*>(to + four) = make_uint4(r[four], r[four + 1], r[four + 2], r[four + 3]);
                }
            }
            if (m > 0 && left > 16 - m && !(after && left > 16)) {  // the last m elements have no lane behind to write them
                if (left >= 16) {
                    uint32_t* const to = reinterpret_cast<uint32_t*>(p + 16 - m);  // on a word
                    auto reg = [&](int j) { return wordAt<T>(run, E + 16 - m + j * PER); };
                    constexpr int n = m / PER;  // whole registers
                    if constexpr (n >= 4) *reinterpret_cast<uint4*>(to) = make_uint4(reg(0), reg(1), reg(2), reg(3));
                    if constexpr (n % 4 >= 2) *reinterpret_cast<uint2*>(to + n / 4 * 4) = make_uint2(reg(n / 4 * 4), reg(n / 4 * 4 + 1));
                    if constexpr (n % 2 == 1) to[n - 1] = reg(n - 1);
                    if constexpr (PER == 2 && m % 2 == 1) element(15, own[N - 1] >> 16);
                } else {
#pragma unroll
                    for (int e = 16 - m; e < 16; ++e)
                        if (e < left) element(e, PER == 1 ? own[e] : own[e / 2] >> (16 * (e % 2)));
                }
            }
        });
    }
}
// Rounds sixteen values to T and back: what a reader of the stored tensor sees.
template <class T>
__device__ __forceinline__ void roundTo16(float2 (&v)[8]) {
    if constexpr (sizeof(T) < 4) {
        uint32_t w[kRegs<T>];
        narrow16<T>(v, w);
        widen16<T>(w, v);
    }
}

// ---- a checkpoint's rows ------------------------------------------------------------------------------------
struct Writer {
    uint8_t* codes;
    uint8_t* scales;
    uint32_t code_pitch, scale_pitch;
    int code;
};
struct Reader {
    const uint8_t* codes;
    const uint8_t* scales;
    uint32_t code_pitch, scale_pitch;
    int code;
};

__device__ __forceinline__ uint8_t* codesAt(const Writer& w, uint32_t row, uint32_t col) { return w.codes + rowStart(row, w.code_pitch) + col; }
__device__ __forceinline__ uint8_t* scaleAt(const Writer& w, uint32_t row, uint32_t col) { return w.scales + rowStart(row, w.scale_pitch) + col / kBlock; }

// Sixteen columns of one row by every lane, zero past the row's end; lanes 2 k and 2 k + 1 hold one block.  All 32 lanes call it, with cols = 0
// where a lane has no row.
__device__ __forceinline__ void writeCodes(uint8_t* codes, uint8_t* scale, int code, uint32_t col, uint32_t cols, const float2 (&v)[8]) {
    const uint32_t byte = scaleByte(blockMax(maxAbs16(v)), code);
    if (col >= cols) return;
    __stcs(reinterpret_cast<uint4*>(codes), encode16(v, byte, code));  // the pitch is a multiple of 16
    if (col % kBlock == 0) *scale = static_cast<uint8_t>(byte);
}
struct RawCodes {
    uint4 codes;
    uint32_t scale;
};
__device__ __forceinline__ const uint8_t* codesAt(const Reader& r, uint32_t row, uint32_t col) { return r.codes + rowStart(row, r.code_pitch) + col; }
__device__ __forceinline__ const uint8_t* scaleAt(const Reader& r, uint32_t row, uint32_t col) { return r.scales + rowStart(row, r.scale_pitch) + col / kBlock; }
__device__ __forceinline__ void fetchCodes(const uint8_t* codes, const uint8_t* scale, uint32_t col, uint32_t cols, RawCodes& raw) {
    raw.codes = make_uint4(0u, 0u, 0u, 0u);
    raw.scale = 0;
    if (col >= cols) return;
    raw.codes = __ldcs(reinterpret_cast<const uint4*>(codes));
    raw.scale = __ldg(scale);
}
// CUT: the padding behind the row's end is made zero whatever the block's scale.
template <bool CUT, bool FINITE = false>
__device__ __forceinline__ void expandCodes(int code, uint32_t col, uint32_t cols, const RawCodes& raw, float2 (&v)[8]) {
    decode16<FINITE>(raw.codes, raw.scale, code, v);
    if constexpr (CUT) cutRow(col, cols, v);
}

// ---- odd rows, walked on the tensor's own 32 bytes ---------------------------------------------------------
// For kernels that read a checkpoint and write a tensor element by element: a thread takes the sixteen columns from 16 u - m on, m the elements by which
// the row starts past 32 bytes, so that the tensor's words are whole and what has to be shifted are the codes, a quarter or an eighth of the bytes.
// Elements before m come from the code word u - 1, the others from word u; m is the same for the whole CTA.
// Against shifting the tensors' words: unpack [8192, 8191] bf16 42.0 -> 34.8 us, gated Swish backward 109.5 -> 89.8, GELU backward 66.0 -> 60.8, [2999, 11001]
// fp16 37.6 -> 31.1 and [8000, 5001] fp32 69.0 -> 54.0.
template <class T>
constexpr uint32_t kShifts = 32 / sizeof(T);

struct Place {
    uint32_t first, m, cols;  // columns first - m ..
    __device__ __forceinline__ bool whole() const { return first >= m && first - m + 16 <= cols; }
    __device__ __forceinline__ bool holds(uint32_t i) const { return first + i >= m && first + i - m < cols; }
};
template <class T>
__device__ __forceinline__ Place placeOf(const T* row, uint32_t cols) {
    return Place{(blockIdx.x * blockDim.x + threadIdx.x) * kVec, static_cast<uint32_t>(reinterpret_cast<uintptr_t>(row) / sizeof(T)) % kShifts<T>, cols};
}
template <class T>
__device__ __forceinline__ T* at(const Place& q, T* row) {
    return row + (static_cast<int64_t>(q.first) - q.m);
}
template <class T>
__device__ __forceinline__ void loadPlace(const Place& q, const Rows<T>& in, const T* row, uint32_t (&w)[kRegs<T>]) {
    const T* const p = at(q, row);
    if (p >= in.p && static_cast<const void*>(p + 16) <= in.end) {  // what lies beside the row's columns is the tensor's, too, and not stored
#pragma unroll
        for (int i = 0; i < kRegs<T>; i += 8) {
            uint4 lo, hi;
            load256(lo, hi, reinterpret_cast<const uint32_t*>(p) + i);
            w[i] = lo.x, w[i + 1] = lo.y, w[i + 2] = lo.z, w[i + 3] = lo.w;
            w[i + 4] = hi.x, w[i + 5] = hi.y, w[i + 6] = hi.z, w[i + 7] = hi.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < kRegs<T>; i += 4) {
            const uint4 u = edgeWord<T>(reinterpret_cast<const char*>(p) + 4 * i, in.p, in.end);
            w[i] = u.x, w[i + 1] = u.y, w[i + 2] = u.z, w[i + 3] = u.w;
        }
    }
}
template <class T>
__device__ __forceinline__ void storePlace(const Place& q, T* row, const float2 (&v)[8]) {
    T* const p = at(q, row);
    uint32_t w[kRegs<T>];
    narrow16<T>(v, w);
    if (q.whole()) {
#pragma unroll
        for (int i = 0; i < kRegs<T>; i += 8) store256(reinterpret_cast<uint32_t*>(p) + i, w + i);
    } else if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 16; ++i)
            if (q.holds(i)) reinterpret_cast<uint32_t*>(p)[i] = w[i];
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const bool low = q.holds(2 * i), high = q.holds(2 * i + 1);
            if (low && high) reinterpret_cast<uint32_t*>(p)[i] = w[i];
            else if (low) reinterpret_cast<uint16_t*>(p)[2 * i] = static_cast<uint16_t>(w[i]);
            else if (high) reinterpret_cast<uint16_t*>(p)[2 * i + 1] = static_cast<uint16_t>(w[i] >> 16);
        }
    }
}
// The code words that a place needs and their scale bytes; m = 0 needs one.
struct PlaceCodes {
    uint4 a, b;
    uint32_t scale_a, scale_b;
};
__device__ __forceinline__ PlaceCodes fetchPlace(const Reader& in, const Place& q, uint32_t row) {
    PlaceCodes c{};
    const uint8_t* const codes = codesAt(in, row, 0);
    const uint8_t* const scales = scaleAt(in, row, 0);
    if (q.first > 0 && q.m > 0) {
        c.a = __ldg(reinterpret_cast<const uint4*>(codes + q.first) - 1);  // the neighbouring lane's, too: L1 keeps it
        c.scale_a = __ldg(scales + (q.first - 16) / kBlock);
    }
    if (q.first < q.cols) {
        c.b = __ldg(reinterpret_cast<const uint4*>(codes + q.first));
        c.scale_b = __ldg(scales + q.first / kBlock);
    }
    return c;
}
// The sixteen values of a place.  Which byte goes where and which scale it takes hang on m alone: constants in each of the branches.  ONCE: the
// branches hold the conversion of the codes, too (48 of them); otherwise only the shift and, once more, the scaling.  Once is the faster form (GELU backward
// [8192, 8191] bf16 60.8 us against 67.3; with selects by m instead of branches 69.7), except in 16-bit gated kernels, whose two expansions
// of 48 branches end up in local memory (220 us against 90).
template <class T, bool ONCE, bool FINITE = false>
__device__ __forceinline__ void expandPlace(int code, const Place& q, const PlaceCodes& c, float2 (&v)[8]) {
    const uint32_t r[8] = {c.a.x, c.a.y, c.a.z, c.a.w, c.b.x, c.b.y, c.b.z, c.b.w};
    const float a = scaleValue<FINITE>(c.scale_a), b = scaleValue<FINITE>(c.scale_b);
    auto shifted = [&](auto shift) {
        constexpr int k = 16 - decltype(shift)::value;  // bytes of the first word that are left out
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = k % 4 == 0 ? r[k / 4 + i] : __funnelshift_r(r[k / 4 + i], r[(k / 4 + i + 1) % 8], k % 4 * 8);
        return make_uint4(w[0], w[1], w[2], w[3]);
    };
    auto scale = [&](auto shift) {
        constexpr int m = decltype(shift)::value;
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = mul2(v[i], make_float2(2 * i < m ? a : b, 2 * i + 1 < m ? a : b));
    };
    if constexpr (ONCE) {
        auto convert = [&](auto dtype) {
            byConstant<kShifts<T>>(q.m, [&](auto shift) {
                numbersAs<decltype(dtype)::value>(shifted(shift), v);
                scale(shift);
            });
        };
        if (code == THOR_B200_FP8_E4M3) convert(std::integral_constant<int, THOR_B200_FP8_E4M3>{});
        else if (code == THOR_B200_INT8) convert(std::integral_constant<int, THOR_B200_INT8>{});
        else convert(std::integral_constant<int, THOR_B200_FP8_E5M2>{});
    } else {
        uint4 w;
        byConstant<kShifts<T>>(q.m, [&](auto shift) { w = shifted(shift); });
        numbers16(w, code, v);
        byConstant<kShifts<T>>(q.m, scale);
    }
}

// ---- host side ------------------------------------------------------------------------------------------------
// Whether every row of a tensor starts on 32 bytes.
inline bool rowsAligned(const void* p, int64_t stride, int dtype, uint64_t rows) {
    return p == nullptr || (isAligned(p, 32) && (rows <= 1 || (static_cast<uint64_t>(stride) * dtypeSize(dtype)) % 32 == 0));
}
// Whether two tensors' rows start at the same place of 32 bytes, all of them.
inline bool rowsCongruent(const void* p, int64_t p_stride, const void* q, int64_t q_stride, int dtype) {
    return (reinterpret_cast<uintptr_t>(p) - reinterpret_cast<uintptr_t>(q)) % 32 == 0 &&
           (static_cast<uint64_t>(p_stride) - static_cast<uint64_t>(q_stride)) * dtypeSize(dtype) % 32 == 0;
}
// The stride of checked arguments; one row has none.
inline uint32_t strideOf(int64_t stride, uint64_t rows) { return rows > 1 ? static_cast<uint32_t>(stride) : 0u; }
inline int checkRowStride(const char* who, const char* what, int64_t stride, uint64_t rows, uint64_t cols) {
    TB_REQUIRE(rows <= 1 || (stride >= 0 && static_cast<uint64_t>(stride) >= cols), "%s: the row stride of %s is smaller than a row", who, what);
    TB_REQUIRE(rows <= 1 || stride <= 0xffffffffll, "%s: the row stride of %s is 2^32 elements or more", who, what);
    return THOR_B200_OK;
}
template <class T>
Rows<T> rowsOf(const void* p, int64_t stride, uint64_t rows, uint64_t cols) {
    const T* t = static_cast<const T*>(p);
    return Rows<T>{t, strideOf(stride, rows), t == nullptr ? nullptr : t + (rows - 1) * static_cast<uint64_t>(strideOf(stride, rows)) + cols};
}
template <class F>
int byDtype(int dtype, F&& f) {
    switch (dtype) {
        case THOR_B200_FP32: return f(float{});
        case THOR_B200_FP16: return f(__half{});
        default: return f(__nv_bfloat16{});
    }
}
template <class F>
int byFlag(bool flag, F&& f) {
    return flag ? f(std::true_type{}) : f(std::false_type{});
}

}  // namespace ck8
}  // namespace tb
