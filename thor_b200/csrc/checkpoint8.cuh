// 8-bit activation checkpoints: the device side of their format, shared by every kernel that writes or reads one.
//
// A block is 32 neighbouring columns of one row.  Its scale is the smallest power of two s with max|x| <= s * M, M the
// largest code (448 for e4m3, 57344 for e5m2, 127 for int8), stored as the byte log2(s) + 127 (e8m0); a code is x / s
// rounded to nearest even.  Division and multiplication by a power of two are exact, so a value that is packed again from its
// own unpacked form gives the same code, and pack / unpack have exactly one rounding.  s is clamped at 2^-127 from below (an
// all-zero block has that scale).  A block that holds an infinity or a NaN has the scale byte 255 and codes zero, and
// unpacks as NaN throughout: an overflow stays visible in the backward pass.
//
// A thread holds sixteen neighbouring columns (32 bytes of a 16-bit tensor, one 16-byte word of codes), so two neighbouring lanes
// hold a block.
#pragma once

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
__device__ __forceinline__ float scaleValue(uint32_t byte) {
    return __uint_as_float(byte == 0 ? 0x00400000u : (byte == 255u ? 0x7fc00000u : byte << 23));
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
__device__ __forceinline__ void unpack4(uint32_t c, float2 s, float2& a, float2& b) {
    if constexpr (CODE == THOR_B200_INT8) {
        // byte + 128 in the low bits of 2^23 is the float 2^23 + 128 + value; both steps are exact
        const uint32_t u = c ^ 0x80808080u;
        const float2 off = both(-8388736.0f);
        a = make_float2(__uint_as_float(__byte_perm(u, 0x4b000000u, 0x7440)), __uint_as_float(__byte_perm(u, 0x4b000000u, 0x7441)));
        b = make_float2(__uint_as_float(__byte_perm(u, 0x4b000000u, 0x7442)), __uint_as_float(__byte_perm(u, 0x4b000000u, 0x7443)));
        a = mul2(add2(a, off), s);
        b = mul2(add2(b, off), s);
    } else {
        uint32_t lo, hi;
        if constexpr (CODE == THOR_B200_FP8_E4M3) {
            asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(lo) : "h"(static_cast<uint16_t>(c)));
            asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(hi) : "h"(static_cast<uint16_t>(c >> 16)));
        } else {  // an e5m2 code is the upper byte of the fp16 number of the same value
            lo = __byte_perm(c, 0u, 0x1404);
            hi = __byte_perm(c, 0u, 0x3424);
        }
        a = mul2(__half22float2(*reinterpret_cast<const __half2*>(&lo)), s);
        b = mul2(__half22float2(*reinterpret_cast<const __half2*>(&hi)), s);
    }
}
template <int CODE>
__device__ __forceinline__ void decodeAs(uint4 c, float2 s, float2 (&v)[8]) {
    unpack4<CODE>(c.x, s, v[0], v[1]);
    unpack4<CODE>(c.y, s, v[2], v[3]);
    unpack4<CODE>(c.z, s, v[4], v[5]);
    unpack4<CODE>(c.w, s, v[6], v[7]);
}
__device__ __forceinline__ void decode16(uint4 c, uint32_t byte, int code, float2 (&v)[8]) {
    const float2 s = both(scaleValue(byte));
    if (code == THOR_B200_FP8_E4M3) decodeAs<THOR_B200_FP8_E4M3>(c, s, v);
    else if (code == THOR_B200_INT8) decodeAs<THOR_B200_INT8>(c, s, v);
    else decodeAs<THOR_B200_FP8_E5M2>(c, s, v);
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

// Rows of a tensor that is read.
template <class T>
struct Rows {
    const T* p;
    int64_t stride;   // elements between rows
    const void* end;  // one past the last element
};

// What a thread has loaded of a row.  ALIGNED: rows start on 32 bytes and have a multiple of 16 columns, so sixteen columns are whole or absent
// and are the words themselves.  Otherwise: the 16-byte words that contain the sixteen elements, one more than they fill.
template <class T, bool ALIGNED>
struct Raw {
    uint32_t w[kRegs<T> + (ALIGNED ? 0 : 4)];
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

// Columns col .. col + 15 of a row of `cols`.
template <class T, bool ALIGNED>
__device__ __forceinline__ void fetch16(const Rows<T>& in, uint64_t row, uint32_t col, uint32_t cols, Raw<T, ALIGNED>& raw) {
    const T* p = in.p + row * in.stride + col;
    constexpr int words = (kRegs<T> + (ALIGNED ? 0 : 4)) / 4;
    if (col >= cols) {
#pragma unroll
        for (int i = 0; i < 4 * words; ++i) raw.w[i] = 0;
        return;
    }
    if constexpr (ALIGNED) {
#pragma unroll
        for (int i = 0; i < words; i += 2) {
            uint4 lo, hi;
            load256(lo, hi, reinterpret_cast<const char*>(p) + 16 * i);
            raw.w[4 * i] = lo.x, raw.w[4 * i + 1] = lo.y, raw.w[4 * i + 2] = lo.z, raw.w[4 * i + 3] = lo.w;
            raw.w[4 * i + 4] = hi.x, raw.w[4 * i + 5] = hi.y, raw.w[4 * i + 6] = hi.z, raw.w[4 * i + 7] = hi.w;
        }
    } else {
        const char* const last = reinterpret_cast<const char*>(p + min(16u, cols - col));
        const char* const word0 = reinterpret_cast<const char*>(reinterpret_cast<uintptr_t>(p) & ~static_cast<uintptr_t>(15));
#pragma unroll
        for (int i = 0; i < words; ++i) {
            const char* word = word0 + 16 * i;
            uint4 q = make_uint4(0u, 0u, 0u, 0u);
            if (word < last) {
                if (word >= reinterpret_cast<const char*>(in.p) && word + 16 <= in.end) q = __ldg(reinterpret_cast<const uint4*>(word));  // shared with the neighbouring lane
                else q = edgeWord<T>(word, in.p, in.end);
            }
            raw.w[4 * i] = q.x, raw.w[4 * i + 1] = q.y, raw.w[4 * i + 2] = q.z, raw.w[4 * i + 3] = q.w;
        }
    }
}

// r[i] = bytes 4 i + shift .. of the run of words, shift in 0 .. 16 a multiple of the element's size; MORE words follow the wanted ones.
template <int WANTED, int MORE, bool HALVES>
__device__ __forceinline__ void shiftWords(uint32_t (&r)[WANTED + MORE], uint32_t shift) {
    static_assert(MORE == 4, "shift by up to four words");
#pragma unroll
    for (int i = 0; i < WANTED; ++i) r[i] = shift & 16 ? r[i + 4] : r[i];  // then nothing else is set
#pragma unroll
    for (int i = 0; i < WANTED + 2; ++i) r[i] = shift & 8 ? r[i + 2] : r[i];
#pragma unroll
    for (int i = 0; i < WANTED + 1; ++i) r[i] = shift & 4 ? r[i + 1] : r[i];
    if constexpr (HALVES) {
#pragma unroll
        for (int i = 0; i < WANTED; ++i) r[i] = __funnelshift_r(r[i], r[i + 1], (shift & 2) * 8);
    }
}

// The sixteen values; zero past the row's end.
template <class T, bool ALIGNED>
__device__ __forceinline__ void expand16(const Rows<T>& in, uint64_t row, uint32_t col, uint32_t cols, const Raw<T, ALIGNED>& raw, float2 (&v)[8]) {
    if constexpr (ALIGNED) {
        widen16<T>(raw.w, v);
    } else {
        uint32_t r[kRegs<T> + 4], w[kRegs<T>];
#pragma unroll
        for (int i = 0; i < kRegs<T> + 4; ++i) r[i] = raw.w[i];
        shiftWords<kRegs<T>, 4, sizeof(T) == 2>(r, static_cast<uint32_t>(reinterpret_cast<uintptr_t>(in.p + row * in.stride + col)) & 15u);
#pragma unroll
        for (int i = 0; i < kRegs<T>; ++i) w[i] = r[i];
        widen16<T>(w, v);
        if (col + 16 > cols) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if (col + 2 * i >= cols) v[i].x = 0.0f;
                if (col + 2 * i + 1 >= cols) v[i].y = 0.0f;
            }
        }
    }
}
template <bool ALIGNED, class T>
__device__ __forceinline__ void load16(const Rows<T>& in, uint64_t row, uint32_t col, uint32_t cols, float2 (&v)[8]) {
    Raw<T, ALIGNED> raw;
    fetch16(in, row, col, cols, raw);
    expand16(in, row, col, cols, raw, v);
}

// Writes sixteen values to columns col .. of the row that starts at `row`; a lane with cols = 0 writes nothing.  All 32 lanes call it.
// Not ALIGNED: a lane writes the 16-byte words that start in its range, the first of them with the last elements of the lane before
// it; `before` / `after`: that lane / the lane behind holds the sixteen columns before / behind these.  Words that reach over the row's ends or
// over a missing neighbour are written element by element.
template <bool ALIGNED, class T>
__device__ __forceinline__ void store16(T* row, uint32_t col, uint32_t cols, const float2 (&v)[8], bool before, bool after) {
    if constexpr (ALIGNED) {
        uint32_t w[kRegs<T>];
        narrow16<T>(v, w);
        if (col >= cols) return;
#pragma unroll
        for (int i = 0; i < kRegs<T>; i += 8)
            asm volatile("st.global.cs.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(reinterpret_cast<char*>(row + col) + 4 * i), "r"(w[i]), "r"(w[i + 1]),
                         "r"(w[i + 2]), "r"(w[i + 3]), "r"(w[i + 4]), "r"(w[i + 5]), "r"(w[i + 6]), "r"(w[i + 7])
                         : "memory");
    } else {
        constexpr int N = kRegs<T>, E = 16 / sizeof(T);
        uint32_t own[N], r[N + 4];
        narrow16<T>(v, own);
#pragma unroll
        for (int i = 0; i < 4; ++i) r[i] = __shfl_up_sync(0xffffffffu, own[N - 4 + i], 1);
#pragma unroll
        for (int i = 0; i < N; ++i) r[4 + i] = own[i];
        if (col >= cols) return;
        T* const p = row + col;
        const uint32_t odd = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(p)) & 15u;  // bytes past a 16-byte boundary
        shiftWords<N, 4, sizeof(T) == 2>(r, 16 - odd);
        const int m = static_cast<int>(odd / sizeof(T));  // elements of the first word that belong to the lane before
        const int left = static_cast<int>(min(cols - col, 1u << 20));  // elements up to the row's end
        T* const word0 = p - m;
#pragma unroll
        for (int k = 0; k < N / 4; ++k) {
            const int first = k * E - m;  // of the word, counted from col
            if ((k > 0 || before || m == 0) && first + E <= left) {
                __stcs(reinterpret_cast<uint4*>(word0 + k * E), make_uint4(r[4 * k], r[4 * k + 1], r[4 * k + 2], r[4 * k + 3]));
            } else {
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    if (first + e < left && (k > 0 || before || first + e >= 0)) {
                        if constexpr (sizeof(T) == 4) reinterpret_cast<uint32_t*>(word0)[k * E + e] = r[4 * k + e];
                        else reinterpret_cast<uint16_t*>(word0)[k * E + e] = static_cast<uint16_t>(r[4 * k + e / 2] >> (16 * (e % 2)));
                    }
                }
            }
        }
        if (m > 0 && left > 16 - m && !(after && left > 16)) {  // the last m elements have no lane behind to write them
#pragma unroll
            for (int e = 16 - E + 1; e < 16; ++e) {
                if (e >= 16 - m && e < left) {
                    if constexpr (sizeof(T) == 4) reinterpret_cast<uint32_t*>(p)[e] = own[e];
                    else reinterpret_cast<uint16_t*>(p)[e] = static_cast<uint16_t>(own[e / 2] >> (16 * (e % 2)));
                }
            }
        }
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
    uint64_t code_pitch, scale_pitch;
    int code;
};
struct Reader {
    const uint8_t* codes;
    const uint8_t* scales;
    uint64_t code_pitch, scale_pitch;
    int code;
};

// Sixteen columns of one row by every lane, zero past the row's end; lanes 2 k and 2 k + 1 hold one block.  All 32 lanes call it, with cols = 0
// where a lane has no row.
__device__ __forceinline__ void writeRow16(const Writer& w, uint64_t row, uint32_t col, uint32_t cols, const float2 (&v)[8]) {
    const uint32_t byte = scaleByte(blockMax(maxAbs16(v)), w.code);
    if (col >= cols) return;
    __stcs(reinterpret_cast<uint4*>(w.codes + row * w.code_pitch + col), encode16(v, byte, w.code));  // the pitch is a multiple of 16
    if (col % kBlock == 0) w.scales[row * w.scale_pitch + col / kBlock] = static_cast<uint8_t>(byte);
}
struct RawCodes {
    uint4 codes;
    uint32_t scale;
};
__device__ __forceinline__ void fetchCodes(const Reader& r, uint64_t row, uint32_t col, uint32_t cols, RawCodes& raw) {
    raw.codes = make_uint4(0u, 0u, 0u, 0u);
    raw.scale = 0;
    if (col >= cols) return;
    raw.codes = __ldcs(reinterpret_cast<const uint4*>(r.codes + row * r.code_pitch + col));
    raw.scale = r.scales[row * r.scale_pitch + col / kBlock];
}
// ALIGNED as for the tensors beside it; otherwise the padding behind the row's end is made zero whatever the block's scale.
template <bool ALIGNED>
__device__ __forceinline__ void expandCodes(const Reader& r, uint32_t col, uint32_t cols, const RawCodes& raw, float2 (&v)[8]) {
    decode16(raw.codes, raw.scale, r.code, v);
    if constexpr (!ALIGNED) {
        if (col + 16 > cols) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if (col + 2 * i >= cols) v[i].x = 0.0f;
                if (col + 2 * i + 1 >= cols) v[i].y = 0.0f;
            }
        }
    }
}

// ---- host side ------------------------------------------------------------------------------------------------
// Whether every row of a tensor starts on 32 bytes.
inline bool rowsAligned(const void* p, int64_t stride, int dtype, uint64_t rows) {
    return p == nullptr || (isAligned(p, 32) && (rows <= 1 || (static_cast<uint64_t>(stride) * dtypeSize(dtype)) % 32 == 0));
}
template <class T>
Rows<T> rowsOf(const void* p, int64_t stride, uint64_t rows, uint64_t cols) {
    const T* t = static_cast<const T*>(p);
    return Rows<T>{t, stride, t == nullptr ? nullptr : t + (rows - 1) * static_cast<uint64_t>(rows > 1 ? stride : 0) + cols};
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
