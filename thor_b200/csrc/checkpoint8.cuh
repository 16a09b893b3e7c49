// 8-bit activation checkpoints: the device side of their format, shared by every kernel that writes or reads one.
//
// A block is 32 neighbouring columns of one row.  Its scale is the smallest power of two s with max|x| <= s * M, M the
// largest code (448 for e4m3, 57344 for e5m2, 127 for int8), stored as the byte log2(s) + 127 (e8m0); a code is x / s
// rounded to nearest even.  Division and multiplication by a power of two are exact, so a value that is packed again from its
// own unpacked form gives the same code, and pack / unpack have exactly one rounding.  s is clamped at 2^-127 from below (an
// all-zero block has that scale).  A block that holds an infinity or a NaN has the scale byte 255 and codes zero, and
// unpacks as NaN throughout: an overflow stays visible in the backward pass.
//
// A thread holds eight neighbouring columns, so four neighbouring lanes hold a block.
#pragma once

#include "common.cuh"

namespace tb {
namespace ck8 {

constexpr int kBlock = 32;  // columns of a block
constexpr int kVec = 8;     // columns of a thread

__host__ __device__ inline uint64_t codePitch(uint64_t cols) { return (cols + 15) / 16 * 16; }
__host__ __device__ inline uint64_t scalePitch(uint64_t cols) { return (cols + kBlock - 1) / kBlock; }

inline bool codeDtypeOk(int dt) { return dt == THOR_B200_FP8_E4M3 || dt == THOR_B200_FP8_E5M2 || dt == THOR_B200_INT8; }
inline bool valueDtypeOk(int dt) { return dt == THOR_B200_FP32 || dt == THOR_B200_FP16 || dt == THOR_B200_BF16; }

__device__ __forceinline__ float maxNan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

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

// max|v|, NaN if one of them is NaN
__device__ __forceinline__ float maxAbs8(const float (&v)[8]) {
    float m = fabsf(v[0]);
#pragma unroll
    for (int i = 1; i < 8; ++i) m = maxNan(m, fabsf(v[i]));
    return m;
}
// over the four lanes of a block; all 32 lanes take part
__device__ __forceinline__ float blockMax(float m) {
    m = maxNan(m, __shfl_xor_sync(0xffffffffu, m, 1));
    return maxNan(m, __shfl_xor_sync(0xffffffffu, m, 2));
}

// Scale byte of a block with largest magnitude `amax`: the exponent field, plus one where the significand is above that of
// M (the addition carries exactly then), less the exponent of M.
__device__ __forceinline__ uint32_t scaleByte(float amax, int code) {
    const uint32_t bits = __float_as_uint(amax);
    if (bits >= 0x7f800000u) return 255u;
    const uint32_t carry = code == THOR_B200_INT8 ? 0x7fffffu - 0x7e0000u : 0x7fffffu - 0x600000u;  // 127 = 1.984375 * 2^6, 448 and 57344 = 1.75 * 2^n
    const int exponent = code == THOR_B200_INT8 ? 6 : (code == THOR_B200_FP8_E4M3 ? 8 : 15);
    const int byte = static_cast<int>((bits + carry) >> 23) - exponent;
    return byte < 0 ? 0u : static_cast<uint32_t>(byte);
}
__device__ __forceinline__ float scaleValue(uint32_t byte) {
    return __uint_as_float(byte == 0 ? 0x00400000u : (byte == 255u ? 0x7fc00000u : byte << 23));
}

__device__ __forceinline__ uint32_t pack4(float a, float b, float c, float d, int code) {
    if (code == THOR_B200_INT8) {
        // adding 1.5 * 2^23 rounds to an integer (to nearest even) and leaves it in the low bits in two's complement
        const float magic = 12582912.0f;
        const uint32_t lo = __byte_perm(__float_as_uint(a + magic), __float_as_uint(b + magic), 0x0040);
        const uint32_t hi = __byte_perm(__float_as_uint(c + magic), __float_as_uint(d + magic), 0x0040);
        return __byte_perm(lo, hi, 0x5410);
    }
    uint16_t lo, hi;
    if (code == THOR_B200_FP8_E4M3) {
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
    } else {
        asm("cvt.rn.satfinite.e5m2x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
        asm("cvt.rn.satfinite.e5m2x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
    }
    return static_cast<uint32_t>(lo) | (static_cast<uint32_t>(hi) << 16);
}

// Codes of eight values of a block with scale byte `byte`.
__device__ __forceinline__ uint2 encode8(const float (&v)[8], uint32_t byte, int code) {
    if (byte == 255u) return make_uint2(0u, 0u);
    const float inv = __uint_as_float((254u - byte) << 23);  // 2^(127 - byte); byte <= 249 here
    return make_uint2(pack4(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv, code), pack4(v[4] * inv, v[5] * inv, v[6] * inv, v[7] * inv, code));
}

__device__ __forceinline__ void unpack4(uint32_t c, float s, int code, float& a, float& b, float& x, float& d) {
    if (code == THOR_B200_INT8) {
        // byte + 128 in the low bits of 2^23 is the float 2^23 + 128 + value; both steps are exact
        const uint32_t u = c ^ 0x80808080u;
        const float off = 8388736.0f;
        a = (__uint_as_float(__byte_perm(u, 0x4b000000u, 0x7440)) - off) * s;
        b = (__uint_as_float(__byte_perm(u, 0x4b000000u, 0x7441)) - off) * s;
        x = (__uint_as_float(__byte_perm(u, 0x4b000000u, 0x7442)) - off) * s;
        d = (__uint_as_float(__byte_perm(u, 0x4b000000u, 0x7443)) - off) * s;
        return;
    }
    uint32_t lo, hi;
    const uint16_t c0 = static_cast<uint16_t>(c), c1 = static_cast<uint16_t>(c >> 16);
    if (code == THOR_B200_FP8_E4M3) {
        asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(lo) : "h"(c0));
        asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(hi) : "h"(c1));
    } else {  // an e5m2 code is the upper byte of the fp16 number of the same value
        lo = __byte_perm(c, 0u, 0x1404);
        hi = __byte_perm(c, 0u, 0x3424);
    }
    const float2 f0 = __half22float2(*reinterpret_cast<const __half2*>(&lo)), f1 = __half22float2(*reinterpret_cast<const __half2*>(&hi));
    a = f0.x * s;
    b = f0.y * s;
    x = f1.x * s;
    d = f1.y * s;
}
__device__ __forceinline__ void decode8(uint2 c, float s, int code, float (&v)[8]) {
    unpack4(c.x, s, code, v[0], v[1], v[2], v[3]);
    unpack4(c.y, s, code, v[4], v[5], v[6], v[7]);
}

// ---- eight neighbouring elements of a row ---------------------------------------------------------------
template <class T>
__device__ __forceinline__ float toFloat(T v) {
    return static_cast<float>(v);
}
__device__ __forceinline__ void widen8(const Pack<32>& p, float (&v)[8], float) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = reinterpret_cast<const float*>(&p)[i];
}
__device__ __forceinline__ void widen8(const Pack<16>& p, float (&v)[8], __half) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(reinterpret_cast<const __half2*>(&p)[i]);
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
    }
}
__device__ __forceinline__ void widen8(const Pack<16>& p, float (&v)[8], __nv_bfloat16) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {  // a bf16 number is the upper half of the fp32 number of the same value
        const uint32_t w = reinterpret_cast<const uint32_t*>(&p)[i];
        v[2 * i] = __uint_as_float(w << 16);
        v[2 * i + 1] = __uint_as_float(w & 0xffff0000u);
    }
}
__device__ __forceinline__ void narrow8(const float (&v)[8], Pack<32>& p, float) {
#pragma unroll
    for (int i = 0; i < 8; ++i) reinterpret_cast<float*>(&p)[i] = v[i];
}
__device__ __forceinline__ void narrow8(const float (&v)[8], Pack<16>& p, __half) {
#pragma unroll
    for (int i = 0; i < 4; ++i) reinterpret_cast<__half2*>(&p)[i] = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
}
__device__ __forceinline__ void narrow8(const float (&v)[8], Pack<16>& p, __nv_bfloat16) {
#pragma unroll
    for (int i = 0; i < 4; ++i) reinterpret_cast<__nv_bfloat162*>(&p)[i] = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
}

// Columns col .. col + 7 of a row of `cols`; a column past the row's end is zero.  ALIGNED: the row starts on 16 bytes and
// cols is a multiple of 8, so a chunk is either whole or absent.
template <bool ALIGNED, class T>
__device__ __forceinline__ void loadRow8(const T* row, uint32_t col, uint32_t cols, float (&v)[8]) {
    if constexpr (ALIGNED) {
        Pack<8 * sizeof(T)> p{};
        if (col < cols) loadPack(p, row + col);
        widen8(p, v, T{});
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = col + i < cols ? toFloat(row[col + i]) : 0.0f;
    }
}
template <bool ALIGNED, class T>
__device__ __forceinline__ void storeRow8(T* row, uint32_t col, uint32_t cols, const float (&v)[8]) {
    if constexpr (ALIGNED) {
        Pack<8 * sizeof(T)> p;
        narrow8(v, p, T{});
        if (col < cols) storePack(row + col, p);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (col + i < cols) row[col + i] = static_cast<T>(v[i]);
    }
}
// Rounds eight values to T and back: what a reader of the stored tensor sees.
template <class T>
__device__ __forceinline__ void roundTo8(float (&v)[8]) {
    if constexpr (sizeof(T) < 4) {
        Pack<16> p;
        narrow8(v, p, T{});
        widen8(p, v, T{});
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

// Eight columns of one row by every lane; lanes 4 k .. 4 k + 3 hold one block and columns past the row's end are zero.
// All 32 lanes call it, with active = false where a lane has no row.
__device__ __forceinline__ void writeRow8(const Writer& w, uint64_t row, uint32_t col, uint32_t cols, const float (&v)[8], bool active) {
    const uint32_t byte = scaleByte(blockMax(maxAbs8(v)), w.code);
    if (!active || col >= w.code_pitch) return;  // a chunk between cols and the pitch writes the padding's zeros
    *reinterpret_cast<uint2*>(w.codes + row * w.code_pitch + col) = encode8(v, byte, w.code);
    if (col % kBlock == 0 && col < cols) w.scales[row * w.scale_pitch + col / kBlock] = static_cast<uint8_t>(byte);
}
__device__ __forceinline__ void readRow8(const Reader& r, uint64_t row, uint32_t col, uint32_t cols, float (&v)[8]) {
    if (col >= cols) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = 0.0f;
        return;
    }
    const uint2 c = __ldcs(reinterpret_cast<const uint2*>(r.codes + row * r.code_pitch + col));
    decode8(c, scaleValue(r.scales[row * r.scale_pitch + col / kBlock]), r.code, v);
}

}  // namespace ck8
}  // namespace tb
