// What the LayerNorm kernels share: teams of threads, row sums, parameters, and the checks of the description.
//
// A row belongs to a team: 2, 4 .. 32 neighbouring lanes, or whole warps.  Thread t of a team holds columns 16 t .. of its row (and, in
// kernels with several chunks a thread, 16 (t + k team) ..).  A CTA holds as many teams as fit; every team walks its own rows.
#pragma once

#include "checkpoint8.cuh"

namespace tb {
namespace ln {

using namespace ck8;

constexpr uint32_t kMaxThreads = 512;

// Scratch of a CTA for row sums that several warps share: [slot][team][warp].
struct Scratch {
    float2 part[2][kMaxThreads / 64][16];
};

// Sums of two values over a team; every thread of it gets both.  Consecutive calls use different slots, so one barrier a call is enough.
__device__ __forceinline__ float2 teamSum(float2 v, uint32_t team, uint32_t team_id, Scratch& scratch, int slot) {
    if (team <= 32) {
        for (uint32_t o = team / 2; o > 0; o /= 2) v = add2(v, make_float2(__shfl_xor_sync(0xffffffffu, v.x, o), __shfl_xor_sync(0xffffffffu, v.y, o)));
        return v;
    }
    const uint32_t lane = threadIdx.x % 32, warps = team / 32, warp = threadIdx.x / 32 - team_id * warps;
    // the lower half-warp keeps the first value, the upper half the second: five exchanges for the two sums
    float s = lane < 16 ? v.x : v.y;
    s += __shfl_xor_sync(0xffffffffu, lane < 16 ? v.y : v.x, 16);
#pragma unroll
    for (int o = 8; o > 0; o /= 2) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (lane % 16 == 0) reinterpret_cast<float*>(&scratch.part[slot][team_id][warp])[lane / 16] = s;
    asm volatile("bar.sync %0, %1;" ::"r"(team_id + 1), "r"(team) : "memory");
    s = lane % 16 < warps ? reinterpret_cast<const float*>(&scratch.part[slot][team_id][lane % 16])[lane / 16] : 0.0f;
#pragma unroll
    for (int o = 8; o > 0; o /= 2) s += __shfl_xor_sync(0xffffffffu, s, o);
    const float other = __shfl_xor_sync(0xffffffffu, s, 16);
    return lane < 16 ? make_float2(s, other) : make_float2(other, s);
}
// The same for one row, or for two: four values, a quarter-warp keeps one each (teams of at most 384 threads).
__device__ __forceinline__ void teamSums(float2 (&v)[1], uint32_t team, uint32_t team_id, Scratch& scratch, int slot) { v[0] = teamSum(v[0], team, team_id, scratch, slot); }
__device__ __forceinline__ void teamSums(float2 (&v)[2], uint32_t team, uint32_t team_id, Scratch& scratch, int slot) {
    constexpr uint32_t all = 0xffffffffu;
    const uint32_t lane = threadIdx.x % 32, warps = team / 32, warp = threadIdx.x / 32 - team_id * warps;
    const bool second = lane & 16, odd = lane & 8;  // which row, which of its values a lane keeps
    float2 u = second ? v[1] : v[0];
    const float2 give = second ? v[0] : v[1];
    u = add2(u, make_float2(__shfl_xor_sync(all, give.x, 16), __shfl_xor_sync(all, give.y, 16)));
    float s = odd ? u.y : u.x;
    s += __shfl_xor_sync(all, odd ? u.x : u.y, 8);
#pragma unroll
    for (int o = 4; o > 0; o /= 2) s += __shfl_xor_sync(all, s, o);
    float(*part)[4] = reinterpret_cast<float(*)[4]>(&scratch.part[slot][team_id][0]);  // [warp][value]: one team, or two of six warps
    if (lane % 8 == 0) part[warp][lane / 8] = s;
    asm volatile("bar.sync %0, %1;" ::"r"(team_id + 1), "r"(team) : "memory");
    s = (lane % 8 < warps ? part[lane % 8][lane / 8] : 0.0f) + (lane % 8 + 8 < warps ? part[lane % 8 + 8][lane / 8] : 0.0f);
#pragma unroll
    for (int o = 4; o > 0; o /= 2) s += __shfl_xor_sync(all, s, o);
    v[0] = make_float2(__shfl_sync(all, s, 0), __shfl_sync(all, s, 8));
    v[1] = make_float2(__shfl_sync(all, s, 16), __shfl_sync(all, s, 24));
}
// Columns that a warp of a team holds, `chunks_a_thread` runs of 512 a team apart.
__device__ __forceinline__ float warpColumns(uint32_t warp, uint32_t team, uint32_t cols, int chunks_a_thread) {
    uint32_t n = 0;
    for (int k = 0; k < chunks_a_thread; ++k) {
        const uint32_t first = (warp * 32 + k * team) * kVec;
        n += first < cols ? min(cols - first, 32u * kVec) : 0u;
    }
    return static_cast<float>(n);
}
// Sum over 2, 4 .. 32 neighbouring lanes.
__device__ __forceinline__ float laneSum(float v, uint32_t lanes) {
    if (lanes == 32) v += __shfl_xor_sync(0xffffffffu, v, 16);
    if (lanes >= 16) v += __shfl_xor_sync(0xffffffffu, v, 8);
    if (lanes >= 8) v += __shfl_xor_sync(0xffffffffu, v, 4);
    if (lanes >= 4) v += __shfl_xor_sync(0xffffffffu, v, 2);
    return v + __shfl_xor_sync(0xffffffffu, v, 1);
}

// Sums over a CTA of up to 1024 threads, for the kernels that loop over long rows.
__device__ __forceinline__ float ctaSum(float v, float* slot) {
#pragma unroll
    for (int o = 16; o > 0; o /= 2) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (threadIdx.x % 32 == 0) slot[threadIdx.x / 32] = v;
    __syncthreads();
    v = threadIdx.x % 32 < blockDim.x / 32 ? slot[threadIdx.x % 32] : 0.0f;
#pragma unroll
    for (int o = 16; o > 0; o /= 2) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

__device__ __forceinline__ float sum16(const float2 (&v)[8]) {
    const float2 a = add2(add2(v[0], v[1]), add2(v[2], v[3])), b = add2(add2(v[4], v[5]), add2(v[6], v[7]));
    const float2 s = add2(a, b);
    return s.x + s.y;
}

// A parameter (gamma, beta) of `cols` values of any floating type.
struct Param {
    const void* p;
    int dtype;
    bool aligned;  // 16-byte aligned
};
template <class T>
__device__ __forceinline__ void loadParamAs(const Param& q, uint32_t col, uint32_t cols, float2 (&v)[4]) {
    const T* p = static_cast<const T*>(q.p) + col;
    if (q.aligned && col + 8 <= cols) {
#pragma unroll
        for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i) {
            const uint4 u = __ldg(reinterpret_cast<const uint4*>(p) + i);
            if constexpr (sizeof(T) == 4) {
                v[2 * i] = make_float2(__uint_as_float(u.x), __uint_as_float(u.y));
                v[2 * i + 1] = make_float2(__uint_as_float(u.z), __uint_as_float(u.w));
            } else {
                v[0] = widen(u.x, T{});
                v[1] = widen(u.y, T{});
                v[2] = widen(u.z, T{});
                v[3] = widen(u.w, T{});
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[i].x = col + 2 * i < cols ? static_cast<float>(p[2 * i]) : 0.0f;
            v[i].y = col + 2 * i + 1 < cols ? static_cast<float>(p[2 * i + 1]) : 0.0f;
        }
    }
}
// Eight neighbouring values, `absent` where there is no parameter.
__device__ __forceinline__ void loadParam8(const Param& q, float absent, uint32_t col, uint32_t cols, float2 (&v)[4]) {
    if (q.p == nullptr) {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = both(absent);
    } else if (q.dtype == THOR_B200_FP32) {
        loadParamAs<float>(q, col, cols, v);
    } else if (q.dtype == THOR_B200_FP16) {
        loadParamAs<__half>(q, col, cols, v);
    } else {
        loadParamAs<__nv_bfloat16>(q, col, cols, v);
    }
}

// A parameter in shared memory, for kernels that walk many rows: kept in registers it would take a quarter of them, read from global memory for
// every row it costs the tests of its type.  As fp32, or, PACKED, in the tensors' own 16-bit type where the parameter has it, which halves
// the words that a row reads.  Chunk c's sixteen values lie in planes of 16 bytes a chunk, so that neighbouring threads read neighbouring words.
template <class T, bool PACKED>
struct Staged {
    static constexpr int kPlanes = PACKED ? 2 : 4;
    __device__ __forceinline__ static void stage(const Param& q, float absent, uint4* planes, uint32_t chunks, uint32_t cols) {
        for (uint32_t c = threadIdx.x; c < chunks; c += blockDim.x) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float2 v[4];
                loadParam8(q, absent, c * kVec + 8 * h, cols, v);
                if constexpr (PACKED) {
                    planes[h * chunks + c] = make_uint4(narrow(v[0], T{}), narrow(v[1], T{}), narrow(v[2], T{}), narrow(v[3], T{}));
                } else {
                    planes[(2 * h) * chunks + c] = make_uint4(__float_as_uint(v[0].x), __float_as_uint(v[0].y), __float_as_uint(v[1].x), __float_as_uint(v[1].y));
                    planes[(2 * h + 1) * chunks + c] = make_uint4(__float_as_uint(v[2].x), __float_as_uint(v[2].y), __float_as_uint(v[3].x), __float_as_uint(v[3].y));
                }
            }
        }
    }
    // Values 8 h .. 8 h + 7 of chunk c.
    __device__ __forceinline__ static void read(const uint4* planes, uint32_t chunks, uint32_t c, int h, float2 (&v)[4]) {
        if constexpr (PACKED) {
            const uint4 a = planes[h * chunks + c];
            v[0] = widen(a.x, T{});
            v[1] = widen(a.y, T{});
            v[2] = widen(a.z, T{});
            v[3] = widen(a.w, T{});
        } else {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const uint4 a = planes[(2 * h + i) * chunks + c];
                v[2 * i] = make_float2(__uint_as_float(a.x), __uint_as_float(a.y));
                v[2 * i + 1] = make_float2(__uint_as_float(a.z), __uint_as_float(a.w));
            }
        }
    }
};

// s / count, inverse = 1 / count rounded: the quotient of the product is off by its roundings, the remainder mends it.
__device__ __forceinline__ float divideBy(float s, float count, float inverse) {
    const float q = s * inverse;
    return isfinite(q) ? fmaf(fmaf(-q, count, s), inverse, q) : q;
}
// 1 / sqrt(v): the hardware's approximation and one Newton step (its error squared is below the last place); 0, infinity and NaN as they come.
__device__ __forceinline__ float inverseRoot(float v) {
    float y;
    asm("rsqrt.approx.f32 %0, %1;" : "=f"(y) : "f"(v));
    return v > 0.0f && isfinite(v) ? fmaf(0.5f * y, fmaf(-(v * y), y, 1.0f), y) : y;
}

// ---- host side --------------------------------------------------------------------------------------------
inline Param paramOf(const void* p, int dtype) { return Param{p, dtype, isAligned(p, 16)}; }

// Threads of a row of `chunks` chunks with `per_thread` of them each.
inline uint32_t teamOf(uint64_t chunks, uint64_t per_thread) {
    const uint64_t threads = (chunks + per_thread - 1) / per_thread;
    uint32_t team = 2;
    while (team < 32 && team < threads) team *= 2;
    return team < threads ? static_cast<uint32_t>((threads + 31) / 32 * 32) : team;
}

// Lets a kernel use more than the default 48 KB of shared memory, once a device.
template <auto KERNEL>
int allowShared(size_t bytes) {
    static std::atomic<uint64_t> done{0};
    int device = 0;
    TB_CUDA(cudaGetDevice(&device));
    if (bytes <= (40u << 10) || (done.load(std::memory_order_relaxed) >> (device & 63) & 1)) return THOR_B200_OK;
    TB_CUDA(cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, 160 << 10));
    done.fetch_or(1ull << (device & 63), std::memory_order_relaxed);
    return THOR_B200_OK;
}

inline int checkDesc(const char* who, const thor_b200_layernorm_desc* d) {
    TB_REQUIRE(d != nullptr, "%s: null description", who);
    TB_REQUIRE(valueDtypeOk(d->dtype), "%s: tensors must be fp32, fp16 or bf16, got %s", who, dtypeName(d->dtype));
    TB_REQUIRE(valueDtypeOk(d->param_dtype), "%s: parameters must be fp32, fp16 or bf16, got %s", who, dtypeName(d->param_dtype));
    TB_REQUIRE(d->code_dtype == 0 || codeDtypeOk(d->code_dtype), "%s: codes must be fp8_e4m3, fp8_e5m2 or int8, got %s", who, dtypeName(d->code_dtype));
    TB_REQUIRE(d->reserved == 0, "%s: reserved must be zero", who);
    TB_REQUIRE(d->cols > 0 && d->cols <= 0x7fffffffull, "%s: rows must have 1 to 2^31 - 1 columns", who);
    TB_REQUIRE(d->rows <= 0x7fffffffull, "%s: more than 2^31 - 1 rows", who);
    TB_REQUIRE(d->eps >= 0.0f, "%s: eps must not be negative", who);
    return THOR_B200_OK;
}
inline int checkStride(const char* who, const char* what, int64_t stride, const thor_b200_layernorm_desc& d) { return checkRowStride(who, what, stride, d.rows, d.cols); }
// A tensor that may be absent.
inline int checkPointer(const char* who, const void* p, size_t alignment) {
    TB_REQUIRE(isAligned(p, alignment), "%s: a tensor pointer is not aligned to its elements", who);
    return THOR_B200_OK;
}
inline int checkKept(const char* who, const void* codes, const void* scales, const thor_b200_layernorm_desc& d) {
    TB_REQUIRE((codes != nullptr || scales != nullptr) == (d.code_dtype != 0) && (codes != nullptr) == (scales != nullptr), "%s: codes and scales go with a code_dtype", who);
    TB_REQUIRE(isAligned(codes, 16), "%s: codes must be 16-byte aligned", who);
    return THOR_B200_OK;
}

}  // namespace ln
}  // namespace tb
