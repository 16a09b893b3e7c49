// Packing a tensor into an 8-bit activation checkpoint and unpacking it (the format stands in checkpoint8.cuh), and the
// activations that write a checkpoint in their forward pass and read it in their backward pass.
//
// All four are streaming kernels: each element is read and written once, a thread takes eight neighbouring columns (16 bytes
// of a 16-bit tensor, 8 bytes of codes) and the four lanes of a block of 32 columns agree on its scale with two shuffles.
// A tensor whose rows lie dense and whose width is a multiple of 32 is walked as one row, which saves the index division.
#include <algorithm>

#include "checkpoint8.cuh"

namespace tb {
namespace {

using namespace ck8;

constexpr int kThreads = 256;
constexpr int kUnroll = 2;  // chunks of eight columns per thread, loaded before the first is used

// Chunk number -> row and first column.  Every row has `chunks` of them, a multiple of four, so that a block never spans rows.
struct Walk {
    uint64_t units;
    uint32_t chunks, cols;
};
__device__ __forceinline__ void locate(const Walk& w, uint64_t unit, uint64_t& row, uint32_t& col) {
    if (w.units == w.chunks) {
        row = 0;
        col = static_cast<uint32_t>(unit) * kVec;
    } else if (w.units <= 0xffffffffull) {
        const uint32_t r = static_cast<uint32_t>(unit) / w.chunks;
        row = r;
        col = (static_cast<uint32_t>(unit) - r * w.chunks) * kVec;
    } else {
        row = unit / w.chunks;
        col = static_cast<uint32_t>(unit - row * w.chunks) * kVec;
    }
}

template <class T, bool ALIGNED>
__global__ void __launch_bounds__(kThreads) packKernel(const T* __restrict__ x, int64_t x_stride, Writer out, Walk w) {
    gridDependencyWait();
    gridLaunchDependents();
    float v[kUnroll][8];
    uint64_t row[kUnroll];
    uint32_t col[kUnroll];
    bool active[kUnroll];
#pragma unroll
    for (int k = 0; k < kUnroll; ++k) {
        const uint64_t unit = (static_cast<uint64_t>(blockIdx.x) * kUnroll + k) * kThreads + threadIdx.x;
        active[k] = unit < w.units;
        locate(w, active[k] ? unit : 0, row[k], col[k]);
        loadRow8<ALIGNED>(x + row[k] * x_stride, col[k], active[k] ? w.cols : 0, v[k]);
    }
#pragma unroll
    for (int k = 0; k < kUnroll; ++k) writeRow8(out, row[k], col[k], w.cols, v[k], active[k]);
}

template <class T, bool ALIGNED>
__global__ void __launch_bounds__(kThreads) unpackKernel(Reader in, T* __restrict__ y, int64_t y_stride, Walk w) {
    gridDependencyWait();
    gridLaunchDependents();
    float v[kUnroll][8];
    uint64_t row[kUnroll];
    uint32_t col[kUnroll];
    bool active[kUnroll];
#pragma unroll
    for (int k = 0; k < kUnroll; ++k) {
        const uint64_t unit = (static_cast<uint64_t>(blockIdx.x) * kUnroll + k) * kThreads + threadIdx.x;
        active[k] = unit < w.units;
        locate(w, active[k] ? unit : 0, row[k], col[k]);
        readRow8(in, row[k], col[k], active[k] ? w.cols : 0, v[k]);
    }
#pragma unroll
    for (int k = 0; k < kUnroll; ++k)
        if (active[k]) storeRow8<ALIGNED>(y + row[k] * y_stride, col[k], w.cols, v[k]);
}

// act(x) and act'(x) of two neighbouring columns: gelu(x) = x Phi(x), swish(x) = x sigma(x), as Expression::gelu and
// Expression::swish define them.
//
// sigma(x) = 1 / (1 + 2^(-x log2 e)) and sigma' x + sigma = value (1 - sigma) + sigma.
// Phi(-|x|) = e^(-x^2/2) R(|x|), where R(a) = erfcx(a / sqrt 2) / 2 is smooth and falls from 1/2 like 0.4 / a: R is a polynomial in
// t = 1 / (1 + p a) without a constant term, fitted here for the least relative error over 0 <= a <= 15, past which the
// exponential is below the smallest normal number.  The form keeps the relative accuracy of the far tail, and the exponential is the one
// that the derivative needs.  Degree 9: 2.1e-7 of the value as evaluated in fp32 (fp32 tensors); degree 6: 4.8e-6, a hundredth of
// half a unit of fp16 (16-bit tensors), three instructions a pair less.  For fp32 the rounding of x^2 is carried into the exponent.
// Two elements an instruction (f32x2) and one exponential and one reciprocal an element; the toolkit's erfcf and expf made the backward kernel
// wait for the arithmetic pipes (GELU [2999, 11001] fp16: 112 us).
template <int KIND, bool FULL>
__device__ __forceinline__ void activation2(float2 x, float2& value, float2& slope) {
    if constexpr (KIND == THOR_B200_ACTIVATION_SWISH) {
        const float2 y = mul2(x, both(-1.44269504f));
        const float2 d = add2(make_float2(exp2Approx(y.x), exp2Approx(y.y)), both(1.0f));
        const float2 s = make_float2(reciprocalApprox(d.x), reciprocalApprox(d.y));
        value = mul2(x, s);
        slope = fma2(value, fma2(s, both(-1.0f), both(1.0f)), s);
    } else {
        const float2 a = make_float2(fabsf(x.x), fabsf(x.y));
        const float2 u = fma2(a, both(FULL ? 0.345f : 0.31f), both(1.0f));
        const float2 t = make_float2(reciprocalApprox(u.x), reciprocalApprox(u.y));
        float2 r;
        if constexpr (FULL) {
            r = fma2(t, both(-0.027935062f), both(0.14324534f));
            r = fma2(r, t, both(-0.26724964f));
            r = fma2(r, t, both(0.18303713f));
            r = fma2(r, t, both(-0.034956314f));
            r = fma2(r, t, both(0.11076973f));
            r = fma2(r, t, both(0.117477186f));
            r = fma2(r, t, both(0.13799077f));
            r = fma2(r, t, both(0.13762087f));
        } else {
            r = fma2(t, both(-0.0739324f), both(0.1804593f));
            r = fma2(r, t, both(0.015735528f));
            r = fma2(r, t, both(0.13343409f));
            r = fma2(r, t, both(0.12044038f));
            r = fma2(r, t, both(0.12386077f));
        }
        const float2 square = mul2(x, x);
        const float2 half_log2e = both(-0.72134752f);
        float2 y = mul2(square, half_log2e);
        if constexpr (FULL) {  // square and its rounding error; an infinite x has no error to carry
            const float2 lost = fma2(x, x, make_float2(-square.x, -square.y));
            y = fma2(square, half_log2e, mul2(make_float2(a.x < 1e18f ? lost.x : 0.0f, a.y < 1e18f ? lost.y : 0.0f), half_log2e));
        }
        const float2 e = make_float2(exp2Approx(y.x), exp2Approx(y.y));
        const float2 q = mul2(mul2(r, t), e);
        const float2 phi = make_float2(x.x > 0.0f ? 1.0f - q.x : q.x, x.y > 0.0f ? 1.0f - q.y : q.y);
        value = mul2(x, phi);
        slope = fma2(mul2(x, both(0.39894228f)), e, phi);
    }
}

struct ActivationStrides {
    int64_t x, gate, y;
};

template <class T, int KIND, bool GATED, bool ALIGNED>
__global__ void __launch_bounds__(kThreads) activationKernel(const T* __restrict__ x, const T* __restrict__ gate, T* __restrict__ y, ActivationStrides st, Writer out,
                                                             Writer gate_out, Walk w) {
    gridDependencyWait();
    gridLaunchDependents();
    float v[kUnroll][8], g[GATED ? kUnroll : 1][8];
    uint64_t row[kUnroll];
    uint32_t col[kUnroll];
    bool active[kUnroll];
#pragma unroll
    for (int k = 0; k < kUnroll; ++k) {
        const uint64_t unit = (static_cast<uint64_t>(blockIdx.x) * kUnroll + k) * kThreads + threadIdx.x;
        active[k] = unit < w.units;
        locate(w, active[k] ? unit : 0, row[k], col[k]);
        loadRow8<ALIGNED>(x + row[k] * st.x, col[k], active[k] ? w.cols : 0, v[k]);
        if constexpr (GATED) loadRow8<ALIGNED>(gate + row[k] * st.gate, col[k], active[k] ? w.cols : 0, g[k]);
    }
#pragma unroll
    for (int k = 0; k < kUnroll; ++k) {
        float r[8];
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
            float2 value, slope;
            activation2<KIND, sizeof(T) == 4>(make_float2(v[k][i], v[k][i + 1]), value, slope);
            if constexpr (GATED) value = mul2(value, make_float2(g[k][i], g[k][i + 1]));
            r[i] = value.x;
            r[i + 1] = value.y;
        }
        if (active[k]) storeRow8<ALIGNED>(y + row[k] * st.y, col[k], w.cols, r);
        writeRow8(out, row[k], col[k], w.cols, v[k], active[k]);
        if constexpr (GATED) writeRow8(gate_out, row[k], col[k], w.cols, g[k], active[k]);
    }
}

template <class T, int KIND, bool GATED, bool ALIGNED>
__global__ void __launch_bounds__(kThreads) activationBackwardKernel(const T* __restrict__ grad, Reader in, Reader gate_in, T* __restrict__ grad_x, T* __restrict__ grad_gate,
                                                                     ActivationStrides st, Walk w) {
    gridDependencyWait();
    gridLaunchDependents();
    float d[kUnroll][8], v[kUnroll][8], g[GATED ? kUnroll : 1][8];
    uint64_t row[kUnroll];
    uint32_t col[kUnroll];
    bool active[kUnroll];
#pragma unroll
    for (int k = 0; k < kUnroll; ++k) {
        const uint64_t unit = (static_cast<uint64_t>(blockIdx.x) * kUnroll + k) * kThreads + threadIdx.x;
        active[k] = unit < w.units;
        locate(w, active[k] ? unit : 0, row[k], col[k]);
        const uint32_t cols = active[k] ? w.cols : 0;
        loadRow8<ALIGNED>(grad + row[k] * st.y, col[k], cols, d[k]);
        readRow8(in, row[k], col[k], cols, v[k]);
        if constexpr (GATED) readRow8(gate_in, row[k], col[k], cols, g[k]);
    }
#pragma unroll
    for (int k = 0; k < kUnroll; ++k) {
        if (!active[k]) continue;
        float dx[8], dg[8];
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
            float2 value, slope;
            activation2<KIND, sizeof(T) == 4>(make_float2(v[k][i], v[k][i + 1]), value, slope);
            const float2 grad2 = make_float2(d[k][i], d[k][i + 1]);
            float2 gx = mul2(grad2, slope);
            if constexpr (GATED) {
                const float2 gg = mul2(grad2, value);
                dg[i] = gg.x;
                dg[i + 1] = gg.y;
                gx = mul2(gx, make_float2(g[k][i], g[k][i + 1]));
            }
            dx[i] = gx.x;
            dx[i + 1] = gx.y;
        }
        storeRow8<ALIGNED>(grad_x + row[k] * st.x, col[k], w.cols, dx);
        if constexpr (GATED) storeRow8<ALIGNED>(grad_gate + row[k] * st.gate, col[k], w.cols, dg);
    }
}

// ---- host side --------------------------------------------------------------------------------------------
// A row-strided operand: where its rows start on 16 bytes whatever the row.
bool rowsAligned(const void* p, int64_t stride, int dtype, uint64_t rows) {
    return isAligned(p, 16) && (rows <= 1 || (static_cast<uint64_t>(stride) * dtypeSize(dtype)) % 16 == 0);
}

int planWalk(uint64_t rows, uint64_t cols, bool dense, Walk* w, dim3* grid) {
    if (dense && cols % kBlock == 0 && rows * cols < 0x80000000ull) {  // the checkpoint's rows are dense then, too
        cols *= rows;
        rows = 1;
    }
    w->chunks = static_cast<uint32_t>(scalePitch(cols) * (kBlock / kVec));
    w->cols = static_cast<uint32_t>(cols);
    w->units = rows * w->chunks;
    const uint64_t per_cta = static_cast<uint64_t>(kThreads) * kUnroll;
    const uint64_t ctas = (w->units + per_cta - 1) / per_cta;
    TB_REQUIRE(ctas <= 0x7FFFFFFFull, "checkpoint: too many elements for one grid");
    *grid = dim3(static_cast<unsigned>(ctas));
    return THOR_B200_OK;
}

int checkShape(const char* who, int dtype, int code_dtype, uint64_t rows, uint64_t cols) {
    TB_REQUIRE(valueDtypeOk(dtype), "%s: tensors must be fp32, fp16 or bf16, got %s", who, dtypeName(dtype));
    TB_REQUIRE(codeDtypeOk(code_dtype), "%s: codes must be fp8_e4m3, fp8_e5m2 or int8, got %s", who, dtypeName(code_dtype));
    TB_REQUIRE(cols > 0 && cols <= 0x7fffffffull, "%s: rows must have 1 to 2^31 - 1 columns", who);
    TB_REQUIRE(rows <= (1ull << 62) / (cols + kBlock), "%s: rows * cols overflows", who);
    return THOR_B200_OK;
}
int checkStride(const char* who, const char* what, int64_t stride, uint64_t rows, uint64_t cols) {
    TB_REQUIRE(rows <= 1 || (stride >= 0 && static_cast<uint64_t>(stride) >= cols), "%s: the row stride of %s is smaller than a row", who, what);
    return THOR_B200_OK;
}
int checkCheckpoint(const char* who, const void* codes, const void* scales) {
    TB_REQUIRE(codes != nullptr && scales != nullptr, "%s: null checkpoint pointer", who);
    TB_REQUIRE(isAligned(codes, 16), "%s: codes must be 16-byte aligned", who);
    return THOR_B200_OK;
}
Writer writerOf(void* codes, void* scales, uint64_t cols, int code) {
    return Writer{static_cast<uint8_t*>(codes), static_cast<uint8_t*>(scales), codePitch(cols), scalePitch(cols), code};
}
Reader readerOf(const void* codes, const void* scales, uint64_t cols, int code) {
    return Reader{static_cast<const uint8_t*>(codes), static_cast<const uint8_t*>(scales), codePitch(cols), scalePitch(cols), code};
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

int checkActivation(const char* who, const thor_b200_checkpointed_activation_desc* d) {
    TB_REQUIRE(d != nullptr, "%s: null description", who);
    TB_REQUIRE(d->kind == THOR_B200_ACTIVATION_GELU || d->kind == THOR_B200_ACTIVATION_SWISH, "%s: unknown activation %d", who, d->kind);
    if (int st = checkShape(who, d->dtype, d->code_dtype, d->rows, d->cols)) return st;
    if (int st = checkStride(who, "x", d->x_stride, d->rows, d->cols)) return st;
    if (d->gated)
        if (int st = checkStride(who, "gate", d->gate_stride, d->rows, d->cols)) return st;
    return checkStride(who, "y", d->y_stride, d->rows, d->cols);
}
bool denseRows(int64_t stride, uint64_t rows, uint64_t cols) { return rows <= 1 || static_cast<uint64_t>(stride) == cols; }

}  // namespace
}  // namespace tb

extern "C" {

uint64_t thor_b200_checkpoint_code_pitch(uint64_t cols) { return tb::ck8::codePitch(cols); }
uint64_t thor_b200_checkpoint_scale_pitch(uint64_t cols) { return tb::ck8::scalePitch(cols); }

int thor_b200_checkpoint_pack_launch(const thor_b200_checkpoint_desc* d, const void* x, void* codes, void* scales, void* stream_v) {
    using namespace tb;
    TB_REQUIRE(d != nullptr, "checkpoint_pack: null description");
    if (int st = checkShape("checkpoint_pack", d->dtype, d->code_dtype, d->rows, d->cols)) return st;
    if (int st = checkStride("checkpoint_pack", "the tensor", d->stride, d->rows, d->cols)) return st;
    if (d->rows == 0) return THOR_B200_OK;
    TB_REQUIRE(x != nullptr, "checkpoint_pack: null tensor pointer");
    if (int st = checkCheckpoint("checkpoint_pack", codes, scales)) return st;
    Walk w;
    dim3 grid;
    if (int st = planWalk(d->rows, d->cols, denseRows(d->stride, d->rows, d->cols), &w, &grid)) return st;
    const Writer out = writerOf(codes, scales, w.cols, d->code_dtype);
    cudaStream_t stream = static_cast<cudaStream_t>(stream_v);
    const bool aligned = rowsAligned(x, d->stride, d->dtype, d->rows) && d->cols % ck8::kVec == 0;
    return byDtype(d->dtype, [&](auto t) {
        using T = decltype(t);
        return byFlag(aligned, [&](auto a) {
            TB_CUDA(launchDependent(packKernel<T, decltype(a)::value>, grid, dim3(kThreads), 0, stream, static_cast<const T*>(x), d->stride, out, w));
            countLaunch();
            return static_cast<int>(THOR_B200_OK);
        });
    });
}

int thor_b200_checkpoint_unpack_launch(const thor_b200_checkpoint_desc* d, const void* codes, const void* scales, void* y, void* stream_v) {
    using namespace tb;
    TB_REQUIRE(d != nullptr, "checkpoint_unpack: null description");
    if (int st = checkShape("checkpoint_unpack", d->dtype, d->code_dtype, d->rows, d->cols)) return st;
    if (int st = checkStride("checkpoint_unpack", "the tensor", d->stride, d->rows, d->cols)) return st;
    if (d->rows == 0) return THOR_B200_OK;
    TB_REQUIRE(y != nullptr, "checkpoint_unpack: null tensor pointer");
    if (int st = checkCheckpoint("checkpoint_unpack", codes, scales)) return st;
    Walk w;
    dim3 grid;
    if (int st = planWalk(d->rows, d->cols, denseRows(d->stride, d->rows, d->cols), &w, &grid)) return st;
    const Reader in = readerOf(codes, scales, w.cols, d->code_dtype);
    cudaStream_t stream = static_cast<cudaStream_t>(stream_v);
    const bool aligned = rowsAligned(y, d->stride, d->dtype, d->rows) && d->cols % ck8::kVec == 0;
    return byDtype(d->dtype, [&](auto t) {
        using T = decltype(t);
        return byFlag(aligned, [&](auto a) {
            TB_CUDA(launchDependent(unpackKernel<T, decltype(a)::value>, grid, dim3(kThreads), 0, stream, in, static_cast<T*>(y), d->stride, w));
            countLaunch();
            return static_cast<int>(THOR_B200_OK);
        });
    });
}

int thor_b200_checkpointed_activation_launch(const thor_b200_checkpointed_activation_desc* d, const void* x, const void* gate, void* y, void* codes, void* scales,
                                             void* gate_codes, void* gate_scales, void* stream_v) {
    using namespace tb;
    const char* who = "checkpointed_activation";
    if (int st = checkActivation(who, d)) return st;
    if (d->rows == 0) return THOR_B200_OK;
    TB_REQUIRE(x != nullptr && y != nullptr && (!d->gated || gate != nullptr), "%s: null tensor pointer", who);
    if (int st = checkCheckpoint(who, codes, scales)) return st;
    if (d->gated)
        if (int st = checkCheckpoint(who, gate_codes, gate_scales)) return st;
    Walk w;
    dim3 grid;
    const bool dense = denseRows(d->x_stride, d->rows, d->cols) && denseRows(d->y_stride, d->rows, d->cols) && (!d->gated || denseRows(d->gate_stride, d->rows, d->cols));
    if (int st = planWalk(d->rows, d->cols, dense, &w, &grid)) return st;
    const Writer out = writerOf(codes, scales, w.cols, d->code_dtype), gate_out = writerOf(gate_codes, gate_scales, w.cols, d->code_dtype);
    const ActivationStrides strides{d->x_stride, d->gate_stride, d->y_stride};
    cudaStream_t stream = static_cast<cudaStream_t>(stream_v);
    const bool aligned = rowsAligned(x, d->x_stride, d->dtype, d->rows) && rowsAligned(y, d->y_stride, d->dtype, d->rows) &&
                         (!d->gated || rowsAligned(gate, d->gate_stride, d->dtype, d->rows)) && d->cols % ck8::kVec == 0;
    return byDtype(d->dtype, [&](auto t) {
        using T = decltype(t);
        return byFlag(aligned, [&](auto a) {
            return byFlag(d->gated != 0, [&](auto gated) {
                return byFlag(d->kind == THOR_B200_ACTIVATION_SWISH, [&](auto swish) {
                    constexpr int kind = decltype(swish)::value ? THOR_B200_ACTIVATION_SWISH : THOR_B200_ACTIVATION_GELU;
                    TB_CUDA(launchDependent(activationKernel<T, kind, decltype(gated)::value, decltype(a)::value>, grid, dim3(kThreads), 0, stream,
                                            static_cast<const T*>(x), static_cast<const T*>(gate), static_cast<T*>(y), strides, out, gate_out, w));
                    countLaunch();
                    return static_cast<int>(THOR_B200_OK);
                });
            });
        });
    });
}

int thor_b200_checkpointed_activation_backward_launch(const thor_b200_checkpointed_activation_desc* d, const void* grad_output, const void* codes, const void* scales,
                                                      const void* gate_codes, const void* gate_scales, void* grad_input, void* grad_gate, void* stream_v) {
    using namespace tb;
    const char* who = "checkpointed_activation_backward";
    if (int st = checkActivation(who, d)) return st;
    if (d->rows == 0) return THOR_B200_OK;
    TB_REQUIRE(grad_output != nullptr && grad_input != nullptr && (!d->gated || grad_gate != nullptr), "%s: null tensor pointer", who);
    if (int st = checkCheckpoint(who, codes, scales)) return st;
    if (d->gated)
        if (int st = checkCheckpoint(who, gate_codes, gate_scales)) return st;
    Walk w;
    dim3 grid;
    const bool dense = denseRows(d->x_stride, d->rows, d->cols) && denseRows(d->y_stride, d->rows, d->cols) && (!d->gated || denseRows(d->gate_stride, d->rows, d->cols));
    if (int st = planWalk(d->rows, d->cols, dense, &w, &grid)) return st;
    const Reader in = readerOf(codes, scales, w.cols, d->code_dtype), gate_in = readerOf(gate_codes, gate_scales, w.cols, d->code_dtype);
    const ActivationStrides strides{d->x_stride, d->gate_stride, d->y_stride};
    cudaStream_t stream = static_cast<cudaStream_t>(stream_v);
    const bool aligned = rowsAligned(grad_output, d->y_stride, d->dtype, d->rows) && rowsAligned(grad_input, d->x_stride, d->dtype, d->rows) &&
                         (!d->gated || rowsAligned(grad_gate, d->gate_stride, d->dtype, d->rows)) && d->cols % ck8::kVec == 0;
    return byDtype(d->dtype, [&](auto t) {
        using T = decltype(t);
        return byFlag(aligned, [&](auto a) {
            return byFlag(d->gated != 0, [&](auto gated) {
                return byFlag(d->kind == THOR_B200_ACTIVATION_SWISH, [&](auto swish) {
                    constexpr int kind = decltype(swish)::value ? THOR_B200_ACTIVATION_SWISH : THOR_B200_ACTIVATION_GELU;
                    TB_CUDA(launchDependent(activationBackwardKernel<T, kind, decltype(gated)::value, decltype(a)::value>, grid, dim3(kThreads), 0, stream,
                                            static_cast<const T*>(grad_output), in, gate_in, static_cast<T*>(grad_input), static_cast<T*>(grad_gate), strides, w));
                    countLaunch();
                    return static_cast<int>(THOR_B200_OK);
                });
            });
        });
    });
}

}  // extern "C"
