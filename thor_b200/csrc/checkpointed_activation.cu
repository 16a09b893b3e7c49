// Activations that write the 8-bit checkpoint of their input in the forward pass and read it in the backward pass (the format stands in
// checkpoint8.cuh): streaming kernels, each element read and written once.
#include "checkpoint_walk.cuh"

namespace tb {
namespace {

using namespace ck8;

// act(x) and act'(x) of two neighbouring columns: gelu(x) = x Phi(x), swish(x) = x sigma(x), as Expression::gelu and
// Expression::swish define them.
//
// sigma(x) = 1 / (1 + 2^(-x log2 e)) and sigma' x + sigma = value (1 - sigma) + sigma.  For fp32 tensors e = exp(-|x|) is the toolkit's: of the approximation's
// argument the rounding alone (2^-17 of an exponent at x = -90) is more than the rest of the arithmetic errs.  sigma(|x|) = 1 / (1 + e) and sigma(-|x|) = e / (1 + e) are each
// other's 1 - sigma without a difference, and e reaches below the smallest normal number, where swish(-88) = -5.3e-37 still is one.  Memory bound all the same: [8192, 8192]
// 89.9 us forward and 88.3 backward, [8192, 8191] 96.2 and 96.8 (90.8 and 90.0 with the approximation).
// Phi(-|x|) = e^(-x^2/2) R(|x|), where R(a) = erfcx(a / sqrt 2) / 2 is smooth and falls from 1/2 like 0.4 / a: R is a polynomial in
// t = 1 / (1 + p a) without a constant term, fitted here for the least relative error over 0 <= a <= 15, past which the
// exponential is below the smallest normal number.  The form keeps the relative accuracy of the far tail, and the exponential is the one
// that the derivative needs.  Degree 9: 2.1e-7 of R as evaluated in fp32 (fp32 tensors); degree 6: 4.8e-6, a hundredth of
// half a unit of fp16 (16-bit tensors), three instructions a pair less.  For fp32 what the exponent's roundings lose is carried into the exponential: gelu is off by at
// most 8 units of 2^-24 of itself, by 66 where the exponent keeps its own rounding ([8192, 8192] 89 -> 90 us forward, 142 -> 145 gated backward; [8192, 8191] 102 -> 108
// forward, 101 -> 105 and, gated, 142 -> 160 backward).
// Two elements an instruction (f32x2) and one exponential and one reciprocal an element; with the toolkit's erfcf and expf the backward kernel
// waited for the arithmetic pipes.
template <class T, int KIND>
__device__ __forceinline__ void activation2(float2 x, float2& value, float2& slope) {
    constexpr bool FULL = sizeof(T) == 4;
    if constexpr (KIND == THOR_B200_ACTIVATION_SWISH && FULL) {
        const float2 e = make_float2(expf(-fabsf(x.x)), expf(-fabsf(x.y)));
        const float2 d = add2(e, both(1.0f));
        const float2 r = make_float2(reciprocalApprox(d.x), reciprocalApprox(d.y)), er = mul2(e, r);
        const bool right_x = x.x > 0.0f, right_y = x.y > 0.0f;
        const float2 s = make_float2(right_x ? r.x : er.x, right_y ? r.y : er.y), rest = make_float2(right_x ? er.x : r.x, right_y ? er.y : r.y);
        value = mul2(x, s);
        slope = fma2(value, rest, s);
    } else if constexpr (KIND == THOR_B200_ACTIVATION_SWISH && std::is_same<T, __nv_bfloat16>::value) {
        // The reciprocal of 2^-16 (1 + 2^y): of 1 + 2^y it would be zero below 2^-126, left of x = -87.3.  fp16 has no results so small.
        const float2 y = fma2(x, both(-1.44269504f), both(-16.0f)), low = both(1.52587890625e-5f);
        const float2 d = add2(make_float2(exp2Approx(y.x), exp2Approx(y.y)), low);
        const float2 s = mul2(make_float2(reciprocalApprox(d.x), reciprocalApprox(d.y)), low);
        value = mul2(x, s);
        slope = fma2(value, fma2(s, both(-1.0f), both(1.0f)), s);
    } else if constexpr (KIND == THOR_B200_ACTIVATION_SWISH) {
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
        float2 e;
        if constexpr (FULL) {
            // y = -square log2(e) / 2 and what it lacks: its own rounding, that of the constant, and what square lost.  Past 32 nothing is left of e.
            const float2 c = make_float2(fminf(a.x, 32.0f), fminf(a.y, 32.0f)), square = mul2(c, c), n = mul2(square, both(0.72134752f));
            const float2 lost = fma2(c, c, make_float2(-square.x, -square.y));
            float2 low = fma2(square, both(-0.72134752f), n);
            low = fma2(lost, both(-0.72134752f), low);
            low = fma2(square, both(-9.629814956e-9f), low);
            e = make_float2(exp2Approx(-n.x), exp2Approx(-n.y));
            e = fma2(mul2(e, both(0.69314718f)), low, e);
        } else {
            const float2 y = mul2(mul2(x, x), both(-0.72134752f));
            e = make_float2(exp2Approx(y.x), exp2Approx(y.y));
        }
        const float2 rt = mul2(r, t);
        const float2 q = mul2(rt, e), p = mul2(fma2(a, both(-0.39894228f), rt), e);  // Phi and slope at -|x|; those at x and -x add up to one
        const float2 phi = make_float2(x.x > 0.0f ? 1.0f - q.x : q.x, x.y > 0.0f ? 1.0f - q.y : q.y);
        value = mul2(x, phi);
        slope = make_float2(x.x > 0.0f ? 1.0f - p.x : p.x, x.y > 0.0f ? 1.0f - p.y : p.y);
    }
}

// CTAs of 256 threads that an SM shall hold, which caps the registers (left alone the compiler takes 56 to 80 and too few warps are there to wait with).
// GELU backward [8192, 8192] bf16: 76.1 us uncapped, 57.2 with five, 52.9 with six; gated Swish backward 90.4, 80.8, 81.6.  Odd rows of fp32
// spill under any of these; the gated forward pass takes three (Swish [8192, 8191] 181 us uncapped, 151 with three; GELU 182 and 163).
template <class T, bool GATED, bool ALIGNED, bool BACKWARD>
constexpr int residentCtas() {
    if (sizeof(T) == 4) return ALIGNED || (!GATED && !BACKWARD) ? 5 : (BACKWARD ? 1 : 3);
    return GATED || (BACKWARD && !ALIGNED) ? 5 : 6;
}

template <class T, int KIND, bool GATED, bool ALIGNED>
__global__ void __launch_bounds__(kThreads, residentCtas<T, GATED, ALIGNED, false>()) activationKernel(Rows<T> x, Rows<T> gate, T* __restrict__ y, uint32_t y_stride, Writer out, Writer gate_out, Walk w) {
    gridDependencyWait();
    gridLaunchDependents();
    uint32_t row, col, cols;
    locate(w, row, col, cols);
    Raw<T, ALIGNED> raw, raw_gate;
    const T* const x_at = x.p + rowStart(row, x.stride) + col;
    const T* const gate_at = gate.p + rowStart(row, gate.stride) + col;
    fetch16(x, x_at, col, cols, raw);
    if constexpr (GATED) fetch16(gate, gate_at, col, cols, raw_gate);
    float2 v[8], r[8];
    expand16(x_at, col, cols, raw, v);
    writeCodes(codesAt(out, row, col), scaleAt(out, row, col), out.code, col, cols, v);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        float2 slope;
        activation2<T, KIND>(v[i], r[i], slope);
    }
    if constexpr (GATED) {
        expand16(gate_at, col, cols, raw_gate, v);
        writeCodes(codesAt(gate_out, row, col), scaleAt(gate_out, row, col), gate_out.code, col, cols, v);
#pragma unroll
        for (int i = 0; i < 8; ++i) r[i] = mul2(r[i], v[i]);
    }
    const uint32_t lane = threadIdx.x % 32;
    store16<ALIGNED>(y + rowStart(row, y_stride) + col, col, cols, r, lane > 0 && col > 0, lane < 31);
}

template <class T, int KIND, bool GATED, bool ALIGNED>
__global__ void __launch_bounds__(kThreads, residentCtas<T, GATED, ALIGNED, true>()) activationBackwardKernel(Rows<T> grad, Reader in, Reader gate_in, T* __restrict__ grad_x, uint32_t grad_x_stride,
                                                                     T* __restrict__ grad_gate, uint32_t grad_gate_stride, Walk w) {
    gridDependencyWait();
    gridLaunchDependents();
    uint32_t row, col, cols;
    locate(w, row, col, cols);
    Raw<T, ALIGNED> raw;
    RawCodes codes, gate_codes;
    const T* const grad_at = grad.p + rowStart(row, grad.stride) + col;
    fetch16(grad, grad_at, col, cols, raw);
    fetchCodes(codesAt(in, row, col), scaleAt(in, row, col), col, cols, codes);
    if constexpr (GATED) fetchCodes(codesAt(gate_in, row, col), scaleAt(gate_in, row, col), col, cols, gate_codes);
    float2 d[8], v[8], dx[8];
    expandCodes<false, true>(in.code, col, cols, codes, v);  // columns past the row's end are not stored
    expand16(grad_at, col, cols, raw, d);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        float2 value, slope;
        activation2<T, KIND>(v[i], value, slope);
        dx[i] = mul2(d[i], slope);
        d[i] = mul2(d[i], value);  // the gate's gradient
    }
    const uint32_t lane = threadIdx.x % 32;
    const bool before = lane > 0 && col > 0, after = lane < 31;
    if constexpr (GATED) {
        store16<ALIGNED>(grad_gate + rowStart(row, grad_gate_stride) + col, col, cols, d, before, after);
        expandCodes<false, true>(gate_in.code, col, cols, gate_codes, v);
#pragma unroll
        for (int i = 0; i < 8; ++i) dx[i] = mul2(dx[i], v[i]);
    }
    store16<ALIGNED>(grad_x + rowStart(row, grad_x_stride) + col, col, cols, dx, before, after);
}

// Odd rows of at least 2048 columns whose tensors all start at the same place of 32 bytes.  (Columns beside the row's may be loaded; they are not stored.)
template <class T, int KIND, bool GATED>
__global__ void __launch_bounds__(kThreads, sizeof(T) == 4 ? 4 : GATED ? 5 : 6) activationBackwardShiftedKernel(Rows<T> grad, Reader in, Reader gate_in, T* __restrict__ grad_x,
                                                                     uint32_t grad_x_stride, T* __restrict__ grad_gate, uint32_t grad_gate_stride, uint32_t cols) {
    gridDependencyWait();
    gridLaunchDependents();
    const uint32_t row = blockIdx.y;
    const T* const grad_row = grad.p + rowStart(row, grad.stride);
    const Place place = placeOf(grad_row, cols);
    if (place.first >= cols + place.m) return;
    constexpr bool ONCE = !GATED || sizeof(T) == 4;
    uint32_t raw[kRegs<T>];
    PlaceCodes gate_codes;
    loadPlace(place, grad, grad_row, raw);
    const PlaceCodes codes = fetchPlace(in, place, row);
    if constexpr (GATED) gate_codes = fetchPlace(gate_in, place, row);
    float2 d[8], v[8], dx[8];
    expandPlace<T, ONCE, true>(in.code, place, codes, v);
    widen16<T>(raw, d);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        float2 value, slope;
        activation2<T, KIND>(v[i], value, slope);
        dx[i] = mul2(d[i], slope);
        d[i] = mul2(d[i], value);
    }
    if constexpr (GATED) {
        storePlace(place, grad_gate + rowStart(row, grad_gate_stride), d);
        expandPlace<T, ONCE, true>(gate_in.code, place, gate_codes, v);
#pragma unroll
        for (int i = 0; i < 8; ++i) dx[i] = mul2(dx[i], v[i]);
    }
    storePlace(place, grad_x + rowStart(row, grad_x_stride), dx);
}

int checkActivation(const char* who, const thor_b200_checkpointed_activation_desc* d) {
    TB_REQUIRE(d != nullptr, "%s: null description", who);
    TB_REQUIRE(d->kind == THOR_B200_ACTIVATION_GELU || d->kind == THOR_B200_ACTIVATION_SWISH, "%s: unknown activation %d", who, d->kind);
    if (int st = checkShape(who, d->dtype, d->code_dtype, d->rows, d->cols)) return st;
    if (int st = checkRowStride(who, "x", d->x_stride, d->rows, d->cols)) return st;
    if (d->gated)
        if (int st = checkRowStride(who, "gate", d->gate_stride, d->rows, d->cols)) return st;
    return checkRowStride(who, "y", d->y_stride, d->rows, d->cols);
}
// The tensors that play x, gate and y (their gradients in the backward pass) and the checkpoints.
int checkOperands(const char* who, const thor_b200_checkpointed_activation_desc& d, const void* x, const void* gate, const void* y, const void* codes, const void* scales,
                  const void* gate_codes, const void* gate_scales) {
    if (int st = checkTensor(who, x, d.dtype)) return st;
    if (int st = checkTensor(who, y, d.dtype)) return st;
    if (int st = checkCheckpoint(who, codes, scales)) return st;
    if (!d.gated) return THOR_B200_OK;
    if (int st = checkTensor(who, gate, d.dtype)) return st;
    return checkCheckpoint(who, gate_codes, gate_scales);
}
int planActivation(const thor_b200_checkpointed_activation_desc& d, const void* x, const void* gate, const void* y, Walk* w, dim3* grid, dim3* block, bool* aligned) {
    *aligned = d.cols % kVec == 0 && rowsAligned(x, d.x_stride, d.dtype, d.rows) && rowsAligned(y, d.y_stride, d.dtype, d.rows) &&
               (!d.gated || rowsAligned(gate, d.gate_stride, d.dtype, d.rows));
    const bool dense = denseRows(d.x_stride, d.rows, d.cols) && denseRows(d.y_stride, d.rows, d.cols) && (!d.gated || denseRows(d.gate_stride, d.rows, d.cols));
    return planWalk(d.rows, d.cols, dense, w, grid, block);
}
// f(element, kind, gated, aligned) with the last three as integral constants
template <class F>
int byVariant(const thor_b200_checkpointed_activation_desc& d, bool aligned, F&& f) {
    return byDtype(d.dtype, [&](auto t) {
        return byFlag(d.kind == THOR_B200_ACTIVATION_SWISH, [&](auto swish) {
            return byFlag(d.gated != 0, [&](auto gated) {
                return byFlag(aligned, [&](auto a) {
                    return f(t, std::integral_constant<int, decltype(swish)::value ? THOR_B200_ACTIVATION_SWISH : THOR_B200_ACTIVATION_GELU>{}, gated, a);
                });
            });
        });
    });
}

}  // namespace
}  // namespace tb

extern "C" {

int thor_b200_checkpointed_activation_launch(const thor_b200_checkpointed_activation_desc* d, const void* x, const void* gate, void* y, void* codes, void* scales,
                                             void* gate_codes, void* gate_scales, void* stream_v) {
    using namespace tb;
    using namespace tb::ck8;
    const char* who = "checkpointed_activation";
    if (int st = checkActivation(who, d)) return st;
    if (d->rows == 0) return THOR_B200_OK;
    if (int st = checkOperands(who, *d, x, gate, y, codes, scales, gate_codes, gate_scales)) return st;
    Walk w;
    dim3 grid, block;
    bool aligned = false;
    if (int st = planActivation(*d, x, gate, y, &w, &grid, &block, &aligned)) return st;
    const Writer out = writerOf(codes, scales, w.cols, d->code_dtype), gate_out = writerOf(gate_codes, gate_scales, w.cols, d->code_dtype);
    return byVariant(*d, aligned, [&](auto t, auto kind, auto gated, auto a) {
        using T = decltype(t);
        TB_CUDA(launchDependent(activationKernel<T, decltype(kind)::value, decltype(gated)::value, decltype(a)::value>, grid, block, 0,
                                static_cast<cudaStream_t>(stream_v), rowsOf<T>(x, d->x_stride, d->rows, d->cols), rowsOf<T>(gate, d->gate_stride, d->rows, d->cols),
                                static_cast<T*>(y), strideOf(d->y_stride, d->rows), out, gate_out, w));
        countLaunch();
        return static_cast<int>(THOR_B200_OK);
    });
}

int thor_b200_checkpointed_activation_backward_launch(const thor_b200_checkpointed_activation_desc* d, const void* grad_output, const void* codes, const void* scales,
                                                      const void* gate_codes, const void* gate_scales, void* grad_input, void* grad_gate, void* stream_v) {
    using namespace tb;
    using namespace tb::ck8;
    const char* who = "checkpointed_activation_backward";
    if (int st = checkActivation(who, d)) return st;
    if (d->rows == 0) return THOR_B200_OK;
    if (int st = checkOperands(who, *d, grad_input, grad_gate, grad_output, codes, scales, gate_codes, gate_scales)) return st;
    Walk w;
    dim3 grid, block;
    bool aligned = false;
    if (int st = planActivation(*d, grad_input, grad_gate, grad_output, &w, &grid, &block, &aligned)) return st;
    const Reader in = readerOf(codes, scales, w.cols, d->code_dtype), gate_in = readerOf(gate_codes, gate_scales, w.cols, d->code_dtype);
    const bool shifted = !aligned && w.row_a_cta && rowsCongruent(grad_output, d->y_stride, grad_input, d->x_stride, d->dtype) &&
                         (!d->gated || rowsCongruent(grad_output, d->y_stride, grad_gate, d->gate_stride, d->dtype));
    return byVariant(*d, aligned, [&](auto t, auto kind, auto gated, auto a) {
        using T = decltype(t);
        if constexpr (!decltype(a)::value) {
            if (shifted) {
                shiftedGrid<T>(d->rows, d->cols, &grid, &block);
                TB_CUDA(launchDependent(activationBackwardShiftedKernel<T, decltype(kind)::value, decltype(gated)::value>, grid, block, 0, static_cast<cudaStream_t>(stream_v),
                                        rowsOf<T>(grad_output, d->y_stride, d->rows, d->cols), in, gate_in, static_cast<T*>(grad_input), strideOf(d->x_stride, d->rows),
                                        static_cast<T*>(grad_gate), strideOf(d->gate_stride, d->rows), static_cast<uint32_t>(d->cols)));
                countLaunch();
                return static_cast<int>(THOR_B200_OK);
            }
        }
        TB_CUDA(launchDependent(activationBackwardKernel<T, decltype(kind)::value, decltype(gated)::value, decltype(a)::value>, grid, block, 0,
                                static_cast<cudaStream_t>(stream_v), rowsOf<T>(grad_output, d->y_stride, d->rows, d->cols), in, gate_in, static_cast<T*>(grad_input),
                                strideOf(d->x_stride, d->rows), static_cast<T*>(grad_gate), strideOf(d->gate_stride, d->rows), w));
        countLaunch();
        return static_cast<int>(THOR_B200_OK);
    });
}

}  // extern "C"
