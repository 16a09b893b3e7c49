// Packing a tensor into an 8-bit activation checkpoint and unpacking it (the format stands in checkpoint8.cuh): streaming kernels, each
// element read and written once.
#include "checkpoint_walk.cuh"

namespace tb {
namespace {

using namespace ck8;

template <class T, bool ALIGNED>
__global__ void __launch_bounds__(kThreads) packKernel(Rows<T> x, Writer out, Walk w) {
    gridDependencyWait();
    gridLaunchDependents();
    uint32_t row, col, cols;
    locate(w, row, col, cols);
    float2 v[8];
    load16<ALIGNED>(x, x.p + rowStart(row, x.stride) + col, col, cols, v);
    writeCodes(codesAt(out, row, col), scaleAt(out, row, col), out.code, col, cols, v);
}

template <class T, bool ALIGNED>
__global__ void __launch_bounds__(kThreads) unpackKernel(Reader in, T* __restrict__ y, uint32_t y_stride, Walk w) {
    gridDependencyWait();
    gridLaunchDependents();
    uint32_t row, col, cols;
    locate(w, row, col, cols);
    RawCodes raw;
    fetchCodes(codesAt(in, row, col), scaleAt(in, row, col), col, cols, raw);
    float2 v[8];
    expandCodes<false>(in.code, col, cols, raw, v);  // columns past the row's end are not stored
    const uint32_t lane = threadIdx.x % 32;
    store16<ALIGNED>(y + rowStart(row, y_stride) + col, col, cols, v, lane > 0 && col > 0, lane < 31);
}

// Odd rows of at least 2048 columns.
template <class T>
__global__ void __launch_bounds__(kThreads) unpackShiftedKernel(Reader in, T* __restrict__ y, uint32_t y_stride, uint32_t cols) {
    gridDependencyWait();
    gridLaunchDependents();
    const uint32_t row = blockIdx.y;
    T* const out = y + rowStart(row, y_stride);
    const Place place = placeOf(out, cols);
    if (place.first >= cols + place.m) return;
    float2 v[8];
    expandPlace<T, true>(in.code, place, fetchPlace(in, place, row), v);
    storePlace(place, out, v);
}

}  // namespace
}  // namespace tb

extern "C" {

uint64_t thor_b200_checkpoint_code_pitch(uint64_t cols) { return tb::ck8::codePitch(cols); }
uint64_t thor_b200_checkpoint_scale_pitch(uint64_t cols) { return tb::ck8::scalePitch(cols); }

int thor_b200_checkpoint_pack_launch(const thor_b200_checkpoint_desc* d, const void* x, void* codes, void* scales, void* stream_v) {
    using namespace tb;
    using namespace tb::ck8;
    const char* who = "checkpoint_pack";
    TB_REQUIRE(d != nullptr, "%s: null description", who);
    if (int st = checkShape(who, d->dtype, d->code_dtype, d->rows, d->cols)) return st;
    if (int st = checkRowStride(who, "the tensor", d->stride, d->rows, d->cols)) return st;
    if (d->rows == 0) return THOR_B200_OK;
    if (int st = checkTensor(who, x, d->dtype)) return st;
    if (int st = checkCheckpoint(who, codes, scales)) return st;
    Walk w;
    dim3 grid, block;
    if (int st = planWalk(d->rows, d->cols, denseRows(d->stride, d->rows, d->cols), &w, &grid, &block)) return st;
    const Writer out = writerOf(codes, scales, w.cols, d->code_dtype);
    cudaStream_t stream = static_cast<cudaStream_t>(stream_v);
    const bool aligned = rowsAligned(x, d->stride, d->dtype, d->rows) && d->cols % kVec == 0;
    return byDtype(d->dtype, [&](auto t) {
        using T = decltype(t);
        return byFlag(aligned, [&](auto a) {
            TB_CUDA(launchDependent(packKernel<T, decltype(a)::value>, grid, block, 0, stream, rowsOf<T>(x, d->stride, d->rows, d->cols), out, w));
            countLaunch();
            return static_cast<int>(THOR_B200_OK);
        });
    });
}

int thor_b200_checkpoint_unpack_launch(const thor_b200_checkpoint_desc* d, const void* codes, const void* scales, void* y, void* stream_v) {
    using namespace tb;
    using namespace tb::ck8;
    const char* who = "checkpoint_unpack";
    TB_REQUIRE(d != nullptr, "%s: null description", who);
    if (int st = checkShape(who, d->dtype, d->code_dtype, d->rows, d->cols)) return st;
    if (int st = checkRowStride(who, "the tensor", d->stride, d->rows, d->cols)) return st;
    if (d->rows == 0) return THOR_B200_OK;
    if (int st = checkTensor(who, y, d->dtype)) return st;
    if (int st = checkCheckpoint(who, codes, scales)) return st;
    Walk w;
    dim3 grid, block;
    if (int st = planWalk(d->rows, d->cols, denseRows(d->stride, d->rows, d->cols), &w, &grid, &block)) return st;
    const Reader in = readerOf(codes, scales, w.cols, d->code_dtype);
    cudaStream_t stream = static_cast<cudaStream_t>(stream_v);
    const bool aligned = rowsAligned(y, d->stride, d->dtype, d->rows) && d->cols % kVec == 0;
    return byDtype(d->dtype, [&](auto t) {
        using T = decltype(t);
        if (!aligned && w.row_a_cta) {
            shiftedGrid<T>(d->rows, d->cols, &grid, &block);
            TB_CUDA(launchDependent(unpackShiftedKernel<T>, grid, block, 0, stream, in, static_cast<T*>(y), strideOf(d->stride, d->rows), static_cast<uint32_t>(d->cols)));
            countLaunch();
            return static_cast<int>(THOR_B200_OK);
        }
        return byFlag(aligned, [&](auto a) {
            TB_CUDA(launchDependent(unpackKernel<T, decltype(a)::value>, grid, block, 0, stream, in, static_cast<T*>(y), strideOf(d->stride, d->rows), w));
            countLaunch();
            return static_cast<int>(THOR_B200_OK);
        });
    });
}

}  // extern "C"
