// How the elementwise kernels of the 8-bit checkpoints walk a [rows, cols] tensor, and the checks of their arguments.
//
// One chunk of sixteen columns per thread and one wave of CTAs after another: each thread has all its loads in flight before it uses the first.  A
// tensor whose rows lie dense and whose width is a multiple of 32 is walked as one row; other rows of at least 2048 columns get CTAs of their
// own (blockIdx.y is the row: no index division, addresses the same for the whole CTA; Swish backward [8192, 8191] bf16 66.8 -> 59.9 us),
// which kernels that only read a checkpoint use to walk odd rows on the tensor's own 32 bytes; shorter ones share CTAs.
#pragma once

#include "checkpoint8.cuh"

namespace tb {
namespace ck8 {

constexpr int kThreads = 256;

// Chunk of sixteen columns -> row and first column.  Every row has `chunks` of them, an even number, so that a block never spans rows.
struct Walk {
    uint64_t units;
    uint32_t chunks, cols;
    bool row_a_cta;
};
// This thread's chunk; cols = 0 where there is none left.
__device__ __forceinline__ void locate(const Walk& w, uint32_t& row, uint32_t& col, uint32_t& cols) {
    if (w.row_a_cta) {
        row = blockIdx.y;
        col = (blockIdx.x * blockDim.x + threadIdx.x) * kVec;
        cols = w.cols;
        return;
    }
    const uint64_t unit = static_cast<uint64_t>(blockIdx.x) * kThreads + threadIdx.x;
    row = 0;
    cols = unit < w.units ? w.cols : 0;
    if (w.units == w.chunks) {
        col = static_cast<uint32_t>(unit) * kVec;
    } else if (w.units <= 0xffffffffull) {
        const uint32_t r = static_cast<uint32_t>(unit) / w.chunks;
        row = r;
        col = (static_cast<uint32_t>(unit) - r * w.chunks) * kVec;
    } else {
        row = static_cast<uint32_t>(unit / w.chunks);
        col = static_cast<uint32_t>(unit - static_cast<uint64_t>(row) * w.chunks) * kVec;
    }
}

// A CTA for every row, or several where the row is longer than its threads take.
inline void rowGrid(uint64_t rows, uint32_t chunks, dim3* grid, dim3* block) {
    const uint32_t segments = (chunks + kThreads - 1) / kThreads;
    *grid = dim3(segments, static_cast<unsigned>(rows));
    *block = dim3(((chunks + segments - 1) / segments + 31) / 32 * 32);
}
// The same for odd rows that are walked on the tensor's own 32 bytes.
template <class T>
void shiftedGrid(uint64_t rows, uint64_t cols, dim3* grid, dim3* block) {
    rowGrid(rows, static_cast<uint32_t>((cols + kShifts<T> - 1 + kVec - 1) / kVec), grid, block);
}

inline int planWalk(uint64_t rows, uint64_t cols, bool dense, Walk* w, dim3* grid, dim3* block) {
    if (dense && cols % kBlock == 0 && rows * cols < 0x80000000ull) {  // the checkpoint's rows are dense then, too
        cols *= rows;
        rows = 1;
    }
    w->chunks = static_cast<uint32_t>(scalePitch(cols) * (kBlock / kVec));
    w->cols = static_cast<uint32_t>(cols);
    w->units = rows * w->chunks;
    w->row_a_cta = rows > 1 && rows <= 65535 && w->chunks >= 128;
    if (w->row_a_cta) {
        rowGrid(rows, w->chunks, grid, block);
        return THOR_B200_OK;
    }
    const uint64_t ctas = (w->units + kThreads - 1) / kThreads;
    TB_REQUIRE(ctas <= 0x7FFFFFFFull, "checkpoint: too many elements for one grid");
    *grid = dim3(static_cast<unsigned>(ctas));
    *block = dim3(kThreads);
    return THOR_B200_OK;
}

inline int checkShape(const char* who, int dtype, int code_dtype, uint64_t rows, uint64_t cols) {
    TB_REQUIRE(valueDtypeOk(dtype), "%s: tensors must be fp32, fp16 or bf16, got %s", who, dtypeName(dtype));
    TB_REQUIRE(codeDtypeOk(code_dtype), "%s: codes must be fp8_e4m3, fp8_e5m2 or int8, got %s", who, dtypeName(code_dtype));
    TB_REQUIRE(cols > 0 && cols <= 0x7fffffffull, "%s: rows must have 1 to 2^31 - 1 columns", who);
    TB_REQUIRE(rows <= (1ull << 62) / (cols + kBlock), "%s: rows * cols overflows", who);
    TB_REQUIRE(rows <= 0xffffffffull, "%s: more than 2^32 - 1 rows", who);
    return THOR_B200_OK;
}
inline int checkTensor(const char* who, const void* p, int dtype) {
    TB_REQUIRE(p != nullptr, "%s: null tensor pointer", who);
    TB_REQUIRE(isAligned(p, dtypeSize(dtype)), "%s: a tensor pointer is not aligned to its elements", who);
    return THOR_B200_OK;
}
inline int checkCheckpoint(const char* who, const void* codes, const void* scales) {
    TB_REQUIRE(codes != nullptr && scales != nullptr, "%s: null checkpoint pointer", who);
    TB_REQUIRE(isAligned(codes, 16), "%s: codes must be 16-byte aligned", who);
    return THOR_B200_OK;
}
inline Writer writerOf(void* codes, void* scales, uint64_t cols, int code) {
    return Writer{static_cast<uint8_t*>(codes), static_cast<uint8_t*>(scales), static_cast<uint32_t>(codePitch(cols)), static_cast<uint32_t>(scalePitch(cols)), code};
}
inline Reader readerOf(const void* codes, const void* scales, uint64_t cols, int code) {
    return Reader{static_cast<const uint8_t*>(codes), static_cast<const uint8_t*>(scales), static_cast<uint32_t>(codePitch(cols)), static_cast<uint32_t>(scalePitch(cols)), code};
}
inline bool denseRows(int64_t stride, uint64_t rows, uint64_t cols) { return rows <= 1 || static_cast<uint64_t>(stride) == cols; }

}  // namespace ck8
}  // namespace tb
