// LayerNorm backward: the input's gradient and the column sums of the parameters' gradients in one pass over the rows.
//
// Rows of up to 8192 columns: one persistent CTA an SM, whose teams walk their rows.  A thread owns sixteen columns for the whole kernel and
// keeps their two column sums in registers; per row it needs one exchange with its team, for the two row sums.  At the end the CTA adds its
// teams and leaves one partial row of each sum in the workspace, and a second kernel adds the partial rows in order.  Up to 512 rows take one
// launch whose CTAs share the two tasks.  Rows of more columns take two kernels that read the row twice and once more.
#include <algorithm>

#include "layernorm_common.cuh"

namespace tb {
namespace {

using namespace ln;

constexpr uint64_t kFusedCols = static_cast<uint64_t>(kMaxThreads) * kVec;  // longest row of the fused kernel
constexpr uint32_t kPartialRows = 148;                                       // one CTA an SM

template <class T>
struct Backward {
    Rows<T> grad;      // of the output
    Rows<T> x;         // the saved input, p == nullptr: from the checkpoint
    Rows<T> grad_sum;  // p == nullptr: none
    T* grad_input;
    const float* mean;
    const float* rstd;
    Param gamma;
    Reader kept;
    uint32_t rows, cols, team;
    float inverse;  // 1 / cols
    float* partial;    // [partial rows][2][padded], nullptr: no parameter gradients
    uint32_t padded;
    uint32_t slab_rows;  // rows of a partial row, in the kernels for long rows
};

// Normalised values of sixteen columns; what lies past the row's end meets a gradient of zero.
template <bool KEPT, bool ALIGNED, class T>
struct Normal {
    Raw<T, ALIGNED> raw;
    __device__ __forceinline__ void fetch(const Backward<T>& b, uint32_t row, uint32_t col, uint32_t cols) { fetch16(b.x, b.x.p + rowStart(row, b.x.stride) + col, col, cols, raw); }
    template <bool MIXED = false>
    __device__ __forceinline__ void expand(const Backward<T>& b, uint32_t row, uint32_t col, uint32_t cols, float mean, float rstd, float2 (&n)[8]) const {
        expand16<T, ALIGNED, MIXED>(b.x.p + rowStart(row, b.x.stride) + col, col, cols, raw, n);
#pragma unroll
        for (int i = 0; i < 8; ++i) n[i] = mul2(add2(n[i], both(-mean)), both(rstd));
    }
};
template <bool ALIGNED, class T>
struct Normal<true, ALIGNED, T> {
    RawCodes raw;
    __device__ __forceinline__ void fetch(const Backward<T>& b, uint32_t row, uint32_t col, uint32_t cols) { fetchCodes(codesAt(b.kept, row, col), scaleAt(b.kept, row, col), col, cols, raw); }
    template <bool MIXED = false>
    __device__ __forceinline__ void expand(const Backward<T>& b, uint32_t, uint32_t col, uint32_t cols, float, float, float2 (&n)[8]) const {
        expandCodes<!ALIGNED>(b.kept.code, col, cols, raw, n);
    }
};

// w = grad * gamma, and what the row sums of w and w n gain
template <class T>
__device__ __forceinline__ void weigh16(const Backward<T>& b, uint32_t col, uint32_t cols, float2 (&w)[8], const float2 (&n)[8], float2& s1, float2& s2) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        float2 g[4];
        loadParam8(b.gamma, 1.0f, col + 8 * h, cols, g);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            w[4 * h + i] = mul2(w[4 * h + i], g[i]);
            s1 = add2(s1, w[4 * h + i]);
            s2 = fma2(w[4 * h + i], n[4 * h + i], s2);
        }
    }
}
// rstd * (w - c1 - n c2) [+ grad_sum]
template <bool ALIGNED, class T>
__device__ __forceinline__ void finish16(const Backward<T>& b, uint32_t row, uint32_t col, uint32_t cols, float2 (&w)[8], const float2 (&n)[8], float c1, float c2, float rstd,
                                         const Raw<T, ALIGNED>& stream, bool before, bool after) {
    const float2 scale = both(rstd), shift = both(-rstd * c1), slope = both(-rstd * c2);
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = fma2(n[i], slope, fma2(w[i], scale, shift));
    if (b.grad_sum.p != nullptr) {
        float2 r[8];
        expand16(b.grad_sum.p + rowStart(row, b.grad_sum.stride) + col, col, cols, stream, r);
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = add2(w[i], r[i]);
    }
    store16<ALIGNED>(b.grad_input + rowStart(row, b.cols) + col, col, cols, w, before, after);
}

// Asks L2 for the row that a team takes kRowsAhead turns from now.  A register load one turn ahead hides L2's latency, not that of the memory behind it:
// [32768, 8192] bf16 from a checkpoint 266 us without, 248 with it; from the saved input 278 and 249.  Three or five turns ahead are no better
// than two.  Teams of fewer than 64 threads do not ask, nor of fewer than 128 where the input was saved or the width is odd: there the
// requests cost more than they give ([65536, 1024] fp32 131 us with, 127 without).
constexpr uint32_t kRowsAhead = 2;
template <bool ALIGNED>
__device__ __forceinline__ void requestBytes(const void* from, uint32_t bytes) {
    uint64_t first = reinterpret_cast<uintptr_t>(from);
    if constexpr (!ALIGNED) {  // whole 16 bytes of the row only
        const uint64_t last = (first + bytes) & ~15ull;
        first = (first + 15) & ~15ull;
        if (last <= first) return;
        bytes = static_cast<uint32_t>(last - first);
    }
    asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(first), "r"(bytes) : "memory");
}
template <class T, bool ALIGNED>
__device__ __forceinline__ void requestRow(const Backward<T>& b, uint32_t row) {
    if (row >= b.rows) return;
    requestBytes<ALIGNED>(b.grad.p + rowStart(row, b.grad.stride), b.cols * static_cast<uint32_t>(sizeof(T)));
    if (b.x.p == nullptr) requestBytes<true>(codesAt(b.kept, row, 0), b.kept.code_pitch);
    else requestBytes<ALIGNED>(b.x.p + rowStart(row, b.x.stride), b.cols * static_cast<uint32_t>(sizeof(T)));
}

// Teams that leave a quarter of the threads unused or more (a width of 5120 makes one of 320) work on two rows at once, with the registers that are left
// over: twice the arithmetic between two barriers.  [32768, 5120] bf16 from a checkpoint 202 -> 167 us, [32768, 6144] 214 -> 183, [65536, 3008] 211 -> 179.
// From the saved input (194 -> 206 us) and with odd rows (333 -> 404) two rows do not fit the registers, nor in fp32.
constexpr uint32_t kPairThreads = 384;

// ROWS: rows that a team works on at once.
template <class T, int ROWS, bool KEPT, bool ALIGNED>
__global__ void __launch_bounds__(ROWS == 2 ? kPairThreads : kMaxThreads, 1) backwardKernel(const __grid_constant__ Backward<T> b) {
    // the next row is loaded while this one is worked on; odd rows of fp32 have no registers for it ([32768, 5001] bf16 405 -> 333 us)
    constexpr bool kAhead = ALIGNED || sizeof(T) == 2;
    __shared__ Scratch scratch;
    using Params = Staged<T, false>;
    __shared__ uint4 shared[4 * kMaxThreads];  // gamma's planes, then the teams' column sums
    gridDependencyWait();
    gridLaunchDependents();
    const uint32_t team = b.team, team_id = threadIdx.x / team, t = threadIdx.x - team_id * team, teams = blockDim.x / team;
    const uint32_t lane = threadIdx.x % 32, col = t * kVec;
    const bool before = team < 32 ? t > 0 : lane > 0, after = team < 32 ? t + 1 < team : lane < 31;
    const uint32_t step = gridDim.x * teams;
    uint32_t row = blockIdx.x * teams + team_id;
    Raw<T, ALIGNED> grad[ROWS];
    Normal<KEPT, ALIGNED, T> normal[ROWS];
    float rstd[ROWS], mean[ROWS];
    uint32_t cols[ROWS];
    auto fetch = [&](uint32_t first) {
#pragma unroll
        for (int k = 0; k < ROWS; ++k) {
            const uint32_t r = first + k * step;
            const bool there = r < b.rows;
            cols[k] = there ? b.cols : 0;
            fetch16(b.grad, b.grad.p + rowStart(r, b.grad.stride) + col, col, cols[k], grad[k]);
            normal[k].fetch(b, r, col, cols[k]);
            rstd[k] = there ? __ldg(b.rstd + r) : 0.0f;
            mean[k] = !KEPT && there ? __ldg(b.mean + r) : 0.0f;
        }
    };
    float2 dg[8], db[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) dg[i] = db[i] = both(0.0f);
    fetch(row);
    Params::stage(b.gamma, 1.0f, shared, team, b.cols);
    __syncthreads();
    int slot = 0;
    const bool asks = team >= (KEPT && ALIGNED ? 64 : 128) && t == 0;
    // the same number of turns for the whole CTA; a team without a row has cols = 0
    for (uint32_t base = blockIdx.x * teams; base < b.rows; base += ROWS * step, row += ROWS * step) {
        float2 w[ROWS][8], n[ROWS][8], sums[ROWS];
        uint32_t now_cols[ROWS];
        float now_rstd[ROWS];
#pragma unroll
        for (int k = 0; k < ROWS; ++k) {
            expand16(b.grad.p + rowStart(row + k * step, b.grad.stride) + col, col, cols[k], grad[k], w[k]);
            normal[k].expand(b, row + k * step, col, cols[k], mean[k], rstd[k], n[k]);
            now_cols[k] = cols[k];
            now_rstd[k] = rstd[k];
            if (asks) requestRow<T, ALIGNED>(b, row + (kRowsAhead * ROWS + k) * step);
        }
        if constexpr (kAhead) fetch(row + ROWS * step);
        Raw<T, ALIGNED> stream[ROWS];
        if (b.grad_sum.p != nullptr) {
#pragma unroll
            for (int k = 0; k < ROWS; ++k)
                fetch16(b.grad_sum, b.grad_sum.p + rowStart(row + k * step, b.grad_sum.stride) + col, col, now_cols[k], stream[k]);
        }
#pragma unroll
        for (int k = 0; k < ROWS; ++k) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                dg[i] = fma2(w[k][i], n[k][i], dg[i]);
                db[i] = add2(db[i], w[k][i]);
            }
        }
        float2 s1[ROWS], s2[ROWS];
#pragma unroll
        for (int k = 0; k < ROWS; ++k) s1[k] = s2[k] = both(0.0f);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float2 g[4];
            Params::read(shared, team, t, h, g);
#pragma unroll
            for (int k = 0; k < ROWS; ++k) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    w[k][4 * h + i] = mul2(w[k][4 * h + i], g[i]);
                    s1[k] = add2(s1[k], w[k][4 * h + i]);
                    s2[k] = fma2(w[k][4 * h + i], n[k][4 * h + i], s2[k]);
                }
            }
        }
#pragma unroll
        for (int k = 0; k < ROWS; ++k) sums[k] = make_float2(s1[k].x + s1[k].y, s2[k].x + s2[k].y);
        teamSums(sums, team, team_id, scratch, slot);
        slot ^= 1;
#pragma unroll
        for (int k = 0; k < ROWS; ++k)
            finish16<ALIGNED>(b, row + k * step, col, now_cols[k], w[k], n[k], sums[k].x * b.inverse, sums[k].y * b.inverse, now_rstd[k], stream[k], before, after);
        if constexpr (!kAhead) fetch(row + ROWS * step);
    }
    if (b.partial == nullptr) return;
    // A partial row keeps the threads' order: value i of thread t at i * team + t.
    float* const gather = reinterpret_cast<float*>(shared);
    float* out = b.partial + static_cast<uint64_t>(blockIdx.x) * 2 * b.padded;
    for (int which = 0; which < 2; ++which, out += b.padded) {
        if (teams == 1) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float2 v = which == 0 ? dg[i] : db[i];
                out[(2 * i) * team + t] = v.x;
                out[(2 * i + 1) * team + t] = v.y;
            }
            continue;
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float2 v = which == 0 ? dg[i] : db[i];
            gather[(2 * i) * kMaxThreads + threadIdx.x] = v.x;
            gather[(2 * i + 1) * kMaxThreads + threadIdx.x] = v.y;
        }
        __syncthreads();
        for (uint32_t j = threadIdx.x; j < kVec * team; j += blockDim.x) {
            const uint32_t i = j / team, thread = j - i * team;
            float s = 0.0f;
            for (uint32_t k = 0; k < teams; ++k) s += gather[i * kMaxThreads + k * team + thread];
            out[j] = s;
        }
    }
}

// Few rows: one launch in which some CTAs take rows, as above but without column sums, and the others take the sums of 64 columns over all rows and
// round them.  The rows are read twice, from L2, but no partial rows are written and no second kernel waits for them.
constexpr uint32_t kStripLanes = 4, kStrip = kStripLanes * kVec;  // columns of a CTA; the other lanes of a warp take other rows

template <class T, bool KEPT, bool ALIGNED, class O>
__device__ __forceinline__ void columnStrip(const Backward<T>& b, uint32_t strip, float (&part)[kMaxThreads / 32][2][kStrip], O* grad_gamma, O* grad_beta) {
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32, warps = blockDim.x / 32;
    const uint32_t col = strip * kStrip + lane % kStripLanes * kVec, step = warps * (32 / kStripLanes);
    constexpr int kRows = ALIGNED || sizeof(T) == 2 ? 2 : 1;  // loaded before the first is used
    float2 dg[8], db[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) dg[i] = db[i] = both(0.0f);
    for (uint32_t first = warp * (32 / kStripLanes) + lane / kStripLanes; first < b.rows; first += kRows * step) {
        Raw<T, ALIGNED> grad[kRows];
        Normal<KEPT, ALIGNED, T> normal[kRows];
        float mean[kRows], rstd[kRows];
#pragma unroll
        for (int k = 0; k < kRows; ++k) {
            const uint32_t row = first + k * step;
            const bool there = row < b.rows;
            fetch16(b.grad, b.grad.p + rowStart(row, b.grad.stride) + col, col, there ? b.cols : 0, grad[k]);
            normal[k].fetch(b, row, col, there ? b.cols : 0);
            mean[k] = KEPT || !there ? 0.0f : b.mean[row];
            rstd[k] = KEPT || !there ? 0.0f : b.rstd[row];
        }
#pragma unroll
        for (int k = 0; k < kRows; ++k) {
            const uint32_t row = first + k * step, cols = row < b.rows ? b.cols : 0;
            float2 d[8], n[8];
            expand16<T, ALIGNED, true>(b.grad.p + rowStart(row, b.grad.stride) + col, col, cols, grad[k], d);
            normal[k].template expand<true>(b, row, col, cols, mean[k], rstd[k], n);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                dg[i] = fma2(d[i], n[i], dg[i]);
                db[i] = add2(db[i], d[i]);
            }
        }
    }
    __syncwarp();
#pragma unroll
    for (int which = 0; which < 2; ++which) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            float2 v = which == 0 ? dg[i] : db[i];
#pragma unroll
            for (int o = kStripLanes; o < 32; o *= 2) v = add2(v, make_float2(__shfl_xor_sync(0xffffffffu, v.x, o), __shfl_xor_sync(0xffffffffu, v.y, o)));
            if (lane < kStripLanes) *reinterpret_cast<float2*>(&part[warp][which][lane * kVec + 2 * i]) = v;
        }
    }
    __syncthreads();
    for (uint32_t j = threadIdx.x; j < 2 * kStrip; j += blockDim.x) {
        const uint32_t which = j / kStrip, c = strip * kStrip + j % kStrip;
        if (c >= b.cols) continue;
        float s = 0.0f;
        for (uint32_t k = 0; k < warps; ++k) s += part[k][which][j % kStrip];
        (which == 0 ? grad_gamma : grad_beta)[c] = static_cast<O>(s);
    }
}

template <class T, bool KEPT, bool ALIGNED>
__global__ void __launch_bounds__(kMaxThreads, 1) backwardFewRowsKernel(const __grid_constant__ Backward<T> b, uint32_t row_ctas, int grad_param_dtype, void* grad_gamma, void* grad_beta) {
    __shared__ union {
        Scratch scratch;
        float part[kMaxThreads / 32][2][kStrip];
    } shared;
    gridDependencyWait();
    gridLaunchDependents();
    if (blockIdx.x >= row_ctas) {
        const uint32_t strip = blockIdx.x - row_ctas;
        if (grad_param_dtype == THOR_B200_FP32) columnStrip<T, KEPT, ALIGNED>(b, strip, shared.part, static_cast<float*>(grad_gamma), static_cast<float*>(grad_beta));
        else if (grad_param_dtype == THOR_B200_FP16) columnStrip<T, KEPT, ALIGNED>(b, strip, shared.part, static_cast<__half*>(grad_gamma), static_cast<__half*>(grad_beta));
        else columnStrip<T, KEPT, ALIGNED>(b, strip, shared.part, static_cast<__nv_bfloat16*>(grad_gamma), static_cast<__nv_bfloat16*>(grad_beta));
        return;
    }
    const uint32_t team = b.team, team_id = threadIdx.x / team, t = threadIdx.x - team_id * team, teams = blockDim.x / team;
    const uint32_t lane = threadIdx.x % 32, col = t * kVec;
    const bool before = team < 32 ? t > 0 : lane > 0, after = team < 32 ? t + 1 < team : lane < 31;
    const uint32_t step = row_ctas * teams;
    int slot = 0;
    for (uint32_t base = blockIdx.x * teams; base < b.rows; base += step) {
        const uint32_t row = base + team_id, cols = row < b.rows ? b.cols : 0;
        Raw<T, ALIGNED> grad, stream;
        Normal<KEPT, ALIGNED, T> normal;
        const T* const grad_at = b.grad.p + rowStart(row, b.grad.stride) + col;
        fetch16(b.grad, grad_at, col, cols, grad);
        normal.fetch(b, row, col, cols);
        if (b.grad_sum.p != nullptr) fetch16(b.grad_sum, b.grad_sum.p + rowStart(row, b.grad_sum.stride) + col, col, cols, stream);
        const float rstd = cols > 0 ? b.rstd[row] : 0.0f, mean = cols > 0 && !KEPT ? b.mean[row] : 0.0f;
        float2 w[8], n[8], s1 = both(0.0f), s2 = both(0.0f);
        expand16(grad_at, col, cols, grad, w);
        normal.expand(b, row, col, cols, mean, rstd, n);
        weigh16(b, col, cols, w, n, s1, s2);
        const float2 s = teamSum(make_float2(s1.x + s1.y, s2.x + s2.y), team, team_id, shared.scratch, slot);
        slot ^= 1;
        finish16<ALIGNED>(b, row, col, cols, w, n, s.x * b.inverse, s.y * b.inverse, rstd, stream, before, after);
    }
}

// ---- rows longer than 8192 columns ----------------------------------------------------------------------------
// One CTA a row, two passes over it (the second mostly from L2).
template <class T, bool KEPT, bool ALIGNED>
__global__ void __launch_bounds__(512) gradInputLoopKernel(const __grid_constant__ Backward<T> b) {
    __shared__ float scratch[2][32];
    gridDependencyWait();
    gridLaunchDependents();
    const uint32_t row = blockIdx.x;
    const uint32_t lane = threadIdx.x % 32, step = blockDim.x * kVec;
    const float rstd = b.rstd[row];
    const float mean = KEPT ? 0.0f : b.mean[row];
    float2 w[8], n[8];
    Normal<KEPT, ALIGNED, T> normal;
    float s1 = 0.0f, s2 = 0.0f;
    for (uint64_t at = threadIdx.x * kVec; at < b.cols; at += step) {
        const uint32_t col = static_cast<uint32_t>(at);
        normal.fetch(b, row, col, b.cols);
        load16<ALIGNED>(b.grad, b.grad.p + rowStart(row, b.grad.stride) + col, col, b.cols, w);
        normal.expand(b, row, col, b.cols, mean, rstd, n);
        float2 p1 = both(0.0f), p2 = both(0.0f);
        weigh16(b, col, b.cols, w, n, p1, p2);
        s1 += p1.x + p1.y;
        s2 += p2.x + p2.y;
    }
    const float c1 = ctaSum(s1, scratch[0]) * b.inverse;
    const float c2 = ctaSum(s2, scratch[1]) * b.inverse;
    // the trip count is the same for the whole CTA; a thread past the row's end has columns of none
    for (uint64_t base = 0; base < b.cols; base += step) {
        const uint64_t at = base + threadIdx.x * kVec;
        const uint32_t col = static_cast<uint32_t>(at), cols = at < b.cols ? b.cols : 0;
        Raw<T, ALIGNED> stream;
        if (b.grad_sum.p != nullptr) fetch16(b.grad_sum, b.grad_sum.p + rowStart(row, b.grad_sum.stride) + col, col, cols, stream);
        normal.fetch(b, row, col, cols);
        load16<ALIGNED>(b.grad, b.grad.p + rowStart(row, b.grad.stride) + col, col, cols, w);
        normal.expand(b, row, col, cols, mean, rstd, n);
        float2 p1 = both(0.0f), p2 = both(0.0f);
        weigh16(b, col, cols, w, n, p1, p2);
        finish16<ALIGNED>(b, row, col, cols, w, n, c1, c2, rstd, stream, lane > 0, lane < 31);
    }
}

// Column sums of one slab of rows: a warp takes every eighth row of 512 columns, the CTA's eight warps are added in order.
template <class T, bool KEPT, bool ALIGNED>
__global__ void __launch_bounds__(256) columnSumKernel(const __grid_constant__ Backward<T> b) {
    __shared__ float part[8][512];
    gridDependencyWait();
    gridLaunchDependents();
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const uint32_t first = blockIdx.x * 512, col = first + lane * kVec;
    const uint32_t end = min(b.rows, (blockIdx.y + 1) * b.slab_rows);
    float2 dg[8], db[8], d[8], n[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) dg[i] = db[i] = both(0.0f);
    for (uint32_t row = blockIdx.y * b.slab_rows + warp; row < end; row += 8) {
        Normal<KEPT, ALIGNED, T> normal;
        normal.fetch(b, row, col, b.cols);
        load16<ALIGNED>(b.grad, b.grad.p + rowStart(row, b.grad.stride) + col, col, b.cols, d);
        normal.expand(b, row, col, b.cols, KEPT ? 0.0f : b.mean[row], KEPT ? 0.0f : b.rstd[row], n);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            dg[i] = fma2(d[i], n[i], dg[i]);
            db[i] = add2(db[i], d[i]);
        }
    }
    for (int which = 0; which < 2; ++which) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float2 v = which == 0 ? dg[i] : db[i];
            part[warp][lane * kVec + 2 * i] = v.x;
            part[warp][lane * kVec + 2 * i + 1] = v.y;
        }
        __syncthreads();
        for (uint32_t j = threadIdx.x; j < 512 && first + j < b.padded; j += 256) {
            float s = 0.0f;
#pragma unroll
            for (int k = 0; k < 8; ++k) s += part[k][j];
            b.partial[(static_cast<uint64_t>(blockIdx.y) * 2 + which) * b.padded + first + j] = s;
        }
    }
}

// Adds the partial rows in order and rounds: 32 places a CTA, its eight warps take every eighth partial row.  Place j holds column
// 16 (j mod team) + j / team, or j itself (team = 0).
template <class O>
__global__ void __launch_bounds__(256) foldKernel(const float* __restrict__ partial, uint32_t padded, uint32_t cols, uint32_t team, uint32_t partial_rows,
                                                  O* __restrict__ grad_gamma, O* __restrict__ grad_beta) {
    constexpr int kBatch = 19;
    __shared__ float part[8][33];
    gridDependencyWait();
    gridLaunchDependents();
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const uint32_t j = blockIdx.x * 32 + lane;
    const uint32_t col = team == 0 ? j : kVec * (j % team) + j / team;
    float s = 0.0f;
    if (j < padded) {
        const float* p = partial + static_cast<uint64_t>(blockIdx.y) * padded + j;
        for (uint32_t first = warp; first < partial_rows; first += 8 * kBatch) {
            float v[kBatch];  // all loads of a batch before the first addition: 148 partial rows are one batch
#pragma unroll
            for (int k = 0; k < kBatch; ++k) v[k] = first + 8 * k < partial_rows ? p[static_cast<uint64_t>(first + 8 * k) * 2 * padded] : 0.0f;
#pragma unroll
            for (int k = 0; k < kBatch; ++k) s += v[k];
        }
    }
    part[warp][lane] = s;
    __syncthreads();
    if (warp != 0 || j >= padded || col >= cols) return;
    s = 0.0f;
#pragma unroll
    for (int k = 0; k < 8; ++k) s += part[k][lane];
    (blockIdx.y == 0 ? grad_gamma : grad_beta)[col] = static_cast<O>(s);
}

// ---- host side --------------------------------------------------------------------------------------------
// Up to here one launch is faster than two: [128, 4096] bf16 4.8 us against 10.6, [512, 4096] 7.8 against 13.0, [512, 8192] 10.9 against 12.0,
// [1024, 8192] 20.4 against 15.1.
constexpr uint64_t kFewRows = 512;

struct Plan {
    bool fused, few;
    uint32_t team, teams, partial_rows, padded;
    uint64_t slab_rows;
};
Plan planOf(uint64_t rows, uint64_t cols) {
    Plan p{};
    p.fused = cols <= kFusedCols;
    p.few = p.fused && rows <= kFewRows;
    if (p.fused) {
        p.team = teamOf((cols + kVec - 1) / kVec, 1);
        p.teams = kMaxThreads / p.team;
        p.padded = p.team * kVec;
        p.partial_rows = static_cast<uint32_t>(std::max<uint64_t>(1, std::min<uint64_t>(kPartialRows, (rows + p.teams - 1) / p.teams)));
    } else {  // slabs of at least 32 rows, six CTAs an SM
        p.padded = static_cast<uint32_t>((cols + 7) / 8 * 8);
        const uint64_t strips = (cols + 511) / 512, wanted = std::max<uint64_t>(1, 148 * 6 / strips);
        p.partial_rows = static_cast<uint32_t>(std::max<uint64_t>(1, std::min<uint64_t>(wanted, (rows + 31) / 32)));
        p.slab_rows = (rows + p.partial_rows - 1) / p.partial_rows;
    }
    return p;
}

template <class O>
int launchFold(const float* partial, const Plan& p, uint32_t cols, void* grad_gamma, void* grad_beta, cudaStream_t stream) {
    TB_CUDA(launchDependent(foldKernel<O>, dim3((p.padded + 31) / 32, 2), dim3(256), 0, stream, partial, p.padded, cols, p.team, p.partial_rows, static_cast<O*>(grad_gamma),
                            static_cast<O*>(grad_beta)));
    countLaunch();
    return THOR_B200_OK;
}

template <class T>
int launchBackward(const Backward<T>& b, const Plan& p, bool aligned, int grad_param_dtype, void* grad_gamma, void* grad_beta, cudaStream_t stream) {
    const int st = byFlag(aligned, [&](auto a) {
        return byFlag(b.kept.codes != nullptr, [&](auto k) {
            constexpr bool A = decltype(a)::value, K = decltype(k)::value;
            if (p.few && b.partial != nullptr) {
                TB_CUDA(launchDependent(backwardFewRowsKernel<T, K, A>, dim3(p.partial_rows + (b.cols + kStrip - 1) / kStrip), dim3(p.team * p.teams), 0, stream,
                                        b, p.partial_rows, grad_param_dtype, grad_gamma, grad_beta));
                countLaunch();
                return static_cast<int>(THOR_B200_OK);
            }
            if (p.fused) {
                const uint32_t threads = p.team * p.teams;
                if constexpr (sizeof(T) == 2 && A && K) {
                    if (threads <= kPairThreads) {
                        TB_CUDA(launchDependent(backwardKernel<T, 2, K, A>, dim3(p.partial_rows), dim3(threads), 0, stream, b));
                        countLaunch();
                        return static_cast<int>(THOR_B200_OK);
                    }
                }
                TB_CUDA(launchDependent(backwardKernel<T, 1, K, A>, dim3(p.partial_rows), dim3(threads), 0, stream, b));
                countLaunch();
                return static_cast<int>(THOR_B200_OK);
            }
            TB_CUDA(launchDependent(gradInputLoopKernel<T, K, A>, dim3(static_cast<unsigned>(b.rows)), dim3(512), 0, stream, b));
            countLaunch();
            if (b.partial == nullptr) return static_cast<int>(THOR_B200_OK);
            TB_CUDA(launchDependent(columnSumKernel<T, K, A>, dim3((b.cols + 511) / 512, p.partial_rows), dim3(256), 0, stream, b));
            countLaunch();
            return static_cast<int>(THOR_B200_OK);
        });
    });
    if (st || b.partial == nullptr || p.few) return st;
    switch (grad_param_dtype) {
        case THOR_B200_FP32: return launchFold<float>(b.partial, p, b.cols, grad_gamma, grad_beta, stream);
        case THOR_B200_FP16: return launchFold<__half>(b.partial, p, b.cols, grad_gamma, grad_beta, stream);
        default: return launchFold<__nv_bfloat16>(b.partial, p, b.cols, grad_gamma, grad_beta, stream);
    }
}

}  // namespace
}  // namespace tb

extern "C" {

int thor_b200_layernorm_backward_workspace_bytes(const thor_b200_layernorm_desc* d, size_t* bytes) {
    using namespace tb;
    TB_REQUIRE(bytes != nullptr, "layernorm_backward_workspace_bytes: null argument");
    if (int st = ln::checkDesc("layernorm_backward_workspace_bytes", d)) return st;
    const Plan p = planOf(d->rows, d->cols);
    *bytes = p.few ? 16 : std::max<size_t>(16, static_cast<size_t>(p.partial_rows) * 2 * p.padded * sizeof(float));
    return THOR_B200_OK;
}

int thor_b200_layernorm_backward_launch_count(const thor_b200_layernorm_desc* d, int parameter_gradients) {
    if (d == nullptr || d->rows == 0) return 0;
    const tb::Plan p = tb::planOf(d->rows, d->cols);
    return !parameter_gradients || p.few ? 1 : (p.fused ? 2 : 3);
}

int thor_b200_layernorm_backward_launch(const thor_b200_layernorm_desc* d, const void* grad_output, const void* x, const float* mean, const float* rstd,
                                        const void* codes, const void* scales, const void* gamma, const void* grad_sum, void* grad_input, void* grad_gamma,
                                        void* grad_beta, void* workspace, size_t workspace_bytes, void* stream_v) {
    using namespace tb;
    using namespace tb::ln;
    const char* who = "layernorm_backward";
    if (int st = checkDesc(who, d)) return st;
    if (int st = checkStride(who, "grad_output", d->y_stride, *d)) return st;
    if (x != nullptr)
        if (int st = checkStride(who, "x", d->x_stride, *d)) return st;
    if (grad_sum != nullptr)
        if (int st = checkStride(who, "grad_sum", d->residual_stride, *d)) return st;
    const bool params = grad_gamma != nullptr || grad_beta != nullptr;
    TB_REQUIRE((grad_gamma != nullptr) == (grad_beta != nullptr), "%s: grad_gamma and grad_beta go together", who);
    TB_REQUIRE(!params || valueDtypeOk(d->grad_param_dtype), "%s: parameter gradients must be fp32, fp16 or bf16, got %s", who, dtypeName(d->grad_param_dtype));
    cudaStream_t stream = static_cast<cudaStream_t>(stream_v);
    if (d->rows == 0) {
        if (params) {
            TB_CUDA(cudaMemsetAsync(grad_gamma, 0, d->cols * dtypeSize(d->grad_param_dtype), stream));
            TB_CUDA(cudaMemsetAsync(grad_beta, 0, d->cols * dtypeSize(d->grad_param_dtype), stream));
        }
        return THOR_B200_OK;
    }
    TB_REQUIRE(grad_output != nullptr && grad_input != nullptr && rstd != nullptr, "%s: null tensor pointer", who);
    for (const void* q : {grad_output, x, grad_sum, static_cast<const void*>(grad_input)})
        if (int st = checkPointer(who, q, dtypeSize(d->dtype))) return st;
    if (int st = checkPointer(who, gamma, dtypeSize(d->param_dtype))) return st;
    for (const void* q : {static_cast<const void*>(mean), static_cast<const void*>(rstd)})
        if (int st = checkPointer(who, q, sizeof(float))) return st;
    for (const void* q : {static_cast<const void*>(grad_gamma), static_cast<const void*>(grad_beta)})
        if (int st = checkPointer(who, q, dtypeSize(d->grad_param_dtype))) return st;
    if (int st = checkKept(who, codes, scales, *d)) return st;
    TB_REQUIRE((codes != nullptr) != (x != nullptr) && (x != nullptr) == (mean != nullptr), "%s: needs either the saved input with its mean or the checkpoint", who);
    const Plan p = planOf(d->rows, d->cols);
    size_t needed = 0;
    if (int st = thor_b200_layernorm_backward_workspace_bytes(d, &needed)) return st;
    TB_REQUIRE(!params || (workspace != nullptr && workspace_bytes >= needed && isAligned(workspace, 16)), "%s: needs a 16-byte aligned workspace of %zu bytes", who, needed);
    const bool aligned = d->cols % kVec == 0 && rowsAligned(grad_output, d->y_stride, d->dtype, d->rows) && rowsAligned(x, d->x_stride, d->dtype, d->rows) &&
                         rowsAligned(grad_sum, d->residual_stride, d->dtype, d->rows) && rowsAligned(grad_input, d->cols, d->dtype, d->rows);
    return byDtype(d->dtype, [&](auto t) {
        using T = decltype(t);
        Backward<T> b{};
        b.grad = rowsOf<T>(grad_output, d->y_stride, d->rows, d->cols);
        b.x = rowsOf<T>(x, d->x_stride, d->rows, d->cols);
        b.grad_sum = rowsOf<T>(grad_sum, d->residual_stride, d->rows, d->cols);
        b.grad_input = static_cast<T*>(grad_input);
        b.mean = mean;
        b.rstd = rstd;
        b.gamma = paramOf(gamma, d->param_dtype);
        b.kept = Reader{static_cast<const uint8_t*>(codes), static_cast<const uint8_t*>(scales), static_cast<uint32_t>(codePitch(d->cols)), static_cast<uint32_t>(scalePitch(d->cols)), d->code_dtype};
        b.rows = static_cast<uint32_t>(d->rows);
        b.cols = static_cast<uint32_t>(d->cols);
        b.team = p.team;
        b.inverse = 1.0f / static_cast<float>(d->cols);
        b.partial = params ? static_cast<float*>(workspace) : nullptr;
        b.padded = p.padded;
        b.slab_rows = static_cast<uint32_t>(p.slab_rows);
        return launchBackward<T>(b, p, aligned, d->grad_param_dtype, grad_gamma, grad_beta, stream);
    });
}

}  // extern "C"
