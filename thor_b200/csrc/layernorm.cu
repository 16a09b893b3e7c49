// LayerNorm forward and backward over the last axis, beside the 8-bit checkpoint of the normalised rows.
//
// Forward: a row is read once and stays in registers; the mean, then the mean of the squared differences from it (two passes
// over registers, no cancellation), then the output and the checkpoint.  Short rows (up to 1024 columns) belong to a group of 4 to
// 32 lanes, longer ones to a CTA; a row that no CTA can hold is read three times by a CTA that loops.
// Backward: two row sums, then the input's gradient; the column sums of the parameters' gradients are taken over slabs of rows
// into partial rows in the workspace, which a last kernel adds in order.
#include <algorithm>

#include "checkpoint8.cuh"

namespace tb {
namespace {

using namespace ck8;

constexpr uint32_t kGroupCols = 32 * 4 * kVec;    // longest row of a group of lanes: four chunks a lane
constexpr uint32_t kCtaCols = 1024 * 4 * kVec;    // longest row of a CTA's registers

// Sum over the `lanes` lanes of a row's group (a power of two), or over the CTA: every thread gets it.  `slot` is one of the CTA's
// scratch rows of 32 floats; consecutive calls use different ones, so one barrier per call is enough.
template <bool CTA>
__device__ __forceinline__ float rowSum(float v, int lanes, float* slot) {
    if constexpr (!CTA) {
        for (int o = lanes / 2; o > 0; o /= 2) v += __shfl_xor_sync(0xffffffffu, v, o);
        return v;
    } else {
#pragma unroll
        for (int o = 16; o > 0; o /= 2) v += __shfl_xor_sync(0xffffffffu, v, o);
        if (threadIdx.x % 32 == 0) slot[threadIdx.x / 32] = v;
        __syncthreads();
        v = threadIdx.x % 32 < blockDim.x / 32 ? slot[threadIdx.x % 32] : 0.0f;
#pragma unroll
        for (int o = 16; o > 0; o /= 2) v += __shfl_xor_sync(0xffffffffu, v, o);
        return v;
    }
}

// Eight neighbouring values of a parameter, `absent` where there is none.
struct Param {
    const void* p;
    int dtype;
    bool aligned;  // 16-byte aligned
};
template <class T>
__device__ __forceinline__ void loadParamAs(const Param& q, uint32_t col, uint32_t cols, float (&v)[8]) {
    const T* p = static_cast<const T*>(q.p) + col;
    if (q.aligned && col + kVec <= cols) {
        Pack<8 * sizeof(T)> pack;
#pragma unroll
        for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i) reinterpret_cast<uint4*>(&pack)[i] = __ldg(reinterpret_cast<const uint4*>(p) + i);
        widen8(pack, v, T{});
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = col + i < cols ? toFloat(p[i]) : 0.0f;
    }
}
__device__ __forceinline__ void loadParam8(const Param& q, float absent, uint32_t col, uint32_t cols, float (&v)[8]) {
    if (q.p == nullptr) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = absent;
    } else if (q.dtype == THOR_B200_FP32) {
        loadParamAs<float>(q, col, cols, v);
    } else if (q.dtype == THOR_B200_FP16) {
        loadParamAs<__half>(q, col, cols, v);
    } else {
        loadParamAs<__nv_bfloat16>(q, col, cols, v);
    }
}

template <class T>
struct Forward {
    const T* x;
    const T* residual;
    T* y;
    T* sum;
    float* mean;
    float* rstd;
    int64_t x_stride, residual_stride, y_stride;
    Param gamma, beta;
    Writer kept;  // kept.codes == nullptr: no checkpoint
    uint64_t rows;
    uint32_t cols;
    int lanes;  // of a row's group
    float eps, count;  // count = cols
};

// Eight columns of the row that is normalised: x, or the rounded sum, which is stored.
template <bool ALIGNED, class T>
__device__ __forceinline__ void loadInput8(const Forward<T>& f, uint64_t row, uint32_t col, uint32_t cols, float (&v)[8], bool store) {
    loadRow8<ALIGNED>(f.x + row * f.x_stride, col, cols, v);
    if (f.residual != nullptr) {
        float r[8];
        loadRow8<ALIGNED>(f.residual + row * f.residual_stride, col, cols, r);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] += r[i];
        roundTo8<T>(v);
        if (store && f.sum != nullptr) storeRow8<ALIGNED>(f.sum + row * f.cols, col, cols, v);
    }
}
template <bool ALIGNED, class T>
__device__ __forceinline__ void finish8(const Forward<T>& f, uint64_t row, uint32_t col, float (&v)[8], float mean, float rstd, bool active) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = col + i < f.cols ? (v[i] - mean) * rstd : 0.0f;
    if (f.kept.codes != nullptr) writeRow8(f.kept, row, col, f.cols, v, active);
    if (!active || col >= f.cols) return;
    float g[8], b[8];
    loadParam8(f.gamma, 1.0f, col, f.cols, g);
    loadParam8(f.beta, 0.0f, col, f.cols, b);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = fmaf(v[i], g[i], b[i]);
    storeRow8<ALIGNED>(f.y + row * f.y_stride, col, f.cols, v);
}

// A thread holds chunks t, t + team, t + 2 team ... of its row, `team` the lanes of its group or the threads of the CTA.
template <class T, int CHUNKS, bool CTA, bool ALIGNED>
__global__ void __launch_bounds__(CTA ? 1024 : 256) forwardKernel(const Forward<T> f) {
    __shared__ float scratch[2][32];
    gridDependencyWait();
    gridLaunchDependents();
    const uint32_t team = CTA ? blockDim.x : f.lanes;
    const uint64_t row = CTA ? blockIdx.x : (static_cast<uint64_t>(blockIdx.x) * blockDim.x + threadIdx.x) / team;
    const uint32_t t = CTA ? threadIdx.x : threadIdx.x % team;
    const bool active = row < f.rows;
    const uint32_t cols = active ? f.cols : 0;
    float v[CHUNKS][8];
    float s = 0.0f;
#pragma unroll
    for (int k = 0; k < CHUNKS; ++k) {
        loadInput8<ALIGNED>(f, row, (t + k * team) * kVec, cols, v[k], true);
#pragma unroll
        for (int i = 0; i < 8; ++i) s += v[k][i];
    }
    const float mean = rowSum<CTA>(s, f.lanes, scratch[0]) / f.count;
    s = 0.0f;
#pragma unroll
    for (int k = 0; k < CHUNKS; ++k)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float d = (t + k * team) * kVec + i < cols ? v[k][i] - mean : 0.0f;
            s = fmaf(d, d, s);
        }
    const float rstd = 1.0f / sqrtf(rowSum<CTA>(s, f.lanes, scratch[1]) / f.count + f.eps);
    if (active && t == 0) {
        if (f.mean != nullptr) f.mean[row] = mean;
        if (f.rstd != nullptr) f.rstd[row] = rstd;
    }
#pragma unroll
    for (int k = 0; k < CHUNKS; ++k) finish8<ALIGNED>(f, row, (t + k * team) * kVec, v[k], mean, rstd, active);
}

// Rows of any length: one CTA of 1024 threads a row, three passes over it (the second and third mostly from L2).
template <class T, bool ALIGNED>
__global__ void __launch_bounds__(1024) forwardLoopKernel(const Forward<T> f) {
    __shared__ float scratch[2][32];
    gridDependencyWait();
    gridLaunchDependents();
    const uint64_t row = blockIdx.x;
    const uint32_t step = blockDim.x * kVec;
    float v[8];
    float s = 0.0f;
    for (uint64_t col = threadIdx.x * kVec; col < f.cols; col += step) {
        loadInput8<ALIGNED>(f, row, static_cast<uint32_t>(col), f.cols, v, true);
        s += ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
    }
    const float mean = rowSum<true>(s, 32, scratch[0]) / f.count;
    s = 0.0f;
    for (uint64_t col = threadIdx.x * kVec; col < f.cols; col += step) {
        loadInput8<ALIGNED>(f, row, static_cast<uint32_t>(col), f.cols, v, false);
        float part = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float d = col + i < f.cols ? v[i] - mean : 0.0f;
            part = fmaf(d, d, part);
        }
        s += part;
    }
    const float rstd = 1.0f / sqrtf(rowSum<true>(s, 32, scratch[1]) / f.count + f.eps);
    if (threadIdx.x == 0) {
        if (f.mean != nullptr) f.mean[row] = mean;
        if (f.rstd != nullptr) f.rstd[row] = rstd;
    }
    // the loop's trip count is the same for the whole CTA: the blocks of the checkpoint need all lanes
    for (uint64_t base = 0; base < f.cols; base += step) {
        const uint64_t col = base + threadIdx.x * kVec;
        const bool active = col < (static_cast<uint64_t>(f.cols) + 15) / 16 * 16;
        const uint32_t c = active ? static_cast<uint32_t>(col) : 0u;
        loadInput8<ALIGNED>(f, row, c, active ? f.cols : 0u, v, false);
        if (!active) {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = mean;  // contributes nothing
        }
        finish8<ALIGNED>(f, row, active ? c : 0u, v, mean, rstd, active);
    }
}

// ---- backward ---------------------------------------------------------------------------------------------
template <class T>
struct Backward {
    const T* grad;      // of the output
    const T* x;         // the saved input, or nullptr
    const T* grad_sum;  // or nullptr
    T* grad_input;
    const float* mean;
    const float* rstd;
    int64_t grad_stride, x_stride, sum_stride;
    Param gamma;
    Reader kept;
    uint64_t rows;
    uint32_t cols;
    int lanes;
    float count;  // cols
    float* partial;       // [slabs][2][padded cols]
    uint32_t padded;      // cols rounded up to 8
    uint64_t slab_rows;   // rows of a slab
};

// Normalised values of eight columns; zero past the row's end.
template <bool KEPT, bool ALIGNED, class T>
__device__ __forceinline__ void loadNormal8(const Backward<T>& b, uint64_t row, uint32_t col, uint32_t cols, float mean, float rstd, float (&v)[8]) {
    if constexpr (KEPT) {
        readRow8(b.kept, row, col, cols, v);
        if constexpr (!ALIGNED) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (col + i >= cols) v[i] = 0.0f;  // a NaN block's padding
        }
    } else {
        loadRow8<ALIGNED>(b.x + row * b.x_stride, col, cols, v);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = col + i < cols ? (v[i] - mean) * rstd : 0.0f;
    }
}
// grad_input of eight columns from w = grad * gamma, the normalised values and the two row means.
template <bool ALIGNED, class T>
__device__ __forceinline__ void storeGrad8(const Backward<T>& b, uint64_t row, uint32_t col, float (&w)[8], const float (&n)[8], float c1, float c2, float rstd) {
    if (col >= b.cols) return;
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = __fmul_rn(rstd, fmaf(-n[i], c2, w[i] - c1));
    if (b.grad_sum != nullptr) {
        float r[8];
        loadRow8<ALIGNED>(b.grad_sum + row * b.sum_stride, col, b.cols, r);
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] += r[i];
    }
    storeRow8<ALIGNED>(b.grad_input + row * b.cols, col, b.cols, w);
}

template <class T, int CHUNKS, bool KEPT, bool CTA, bool ALIGNED>
__global__ void __launch_bounds__(CTA ? 1024 : 256) gradInputKernel(const Backward<T> b) {
    __shared__ float scratch[2][32];
    gridDependencyWait();
    gridLaunchDependents();
    const uint32_t team = CTA ? blockDim.x : b.lanes;
    const uint64_t row = CTA ? blockIdx.x : (static_cast<uint64_t>(blockIdx.x) * blockDim.x + threadIdx.x) / team;
    const uint32_t t = CTA ? threadIdx.x : threadIdx.x % team;
    const bool active = row < b.rows;
    const uint32_t cols = active ? b.cols : 0;
    const float rstd = active ? b.rstd[row] : 0.0f;
    const float mean = active && !KEPT ? b.mean[row] : 0.0f;
    float w[CHUNKS][8], n[CHUNKS][8];
    float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
    for (int k = 0; k < CHUNKS; ++k) {
        const uint32_t col = (t + k * team) * kVec;
        float g[8];
        loadRow8<ALIGNED>(b.grad + row * b.grad_stride, col, cols, w[k]);
        loadNormal8<KEPT, ALIGNED>(b, row, col, cols, mean, rstd, n[k]);
        loadParam8(b.gamma, 1.0f, col, cols, g);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            w[k][i] = __fmul_rn(w[k][i], g[i]);  // rounded the same way in every variant of the kernel
            s1 += w[k][i];
            s2 = fmaf(w[k][i], n[k][i], s2);
        }
    }
    const float c1 = rowSum<CTA>(s1, b.lanes, scratch[0]) / b.count;
    const float c2 = rowSum<CTA>(s2, b.lanes, scratch[1]) / b.count;
    if (!active) return;
#pragma unroll
    for (int k = 0; k < CHUNKS; ++k) storeGrad8<ALIGNED>(b, row, (t + k * team) * kVec, w[k], n[k], c1, c2, rstd);
}

template <class T, bool KEPT, bool ALIGNED>
__global__ void __launch_bounds__(1024) gradInputLoopKernel(const Backward<T> b) {
    __shared__ float scratch[2][32];
    gridDependencyWait();
    gridLaunchDependents();
    const uint64_t row = blockIdx.x;
    const uint32_t step = blockDim.x * kVec;
    const float rstd = b.rstd[row];
    const float mean = KEPT ? 0.0f : b.mean[row];
    float w[8], n[8], g[8];
    float s1 = 0.0f, s2 = 0.0f;
    for (uint64_t col = threadIdx.x * kVec; col < b.cols; col += step) {
        loadRow8<ALIGNED>(b.grad + row * b.grad_stride, static_cast<uint32_t>(col), b.cols, w);
        loadNormal8<KEPT, ALIGNED>(b, row, static_cast<uint32_t>(col), b.cols, mean, rstd, n);
        loadParam8(b.gamma, 1.0f, static_cast<uint32_t>(col), b.cols, g);
        float p1 = 0.0f, p2 = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            w[i] = __fmul_rn(w[i], g[i]);
            p1 += w[i];
            p2 = fmaf(w[i], n[i], p2);
        }
        s1 += p1;
        s2 += p2;
    }
    const float c1 = rowSum<true>(s1, 32, scratch[0]) / b.count;
    const float c2 = rowSum<true>(s2, 32, scratch[1]) / b.count;
    for (uint64_t col = threadIdx.x * kVec; col < b.cols; col += step) {
        loadRow8<ALIGNED>(b.grad + row * b.grad_stride, static_cast<uint32_t>(col), b.cols, w);
        loadNormal8<KEPT, ALIGNED>(b, row, static_cast<uint32_t>(col), b.cols, mean, rstd, n);
        loadParam8(b.gamma, 1.0f, static_cast<uint32_t>(col), b.cols, g);
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = __fmul_rn(w[i], g[i]);
        storeGrad8<ALIGNED>(b, row, static_cast<uint32_t>(col), w, n, c1, c2, rstd);
    }
}

// Column sums of one slab of rows: a warp takes every eighth row of 256 columns, the CTA's eight warps are added in order.
template <class T, bool KEPT, bool ALIGNED>
__global__ void __launch_bounds__(256) columnSumKernel(const Backward<T> b) {
    __shared__ float part[8][2][256];
    gridDependencyWait();
    gridLaunchDependents();
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const uint32_t first = blockIdx.x * 256, col = first + lane * kVec;
    const uint64_t end = min(b.rows, (blockIdx.y + 1) * b.slab_rows);
    float dg[8] = {}, db[8] = {};
    for (uint64_t row = blockIdx.y * b.slab_rows + warp; row < end; row += 8) {
        float d[8], n[8];
        loadRow8<ALIGNED>(b.grad + row * b.grad_stride, col, b.cols, d);
        loadNormal8<KEPT, ALIGNED>(b, row, col, b.cols, KEPT ? 0.0f : b.mean[row], KEPT ? 0.0f : b.rstd[row], n);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            dg[i] = fmaf(d[i], n[i], dg[i]);
            db[i] += d[i];
        }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        part[warp][0][lane * kVec + i] = dg[i];
        part[warp][1][lane * kVec + i] = db[i];
    }
    __syncthreads();
    if (first + threadIdx.x >= b.padded) return;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        float s = 0.0f;
#pragma unroll
        for (int k = 0; k < 8; ++k) s += part[k][which][threadIdx.x];
        b.partial[(static_cast<uint64_t>(blockIdx.y) * 2 + which) * b.padded + first + threadIdx.x] = s;
    }
}

// Adds the slabs' partial rows in order and rounds: 32 columns a CTA, its eight warps take every eighth slab.
template <class O>
__global__ void __launch_bounds__(256) foldKernel(const float* __restrict__ partial, uint32_t padded, uint32_t cols, uint32_t slabs, O* __restrict__ grad_gamma,
                                                  O* __restrict__ grad_beta) {
    __shared__ float part[8][33];
    gridDependencyWait();
    gridLaunchDependents();
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const uint32_t col = blockIdx.x * 32 + lane;
    float s = 0.0f;
    if (col < cols) {
        const float* p = partial + static_cast<uint64_t>(blockIdx.y) * padded + col;
#pragma unroll 4
        for (uint32_t k = warp; k < slabs; k += 8) s += p[static_cast<uint64_t>(k) * 2 * padded];
    }
    part[warp][lane] = s;
    __syncthreads();
    if (warp != 0 || col >= cols) return;
    s = 0.0f;
#pragma unroll
    for (int k = 0; k < 8; ++k) s += part[k][lane];
    (blockIdx.y == 0 ? grad_gamma : grad_beta)[col] = static_cast<O>(s);
}

// ---- host side --------------------------------------------------------------------------------------------
bool rowsAligned(const void* p, int64_t stride, int dtype, uint64_t rows) {
    return p == nullptr || (isAligned(p, 16) && (rows <= 1 || (static_cast<uint64_t>(stride) * dtypeSize(dtype)) % 16 == 0));
}
Param paramOf(const void* p, int dtype) { return Param{p, dtype, isAligned(p, 16)}; }

int checkDesc(const char* who, const thor_b200_layernorm_desc* d) {
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
int checkStride(const char* who, const char* what, int64_t stride, const thor_b200_layernorm_desc& d) {
    TB_REQUIRE(d.rows <= 1 || (stride >= 0 && static_cast<uint64_t>(stride) >= d.cols), "%s: the row stride of %s is smaller than a row", who, what);
    return THOR_B200_OK;
}

// Threads of a row: a group of lanes, a CTA, or a CTA that loops.
struct Shape {
    bool group = false, cta = false;
    int chunks = 1;  // of a thread
    unsigned lanes = 32, threads = 256, grid = 1;
};
Shape shapeOf(uint64_t rows, uint64_t cols) {
    Shape s;
    const uint64_t chunks = (cols + kVec - 1) / kVec;
    if (cols <= kGroupCols) {
        s.group = true;
        s.lanes = 4;
        while (s.lanes < 32 && s.lanes < chunks) s.lanes *= 2;
        const uint64_t per = (chunks + s.lanes - 1) / s.lanes;
        s.chunks = per <= 1 ? 1 : (per <= 2 ? 2 : 4);
        s.threads = 256;
        const uint64_t rows_per_cta = s.threads / s.lanes;
        s.grid = static_cast<unsigned>((rows + rows_per_cta - 1) / rows_per_cta);
    } else if (cols <= kCtaCols) {
        s.cta = true;
        s.chunks = chunks <= 1024 ? 2 : 4;
        s.threads = static_cast<unsigned>((chunks + s.chunks - 1) / s.chunks + 31) / 32 * 32;
        s.grid = static_cast<unsigned>(rows);
    } else {
        s.threads = 1024;
        s.grid = static_cast<unsigned>(rows);
    }
    return s;
}

uint32_t paddedCols(uint64_t cols) { return static_cast<uint32_t>((cols + kVec - 1) / kVec * kVec); }
// Slabs of rows for the column sums: enough CTAs for the device, at least 32 rows each.
uint32_t slabsOf(uint64_t rows, uint64_t cols) {
    const uint64_t strips = (cols + 255) / 256;
    const uint64_t wanted = std::max<uint64_t>(1, 148 * 6 / strips);
    return static_cast<uint32_t>(std::max<uint64_t>(1, std::min<uint64_t>(wanted, (rows + 31) / 32)));
}

template <class F>
int byFlag(bool flag, F&& f) {
    return flag ? f(std::true_type{}) : f(std::false_type{});
}
template <class F>
int byChunks(int chunks, F&& f) {
    switch (chunks) {
        case 1: return f(std::integral_constant<int, 1>{});
        case 2: return f(std::integral_constant<int, 2>{});
        default: return f(std::integral_constant<int, 4>{});
    }
}

template <class T>
int launchForward(const Forward<T>& f, bool aligned, cudaStream_t stream) {
    const Shape s = shapeOf(f.rows, f.cols);
    return byFlag(aligned, [&](auto a) {
        constexpr bool A = decltype(a)::value;
        if (!s.group && !s.cta) {
            TB_CUDA(launchDependent(forwardLoopKernel<T, A>, dim3(s.grid), dim3(s.threads), 0, stream, f));
            countLaunch();
            return static_cast<int>(THOR_B200_OK);
        }
        Forward<T> g = f;
        g.lanes = static_cast<int>(s.lanes);
        return byFlag(s.cta, [&](auto cta) {
            return byChunks(s.chunks, [&](auto chunks) {
                TB_CUDA(launchDependent(forwardKernel<T, decltype(chunks)::value, decltype(cta)::value, A>, dim3(s.grid), dim3(s.threads), 0, stream, g));
                countLaunch();
                return static_cast<int>(THOR_B200_OK);
            });
        });
    });
}

template <class T>
int launchBackward(const Backward<T>& b, bool aligned, bool params, int grad_param_dtype, void* grad_gamma, void* grad_beta, cudaStream_t stream) {
    const bool kept = b.kept.codes != nullptr;
    const Shape s = shapeOf(b.rows, b.cols);
    const int st = byFlag(aligned, [&](auto a) {
        constexpr bool A = decltype(a)::value;
        return byFlag(kept, [&](auto k) {
            constexpr bool K = decltype(k)::value;
            if (!s.group && !s.cta) {
                TB_CUDA(launchDependent(gradInputLoopKernel<T, K, A>, dim3(s.grid), dim3(s.threads), 0, stream, b));
            } else {
                Backward<T> g = b;
                g.lanes = static_cast<int>(s.lanes);
                const int st = byFlag(s.cta, [&](auto cta) {
                    return byChunks(s.chunks, [&](auto chunks) {
                        TB_CUDA(launchDependent(gradInputKernel<T, decltype(chunks)::value, K, decltype(cta)::value, A>, dim3(s.grid), dim3(s.threads), 0, stream, g));
                        return static_cast<int>(THOR_B200_OK);
                    });
                });
                if (st) return st;
            }
            countLaunch();
            if (!params) return static_cast<int>(THOR_B200_OK);
            const uint32_t slabs = slabsOf(b.rows, b.cols);
            TB_CUDA(launchDependent(columnSumKernel<T, K, A>, dim3((b.cols + 255) / 256, slabs), dim3(256), 0, stream, b));
            countLaunch();
            return static_cast<int>(THOR_B200_OK);
        });
    });
    if (st || !params) return st;
    const uint32_t slabs = slabsOf(b.rows, b.cols);
    const dim3 grid((b.cols + 31) / 32, 2);
    switch (grad_param_dtype) {
        case THOR_B200_FP32:
            TB_CUDA(launchDependent(foldKernel<float>, grid, dim3(256), 0, stream, b.partial, b.padded, b.cols, slabs, static_cast<float*>(grad_gamma), static_cast<float*>(grad_beta)));
            break;
        case THOR_B200_FP16:
            TB_CUDA(launchDependent(foldKernel<__half>, grid, dim3(256), 0, stream, b.partial, b.padded, b.cols, slabs, static_cast<__half*>(grad_gamma), static_cast<__half*>(grad_beta)));
            break;
        default:
            TB_CUDA(launchDependent(foldKernel<__nv_bfloat16>, grid, dim3(256), 0, stream, b.partial, b.padded, b.cols, slabs, static_cast<__nv_bfloat16*>(grad_gamma),
                                    static_cast<__nv_bfloat16*>(grad_beta)));
    }
    countLaunch();
    return THOR_B200_OK;
}

template <class F>
int byDtype(int dtype, F&& f) {
    switch (dtype) {
        case THOR_B200_FP32: return f(float{});
        case THOR_B200_FP16: return f(__half{});
        default: return f(__nv_bfloat16{});
    }
}

}  // namespace
}  // namespace tb

extern "C" {

int thor_b200_layernorm_launch(const thor_b200_layernorm_desc* d, const void* x, const void* residual, const void* gamma, const void* beta, void* y, void* sum,
                               float* mean, float* rstd, void* codes, void* scales, void* stream) {
    using namespace tb;
    const char* who = "layernorm";
    if (int st = checkDesc(who, d)) return st;
    if (int st = checkStride(who, "x", d->x_stride, *d)) return st;
    if (int st = checkStride(who, "y", d->y_stride, *d)) return st;
    if (residual != nullptr)
        if (int st = checkStride(who, "residual", d->residual_stride, *d)) return st;
    TB_REQUIRE(residual != nullptr || sum == nullptr, "%s: sum without residual", who);
    if (d->rows == 0) return THOR_B200_OK;
    TB_REQUIRE(x != nullptr && y != nullptr, "%s: null tensor pointer", who);
    const bool kept = codes != nullptr || scales != nullptr;
    TB_REQUIRE(kept == (d->code_dtype != 0) && (codes != nullptr) == (scales != nullptr), "%s: codes and scales go with a code_dtype", who);
    TB_REQUIRE(!kept || isAligned(codes, 16), "%s: codes must be 16-byte aligned", who);
    const bool aligned = d->cols % ck8::kVec == 0 && rowsAligned(x, d->x_stride, d->dtype, d->rows) && rowsAligned(residual, d->residual_stride, d->dtype, d->rows) &&
                         rowsAligned(y, d->y_stride, d->dtype, d->rows) && rowsAligned(sum, d->cols, d->dtype, d->rows);
    return byDtype(d->dtype, [&](auto t) {
        using T = decltype(t);
        Forward<T> f{};
        f.x = static_cast<const T*>(x);
        f.residual = static_cast<const T*>(residual);
        f.y = static_cast<T*>(y);
        f.sum = static_cast<T*>(sum);
        f.mean = mean;
        f.rstd = rstd;
        f.x_stride = d->x_stride;
        f.residual_stride = d->residual_stride;
        f.y_stride = d->y_stride;
        f.gamma = paramOf(gamma, d->param_dtype);
        f.beta = paramOf(beta, d->param_dtype);
        f.kept = Writer{static_cast<uint8_t*>(codes), static_cast<uint8_t*>(scales), ck8::codePitch(d->cols), ck8::scalePitch(d->cols), d->code_dtype};
        f.rows = d->rows;
        f.cols = static_cast<uint32_t>(d->cols);
        f.eps = d->eps;
        f.count = static_cast<float>(d->cols);
        return launchForward<T>(f, aligned, static_cast<cudaStream_t>(stream));
    });
}

int thor_b200_layernorm_backward_workspace_bytes(const thor_b200_layernorm_desc* d, size_t* bytes) {
    using namespace tb;
    TB_REQUIRE(bytes != nullptr, "layernorm_backward_workspace_bytes: null argument");
    if (int st = checkDesc("layernorm_backward_workspace_bytes", d)) return st;
    *bytes = std::max<size_t>(16, static_cast<size_t>(slabsOf(d->rows, d->cols)) * 2 * paddedCols(d->cols) * sizeof(float));
    return THOR_B200_OK;
}

int thor_b200_layernorm_backward_launch_count(const thor_b200_layernorm_desc* d, int parameter_gradients) {
    if (d == nullptr || d->rows == 0) return 0;
    return parameter_gradients ? 3 : 1;
}

int thor_b200_layernorm_backward_launch(const thor_b200_layernorm_desc* d, const void* grad_output, const void* x, const float* mean, const float* rstd,
                                        const void* codes, const void* scales, const void* gamma, const void* grad_sum, void* grad_input, void* grad_gamma,
                                        void* grad_beta, void* workspace, size_t workspace_bytes, void* stream_v) {
    using namespace tb;
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
    const bool kept = codes != nullptr || scales != nullptr;
    TB_REQUIRE(kept == (d->code_dtype != 0) && (codes != nullptr) == (scales != nullptr), "%s: codes and scales go with a code_dtype", who);
    TB_REQUIRE(kept != (x != nullptr) && (x != nullptr) == (mean != nullptr), "%s: needs either the saved input with its mean or the checkpoint", who);
    TB_REQUIRE(!kept || isAligned(codes, 16), "%s: codes must be 16-byte aligned", who);
    size_t needed = 0;
    if (int st = thor_b200_layernorm_backward_workspace_bytes(d, &needed)) return st;
    TB_REQUIRE(!params || (workspace != nullptr && workspace_bytes >= needed && isAligned(workspace, 16)), "%s: needs a 16-byte aligned workspace of %zu bytes", who, needed);
    const bool aligned = d->cols % ck8::kVec == 0 && rowsAligned(grad_output, d->y_stride, d->dtype, d->rows) && rowsAligned(x, d->x_stride, d->dtype, d->rows) &&
                         rowsAligned(grad_sum, d->residual_stride, d->dtype, d->rows) && rowsAligned(grad_input, d->cols, d->dtype, d->rows);
    return byDtype(d->dtype, [&](auto t) {
        using T = decltype(t);
        Backward<T> b{};
        b.grad = static_cast<const T*>(grad_output);
        b.x = static_cast<const T*>(x);
        b.grad_sum = static_cast<const T*>(grad_sum);
        b.grad_input = static_cast<T*>(grad_input);
        b.mean = mean;
        b.rstd = rstd;
        b.grad_stride = d->y_stride;
        b.x_stride = d->x_stride;
        b.sum_stride = d->residual_stride;
        b.gamma = paramOf(gamma, d->param_dtype);
        b.kept = Reader{static_cast<const uint8_t*>(codes), static_cast<const uint8_t*>(scales), ck8::codePitch(d->cols), ck8::scalePitch(d->cols), d->code_dtype};
        b.rows = d->rows;
        b.cols = static_cast<uint32_t>(d->cols);
        b.count = static_cast<float>(d->cols);
        b.partial = static_cast<float*>(workspace);
        b.padded = paddedCols(d->cols);
        const uint32_t slabs = slabsOf(d->rows, d->cols);
        b.slab_rows = (d->rows + slabs - 1) / slabs;
        return launchBackward<T>(b, aligned, params, d->grad_param_dtype, grad_gamma, grad_beta, stream);
    });
}

}  // extern "C"
