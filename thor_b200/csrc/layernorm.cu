// LayerNorm forward: residual add, statistics, output and the 8-bit checkpoint of the normalised rows in one pass.
//
// A row stays in registers from its load to its last store.  Every warp takes the mean of its own columns and the squared differences from
// that; the warps' results are put together as M2 = sum of M2_w + n_w (mean_w - mean)^2, so that nothing cancels and a row costs one barrier
// instead of two.  Teams walk their rows and load the next one before they work on the current one.  A row that a CTA's
// registers cannot hold is read three times by a CTA that loops.
#include <algorithm>

#include "layernorm_common.cuh"

namespace tb {
namespace {

using namespace ln;

constexpr uint64_t kRegisterCols = 512ull * 2 * kVec;  // longest row of a team's registers: 512 threads, two chunks each

// CTAs of 512 threads an SM holds: one chunk a thread needs 64 registers, two need 128.  Up to 8192 columns one chunk is the faster form (more warps
// to wait with): [32768, 8192] bf16 with checkpoint, in runs of a few milliseconds, 230 us against 255 with two and 80 registers and 334 with two and 128 (at
// sustained clocks the first takes 250).
constexpr int residentCtas(int chunks) { return chunks == 1 ? 2 : 1; }

template <class T>
struct Forward {
    Rows<T> x, residual;
    T* y;
    T* sum;
    float* mean;
    float* rstd;
    uint32_t y_stride;
    Param gamma, beta;
    bool packable;  // the parameters that are given have the tensors' type
    Writer kept;  // kept.codes == nullptr: no checkpoint
    uint32_t rows, cols, team;
    float eps, count, inverse;  // count = cols, inverse = 1 / cols
};

// v - mean, zero past the row's end
template <bool ALIGNED>
__device__ __forceinline__ void centre16(const float2 (&v)[8], float mean, uint32_t col, uint32_t cols, float2 (&d)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) d[i] = col < cols ? add2(v[i], both(-mean)) : both(0.0f);
    if constexpr (!ALIGNED) cutRow(col, cols, d);
}
__device__ __forceinline__ float squares16(const float2 (&d)[8]) {
    float2 s = mul2(d[0], d[0]), u = mul2(d[1], d[1]);
#pragma unroll
    for (int i = 2; i < 8; i += 2) {
        s = fma2(d[i], d[i], s);
        u = fma2(d[i + 1], d[i + 1], u);
    }
    s = add2(s, u);
    return s.x + s.y;
}

// GROUP: teams of up to 32 lanes; otherwise of whole warps.
template <class T, int CHUNKS, bool GROUP, bool PACKED, bool ALIGNED, bool RESIDUAL>
__global__ void __launch_bounds__(kMaxThreads, residentCtas(CHUNKS)) forwardKernel(const __grid_constant__ Forward<T> f) {
    constexpr bool kAhead = ALIGNED && !RESIDUAL;  // the next row is loaded while this one is worked on
    __shared__ Scratch scratch;
    using Params = Staged<T, PACKED>;
    extern __shared__ uint4 planes[];  // gamma's, then beta's
    gridDependencyWait();
    gridLaunchDependents();
    const uint32_t team = f.team, team_id = threadIdx.x / team, t = threadIdx.x - team_id * team, teams = blockDim.x / team;
    const uint32_t lane = threadIdx.x % 32, chunks = CHUNKS * team;
    const bool before = GROUP ? t > 0 : lane > 0, after = GROUP ? t + 1 < team : lane < 31;
    const uint32_t step = gridDim.x * teams;
    // columns of this warp, and of the warp whose results this lane fetches
    const uint32_t warps = GROUP ? 1 : team / 32, my_warp = GROUP ? 0 : threadIdx.x / 32 - team_id * warps;
    const float own_count = GROUP ? f.count : warpColumns(my_warp, team, f.cols, CHUNKS);
    const float its_count = GROUP || lane % 16 >= warps ? 0.0f : warpColumns(lane % 16, team, f.cols, CHUNKS);
    const float own_inverse = own_count > 0.0f ? 1.0f / own_count : 0.0f, its_inverse = its_count > 0.0f ? 1.0f / its_count : 0.0f;
    const uint32_t span = GROUP ? team : 32;  // lanes that share a row
    int slot = 0;
    uint32_t row = blockIdx.x * teams + team_id;
    uint32_t cols = row < f.rows ? f.cols : 0;
    Raw<T, ALIGNED> next[CHUNKS], next_residual[RESIDUAL ? CHUNKS : 1];
    auto at = [&](const Rows<T>& in, uint32_t r, int k) { return in.p + rowStart(r, in.stride) + (t + k * team) * kVec; };
    auto fetch = [&](uint32_t r, uint32_t n) {
#pragma unroll
        for (int k = 0; k < CHUNKS; ++k) {
            fetch16(f.x, at(f.x, r, k), (t + k * team) * kVec, n, next[k]);
            if constexpr (RESIDUAL) fetch16(f.residual, at(f.residual, r, k), (t + k * team) * kVec, n, next_residual[k]);
        }
    };
    fetch(row, cols);
    const uint4* const beta_planes = planes + Params::kPlanes * chunks;
    Params::stage(f.gamma, 1.0f, planes, chunks, f.cols);
    Params::stage(f.beta, 0.0f, planes + Params::kPlanes * chunks, chunks, f.cols);
    __syncthreads();
    // the same number of turns for the whole CTA; a team without a row has cols = 0
    for (uint32_t base = blockIdx.x * teams; base < f.rows; base += step, row += step) {
        float2 v[CHUNKS][8];
        float s = 0.0f;
#pragma unroll
        for (int k = 0; k < CHUNKS; ++k) {
            const uint32_t col = (t + k * team) * kVec;
            expand16(at(f.x, row, k), col, cols, next[k], v[k]);
            if constexpr (RESIDUAL) {
                float2 r[8];
                expand16(at(f.residual, row, k), col, cols, next_residual[k], r);
#pragma unroll
                for (int i = 0; i < 8; ++i) v[k][i] = add2(v[k][i], r[i]);
                roundTo16<T>(v[k]);
            }
            s += sum16(v[k]);
        }
        const uint32_t next_cols = row + step < f.rows ? f.cols : 0;
        if constexpr (kAhead) fetch(row + step, next_cols);
        if constexpr (RESIDUAL) {
            if (f.sum != nullptr) {
                T* const sum_at = f.sum + rowStart(row, f.cols) + t * kVec;
#pragma unroll
                for (int k = 0; k < CHUNKS; ++k) store16<ALIGNED>(sum_at + k * team * kVec, (t + k * team) * kVec, cols, v[k], before, after);
            }
        }
        s = laneSum(s, span);
        float mean = divideBy(s, own_count, own_inverse), m2 = 0.0f;  // of the warp's columns
#pragma unroll
        for (int k = 0; k < CHUNKS; ++k) {
            float2 d[8];
            centre16<ALIGNED>(v[k], mean, (t + k * team) * kVec, cols, d);
            m2 += squares16(d);
        }
        m2 = laneSum(m2, span);
        if constexpr (!GROUP) {
            if (lane == 0) scratch.part[slot][team_id][my_warp] = make_float2(s, m2);
            asm volatile("bar.sync %0, %1;" ::"r"(team_id + 1), "r"(team) : "memory");
            const float2 its = lane % 16 < warps ? scratch.part[slot][team_id][lane % 16] : make_float2(0.0f, 0.0f);
            slot ^= 1;
            const float row_mean = divideBy(laneSum(its.x, 16), f.count, f.inverse);
            const float off = its_count > 0.0f ? divideBy(its.x, its_count, its_inverse) - row_mean : 0.0f;
            m2 = laneSum(fmaf(its_count * off, off, its.y), 16);
            mean = row_mean;
        }
        const float rstd = inverseRoot(divideBy(m2, f.count, f.inverse) + f.eps);
        if (t == 0 && cols > 0) {
            if (f.mean != nullptr) f.mean[row] = mean;
            if (f.rstd != nullptr) f.rstd[row] = rstd;
        }
#pragma unroll
        for (int k = 0; k < CHUNKS; ++k) {
            const uint32_t col = (t + k * team) * kVec;
            centre16<ALIGNED>(v[k], mean, col, cols, v[k]);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[k][i] = mul2(v[k][i], both(rstd));
            if (f.kept.codes != nullptr) writeCodes(codesAt(f.kept, row, col), scaleAt(f.kept, row, col), f.kept.code, col, cols, v[k]);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float2 g[4], b[4];
                Params::read(planes, chunks, t + k * team, h, g);
                Params::read(beta_planes, chunks, t + k * team, h, b);
#pragma unroll
                for (int i = 0; i < 4; ++i) v[k][4 * h + i] = fma2(v[k][4 * h + i], g[i], b[i]);
            }
            store16<ALIGNED>(f.y + rowStart(row, f.y_stride) + col, col, cols, v[k], before, after);
        }
        cols = next_cols;
        if constexpr (!kAhead) fetch(row + step, cols);
    }
}

// The row that is normalised: x, or the rounded sum.
template <bool ALIGNED, class T>
__device__ __forceinline__ void input16(const Forward<T>& f, uint32_t row, uint32_t col, uint32_t cols, float2 (&v)[8]) {
    load16<ALIGNED>(f.x, f.x.p + rowStart(row, f.x.stride) + col, col, cols, v);
    if (f.residual.p != nullptr) {
        float2 r[8];
        load16<ALIGNED>(f.residual, f.residual.p + rowStart(row, f.residual.stride) + col, col, cols, r);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = add2(v[i], r[i]);
        roundTo16<T>(v);
    }
}
// Rows of any length: one CTA a row, three passes over it (the second and third mostly from L2).
template <class T, bool ALIGNED>
__global__ void __launch_bounds__(512) forwardLoopKernel(const __grid_constant__ Forward<T> f) {
    __shared__ float scratch[2][32];
    gridDependencyWait();
    gridLaunchDependents();
    const uint32_t row = blockIdx.x;
    const uint32_t lane = threadIdx.x % 32, step = blockDim.x * kVec;
    // the loops' trip counts are the same for the whole CTA; a thread past the row's end has columns of none
    float2 v[8];
    float s = 0.0f;
    for (uint64_t base = 0; base < f.cols; base += step) {
        const uint64_t at = base + threadIdx.x * kVec;
        const uint32_t col = static_cast<uint32_t>(at), cols = at < f.cols ? f.cols : 0;
        input16<ALIGNED>(f, row, col, cols, v);
        s += sum16(v);
        if (f.sum != nullptr) store16<ALIGNED>(f.sum + rowStart(row, f.cols) + col, col, cols, v, lane > 0, lane < 31);
    }
    const float mean = divideBy(ctaSum(s, scratch[0]), f.count, f.inverse);
    s = 0.0f;
    for (uint64_t at = threadIdx.x * kVec; at < f.cols; at += step) {
        input16<ALIGNED>(f, row, static_cast<uint32_t>(at), f.cols, v);
        centre16<ALIGNED>(v, mean, static_cast<uint32_t>(at), f.cols, v);
        s += squares16(v);
    }
    const float rstd = inverseRoot(divideBy(ctaSum(s, scratch[1]), f.count, f.inverse) + f.eps);
    if (threadIdx.x == 0) {
        if (f.mean != nullptr) f.mean[row] = mean;
        if (f.rstd != nullptr) f.rstd[row] = rstd;
    }
    for (uint64_t base = 0; base < f.cols; base += step) {
        const uint64_t at = base + threadIdx.x * kVec;
        const uint32_t col = static_cast<uint32_t>(at), cols = at < f.cols ? f.cols : 0;
        input16<ALIGNED>(f, row, col, cols, v);
        centre16<ALIGNED>(v, mean, col, cols, v);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = mul2(v[i], both(rstd));
        if (f.kept.codes != nullptr) writeCodes(codesAt(f.kept, row, col), scaleAt(f.kept, row, col), f.kept.code, col, cols, v);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float2 p[4], q[4];
            loadParam8(f.gamma, 1.0f, col + 8 * h, cols, p);
            loadParam8(f.beta, 0.0f, col + 8 * h, cols, q);
#pragma unroll
            for (int i = 0; i < 4; ++i) v[4 * h + i] = fma2(v[4 * h + i], p[i], q[i]);
        }
        store16<ALIGNED>(f.y + rowStart(row, f.y_stride) + col, col, cols, v, lane > 0, lane < 31);
    }
}

template <class T>
int launchForward(const Forward<T>& given, bool aligned, cudaStream_t stream) {
    Forward<T> f = given;
    const DeviceInfo* device = nullptr;
    if (int st = currentDeviceInfo(&device)) return st;
    const uint64_t chunks = (f.cols + kVec - 1) / kVec;
    return byFlag(aligned, [&](auto a) {
        constexpr bool A = decltype(a)::value;
        if (f.cols > kRegisterCols) {
            TB_CUDA(launchDependent(forwardLoopKernel<T, A>, dim3(static_cast<unsigned>(f.rows)), dim3(512), 0, stream, f));
            countLaunch();
            return static_cast<int>(THOR_B200_OK);
        }
        const int per_thread = chunks <= kMaxThreads ? 1 : 2;
        f.team = teamOf(chunks, per_thread);
        const uint32_t threads = f.team * (kMaxThreads / f.team);
        const uint64_t teams = threads / f.team, ctas = (f.rows + teams - 1) / teams;
        const uint64_t resident = static_cast<uint64_t>(device->sm_count) * (kMaxThreads * residentCtas(per_thread) / threads);
        const dim3 grid(static_cast<unsigned>(std::min(ctas, resident))), block(threads);
        const bool packed = sizeof(T) == 2 && f.packable;
        const size_t shared = (packed ? 4 : 8) * sizeof(uint4) * per_thread * f.team;
        return byFlag(f.residual.p != nullptr, [&](auto residual) {
            constexpr bool R = decltype(residual)::value;
            auto launch = [&](auto chunks_a_thread, auto group, auto in_own_type) {
                constexpr auto kernel = &forwardKernel<T, decltype(chunks_a_thread)::value, decltype(group)::value, decltype(in_own_type)::value, A, R>;
                if (int st = allowShared<kernel>(shared)) return st;
                TB_CUDA(launchDependent(kernel, grid, block, shared, stream, f));
                countLaunch();
                return static_cast<int>(THOR_B200_OK);
            };
            auto launchFor = [&](auto in_own_type) {
                if (f.team <= 32) return launch(std::integral_constant<int, 1>{}, std::true_type{}, in_own_type);
                if (per_thread == 1) return launch(std::integral_constant<int, 1>{}, std::false_type{}, in_own_type);
                return launch(std::integral_constant<int, 2>{}, std::false_type{}, in_own_type);
            };
            if constexpr (sizeof(T) == 2)
                if (packed) return launchFor(std::true_type{});
            return launchFor(std::false_type{});
        });
    });
}

}  // namespace
}  // namespace tb

extern "C" {

int thor_b200_layernorm_launch(const thor_b200_layernorm_desc* d, const void* x, const void* residual, const void* gamma, const void* beta, void* y, void* sum,
                               float* mean, float* rstd, void* codes, void* scales, void* stream) {
    using namespace tb;
    using namespace tb::ln;
    const char* who = "layernorm";
    if (int st = checkDesc(who, d)) return st;
    if (int st = checkStride(who, "x", d->x_stride, *d)) return st;
    if (int st = checkStride(who, "y", d->y_stride, *d)) return st;
    if (residual != nullptr)
        if (int st = checkStride(who, "residual", d->residual_stride, *d)) return st;
    TB_REQUIRE(residual != nullptr || sum == nullptr, "%s: sum without residual", who);
    if (d->rows == 0) return THOR_B200_OK;
    TB_REQUIRE(x != nullptr && y != nullptr, "%s: null tensor pointer", who);
    for (const void* p : {x, residual, static_cast<const void*>(y), static_cast<const void*>(sum)})
        if (int st = checkPointer(who, p, dtypeSize(d->dtype))) return st;
    for (const void* p : {gamma, beta})
        if (int st = checkPointer(who, p, dtypeSize(d->param_dtype))) return st;
    for (const void* p : {static_cast<const void*>(mean), static_cast<const void*>(rstd)})
        if (int st = checkPointer(who, p, sizeof(float))) return st;
    if (int st = checkKept(who, codes, scales, *d)) return st;
    const bool aligned = d->cols % kVec == 0 && rowsAligned(x, d->x_stride, d->dtype, d->rows) && rowsAligned(residual, d->residual_stride, d->dtype, d->rows) &&
                         rowsAligned(y, d->y_stride, d->dtype, d->rows) && rowsAligned(sum, d->cols, d->dtype, d->rows);
    return byDtype(d->dtype, [&](auto t) {
        using T = decltype(t);
        Forward<T> f{};
        f.x = rowsOf<T>(x, d->x_stride, d->rows, d->cols);
        f.residual = rowsOf<T>(residual, d->residual_stride, d->rows, d->cols);
        f.y = static_cast<T*>(y);
        f.sum = static_cast<T*>(sum);
        f.mean = mean;
        f.rstd = rstd;
        f.y_stride = strideOf(d->y_stride, d->rows);
        f.gamma = paramOf(gamma, d->param_dtype);
        f.beta = paramOf(beta, d->param_dtype);
        f.packable = d->param_dtype == d->dtype;
        f.kept = Writer{static_cast<uint8_t*>(codes), static_cast<uint8_t*>(scales), static_cast<uint32_t>(codePitch(d->cols)), static_cast<uint32_t>(scalePitch(d->cols)), d->code_dtype};
        f.rows = static_cast<uint32_t>(d->rows);
        f.cols = static_cast<uint32_t>(d->cols);
        f.eps = d->eps;
        f.count = static_cast<float>(d->cols);
        f.inverse = 1.0f / f.count;
        return launchForward<T>(f, aligned, static_cast<cudaStream_t>(stream));
    });
}

}  // extern "C"
