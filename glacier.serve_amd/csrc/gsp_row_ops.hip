// Row operators around the projections (gfx950): the root-mean-square norm
// with the residual's addition (gsp_rms_norm) and the row quantiser with its
// gated SiLU (gsp_quantize_fp8).  Both end in e4m3 codes with one scale a row,
// which is what gsp_matmul_batch_fp8 takes.
//
// One workgroup takes one row and holds it in registers: every input is read
// once and every output written once, with the row's two reductions (the sum
// of squares, then the largest magnitude) between.  Rows past what a
// workgroup's registers hold (kRowMax values) are read again for each pass, a
// value at a time.
//
// Bound by memory where there is enough of it: 8193 rows of 4096 with a residual
// and all three results 112 us, 5.1 TB/s (a large copy reaches 4.8); 4096 gated rows
// of 18944 135 us, 5.2 TB/s; 4099 rows of 3584 into codes 11.8 us, 6.2 TB/s (the
// inputs lie in the last-level cache); 64 gated rows of 18944 5.0 us, 2.2 TB/s (64 of
// 256 CUs).  A step's small rows are bound by the launch: 8 rows of 896 take 2.8 us on
// the GPU, 64 of 3584 3.8, and a call 3.4 us on the host.  At 4-byte addresses or of
// odd lengths the first take 132 us and the codes of 4099 rows 17.6.  Long rows
// occupy one workgroup each: 4096 of 40000 with all results 919 us (3.0 TB/s), codes
// alone 317 (2.6); 64 of them 54 and 16.
#include <cfloat>

#include "gsp_internal.h"
#include "../../include/glacier_paged.h"

namespace gsp {
namespace {

constexpr float kE4m3Max = 448.0f;
constexpr float kLeastTop = 0x1p-100f;  // the least largest magnitude a scale is taken from
constexpr float kLeastMean = 0x1p-100f;  // of squares; the rounding of a subnormal one is 2^-150 at most
constexpr int kRowMax = 32768;

struct RowArgs {
    const float* x;         // norm: x; quantiser: a
    const float* other;     // norm: the residual or null; quantiser: b or null
    const float* weight;    // norm
    float* sum;             // norm: x + residual, or null
    float* y;               // norm: fp32 result, or null
    uint8_t* codes;         // or null
    float* scale;
    int64_t stride;         // values between rows of x and other
    float eps;
    int32_t dim;
};

enum { kRowNorm = 0, kRowPlain = 1, kRowSilu = 2 };

// Sum and largest value over the workgroup.  Each wave's result crosses LDS;
// every thread gets the total.  The order of the sum is fixed.
template <typename T>
__device__ inline T wave_sum(T v) {
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) v += __shfl_xor(v, m);
    return v;
}
__device__ inline uint32_t wave_max(uint32_t v) {
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) v = max(v, (uint32_t)__shfl_xor((int)v, m));
    return v;
}
template <typename T>
__device__ inline T block_sum(T v, T* lds) {
    v = wave_sum(v);
    const int waves = blockDim.x >> 6;
    if (waves == 1) return v;
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    T t = 0;
    for (int i = 0; i < waves; ++i) t += lds[i];
    return t;
}
__device__ inline uint32_t block_max(uint32_t v, uint32_t* lds) {
    v = wave_max(v);
    const int waves = blockDim.x >> 6;
    if (waves == 1) return v;
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    uint32_t t = 0;
    for (int i = 0; i < waves; ++i) t = max(t, lds[i]);
    return t;
}

// Magnitudes are compared as the integers of their bits, which order finite
// values, then infinity, then NaN: a row that holds one keeps it as its
// largest.
__device__ inline uint32_t mag(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// The row's scale and the factor of its codes from the largest magnitude.
__device__ inline void row_scale(uint32_t top, float* scale, float* inv) {
    const float t = __uint_as_float(max(top, __float_as_uint(kLeastTop)));
    *scale = t / kE4m3Max;
    *inv = kE4m3Max / t;
}

template <int VEC>
struct Piece {
    float v[VEC];
};

template <int VEC>
__device__ inline Piece<VEC> load_piece(const float* p) {
    Piece<VEC> r;
    if constexpr (VEC == 4) {
        const float4 f = *reinterpret_cast<const float4*>(p);
        r.v[0] = f.x, r.v[1] = f.y, r.v[2] = f.z, r.v[3] = f.w;
    } else {
        r.v[0] = *p;
    }
    return r;
}
template <int VEC>
__device__ inline void store_piece(float* p, const Piece<VEC>& r) {
    if constexpr (VEC == 4)
        *reinterpret_cast<float4*>(p) = make_float4(r.v[0], r.v[1], r.v[2], r.v[3]);
    else
        *p = r.v[0];
}
// Rounds to nearest even; the factor keeps every finite value within 448.
template <int VEC>
__device__ inline void store_codes(uint8_t* p, const Piece<VEC>& r, float inv) {
    if constexpr (VEC == 4) {
        int w = __builtin_amdgcn_cvt_pk_fp8_f32(r.v[0] * inv, r.v[1] * inv, 0, false);
        w = __builtin_amdgcn_cvt_pk_fp8_f32(r.v[2] * inv, r.v[3] * inv, w, true);
        *reinterpret_cast<int*>(p) = w;
    } else {
        *p = (uint8_t)__builtin_amdgcn_cvt_pk_fp8_f32(r.v[0] * inv, 0.f, 0, false);
    }
}

// g / (1 + exp(-g)) * u.  exp(-g) is 2^t with t = -g log2(e) rounded, times 1 + ln 2 times what the rounding left,
// which keeps the hardware's 2^t (one step) that exact for every t; the quotient is a product with the hardware's
// reciprocal (one step).  In all four steps, at 12 instructions; with expf and the division the kernel spends
// more time on them than on memory (64 rows of 18944: 6.7 us against 5.2).  Past +-200 the exponential is 0 or
// infinity in fp32 anyway, and the clamp keeps infinities out of the remainder.
__device__ inline float silu_mul(float g, float u) {
    constexpr float kL = 1.44269502f, kLLow = 1.92596299e-8f, kLn2 = 0.693147182f;  // log2(e) in two parts
    const float x = -__builtin_amdgcn_fmed3f(g, -200.0f, 200.0f);
    const float t = x * kL;
    const float left = fmaf(x, kLLow, fmaf(x, kL, -t));
    const float e = __builtin_amdgcn_exp2f(t) * fmaf(left, kLn2, 1.0f);
    return g * __builtin_amdgcn_rcpf(1.0f + e) * u;
}

// The row's values before the norm's factor: x + residual, a, or silu(a) b.
template <int KIND, int VEC>
__device__ inline Piece<VEC> row_value(const RowArgs& a, const float* x, const float* o, int64_t at) {
    Piece<VEC> r = load_piece<VEC>(x + at);
    if (KIND == kRowSilu || (KIND == kRowNorm && o)) {
        const Piece<VEC> q = load_piece<VEC>(o + at);
#pragma unroll
        for (int i = 0; i < VEC; ++i) r.v[i] = KIND == kRowSilu ? silu_mul(r.v[i], q.v[i]) : r.v[i] + q.v[i];
    }
    return r;
}

// The mean of squares plus eps where squares leave fp32's range, with the row scaled by a power of two, which the norm's
// factor undoes: the larger of the row's top and sqrt(eps) goes to 2^39 to 2^40.  32768 of its squares stay below 2^96,
// and what is lost of small values' squares is far below them.  Rows of zeros, or with an infinity or a NaN, keep theirs.
template <int VEC, int E>
__device__ inline float scaled_mean(const RowArgs& a, Piece<VEC> (&r)[E], float* lsum, uint32_t* lmax) {
    uint32_t top = 0;
    float sq = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) top = max(top, mag(r[e].v[i]));
    }
    top = block_max(top, lmax);
    int shift = 0;
    if (top != 0 && top < 0x7f800000u) {
        (void)frexpf(fmaxf(__uint_as_float(top), sqrtf(a.eps)), &shift);
        shift = 40 - shift;
    }
#pragma unroll
    for (int e = 0; e < E; ++e) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            r[e].v[i] = ldexpf(r[e].v[i], shift);
            sq += r[e].v[i] * r[e].v[i];
        }
    }
    return block_sum(sq, lsum) / (float)a.dim + ldexpf(a.eps, 2 * shift);
}

// One row in registers: E pieces of VEC values a thread.
template <int KIND, int VEC, int E>
__global__ __launch_bounds__(1024) void row_kernel(RowArgs a) {
    __shared__ float lsum[16];
    __shared__ uint32_t lmax[16];
    const int64_t row = blockIdx.x;
    const float* x = a.x + row * a.stride;
    const float* o = a.other ? a.other + row * a.stride : nullptr;
    const int step = blockDim.x * VEC;
    const int at0 = threadIdx.x * VEC;
    Piece<VEC> r[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const int at = at0 + e * step;
        if (at < a.dim) {
            r[e] = row_value<KIND, VEC>(a, x, o, at);
        } else {
#pragma unroll
            for (int i = 0; i < VEC; ++i) r[e].v[i] = 0.f;
        }
    }
    if constexpr (KIND == kRowNorm) {
        float sq = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) {
#pragma unroll
            for (int i = 0; i < VEC; ++i) sq += r[e].v[i] * r[e].v[i];
        }
        if (a.sum) {
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const int at = at0 + e * step;
                if (at < a.dim) store_piece<VEC>(a.sum + row * a.dim + at, r[e]);
            }
        }
        Piece<VEC> w[E];
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (at0 + e * step < a.dim) w[e] = load_piece<VEC>(a.weight + at0 + e * step);
        float mean = block_sum(sq, lsum) / (float)a.dim + a.eps;
        // Squares that fp32 does not hold: once more with the row scaled by a power of two.  Every thread has the same sum.
        if (__builtin_expect(!(mean >= kLeastMean && mean <= FLT_MAX), 0)) mean = scaled_mean<VEC, E>(a, r, lsum, lmax);
        const float f = 1.0f / sqrtf(mean);
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int at = at0 + e * step;
            if (at < a.dim) {
#pragma unroll
                for (int i = 0; i < VEC; ++i) r[e].v[i] = r[e].v[i] * f * w[e].v[i];
                if (a.y) store_piece<VEC>(a.y + row * a.dim + at, r[e]);
            }
        }
        if (!a.codes) return;
    }
    uint32_t top = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) top = max(top, mag(r[e].v[i]));
    }
    float scale, inv;
    row_scale(block_max(top, lmax), &scale, &inv);
    if (threadIdx.x == 0) a.scale[row] = scale;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const int at = at0 + e * step;
        if (at < a.dim) store_codes<VEC>(a.codes + row * a.dim + at, r[e], inv);
    }
}

// Rows of more than kRowMax values: each pass reads the row again.  The norm's
// passes after the first read x + residual, then y, back where the caller keeps
// them, so that they may overwrite x or the residual.  A place may be past
// 2^31 - 1 before the loop ends.  A thread adds dim / 1024 squares one after the
// other: they, their sum and the norm's factor hold 64 bits (in fp32 equal values
// of 1.1 put y of a row of 2^24 off by 920 steps).
template <int KIND>
__global__ __launch_bounds__(1024) void long_row_kernel(RowArgs a) {
    __shared__ double lsum[16];
    __shared__ uint32_t lmax[16];
    const int64_t row = blockIdx.x;
    const float* x = a.x + row * a.stride;
    const float* o = a.other ? a.other + row * a.stride : nullptr;
    double f = 1.0;
    if constexpr (KIND == kRowNorm) {
        double sq = 0;
        for (int64_t at = threadIdx.x; at < a.dim; at += blockDim.x) {
            const float v = row_value<KIND, 1>(a, x, o, at).v[0];
            sq += (double)v * v;
            if (a.sum) a.sum[row * a.dim + at] = v;
        }
        if (a.sum) {
            x = a.sum + row * a.dim;  // each thread reads back what it wrote
            o = nullptr;
        }
        f = 1.0 / sqrt(block_sum(sq, lsum) / a.dim + a.eps);
    }
    uint32_t top = 0;
    for (int64_t at = threadIdx.x; at < a.dim; at += blockDim.x) {
        float v = row_value<KIND, 1>(a, x, o, at).v[0];
        if constexpr (KIND == kRowNorm) {
            v = (float)(v * f) * a.weight[at];
            if (a.y) a.y[row * a.dim + at] = v;
        }
        top = max(top, mag(v));
    }
    if (KIND == kRowNorm && !a.codes) return;
    float scale, inv;
    row_scale(block_max(top, lmax), &scale, &inv);
    if (threadIdx.x == 0) a.scale[row] = scale;
    for (int64_t at = threadIdx.x; at < a.dim; at += blockDim.x) {
        Piece<1> r;
        if (KIND == kRowNorm && a.y) {
            r.v[0] = a.y[row * a.dim + at];
        } else {
            r = row_value<KIND, 1>(a, x, o, at);
            if constexpr (KIND == kRowNorm) r.v[0] = (float)(r.v[0] * f) * a.weight[at];
        }
        store_codes<1>(a.codes + row * a.dim + at, r, inv);
    }
}

template <int KIND, int VEC>
void launch_row(const RowArgs& a, int32_t rows, hipStream_t stream) {
    const int pieces = (a.dim + VEC - 1) / VEC;
    // Threads: a piece or two each while the rows alone cannot fill the chip, else four.
    const int per = rows <= 512 ? 1 : 4;
    int threads = (pieces + per - 1) / per;
    threads = std::min(1024, (threads + 63) / 64 * 64);
    const int e = (pieces + threads - 1) / threads;
    const dim3 grid(rows), block(threads);
    if (e <= 1)
        hipLaunchKernelGGL((row_kernel<KIND, VEC, 1>), grid, block, 0, stream, a);
    else if (e <= 2)
        hipLaunchKernelGGL((row_kernel<KIND, VEC, 2>), grid, block, 0, stream, a);
    else if (e <= 4)
        hipLaunchKernelGGL((row_kernel<KIND, VEC, 4>), grid, block, 0, stream, a);
    else if (KIND != kRowNorm && e <= 5)
        // Rows of 16385 to 20480 values (an FFN's 18944): 64 gated ones 5.2 us, 5.3 in eight pieces.  The norm's two arrays
        // do not gain: 4096 rows with every result 258 us in five pieces, 246 in eight.
        hipLaunchKernelGGL((row_kernel<KIND, VEC, KIND == kRowNorm ? 8 : 5>), grid, block, 0, stream, a);
    else if (e <= 8)
        hipLaunchKernelGGL((row_kernel<KIND, VEC, 8>), grid, block, 0, stream, a);
    else if constexpr (VEC == 1) {
        if (e <= 16)
            hipLaunchKernelGGL((row_kernel<KIND, 1, 16>), grid, block, 0, stream, a);
        else
            hipLaunchKernelGGL((row_kernel<KIND, 1, 32>), grid, block, 0, stream, a);
    }
}

template <int KIND>
hipError_t launch_rows(RowArgs a, int32_t rows, hipStream_t stream) {
    const auto al16 = [](const void* p) { return ((uintptr_t)p & 15) == 0; };
    const bool vec = a.dim % 4 == 0 && a.stride % 4 == 0 && al16(a.x) && al16(a.other) && al16(a.weight) &&
                     al16(a.sum) && al16(a.y) && ((uintptr_t)a.codes & 3) == 0;
    // A launch holds fewer than 2^32 threads.
    constexpr int32_t kMostRows = 1 << 21;
    for (int32_t done = 0; done < rows; done += kMostRows) {
        const int32_t n = std::min(kMostRows, rows - done);
        if (a.dim > kRowMax)
            hipLaunchKernelGGL(long_row_kernel<KIND>, dim3(n), dim3(1024), 0, stream, a);
        else if (vec)
            launch_row<KIND, 4>(a, n, stream);
        else
            launch_row<KIND, 1>(a, n, stream);
        a.x += (int64_t)n * a.stride;
        if (a.other) a.other += (int64_t)n * a.stride;
        if (a.sum) a.sum += (int64_t)n * a.dim;
        if (a.y) a.y += (int64_t)n * a.dim;
        if (a.codes) a.codes += (int64_t)n * a.dim;
        if (a.scale) a.scale += n;
        if (rows - done <= kMostRows) break;
    }
    return hipGetLastError();
}

}  // namespace

hipError_t launch_rms_norm(const RmsNormArgs& n, hipStream_t stream) {
    RowArgs a{};
    a.x = n.x;
    a.other = n.residual;
    a.weight = n.weight;
    a.sum = n.sum;
    a.y = n.y;
    a.codes = n.codes;
    a.scale = n.scale;
    a.stride = n.dim;
    a.eps = n.eps;
    a.dim = n.dim;
    return launch_rows<kRowNorm>(a, n.rows, stream);
}

hipError_t launch_quantize_fp8(const QuantizeArgs& q, hipStream_t stream) {
    RowArgs a{};
    a.x = q.a;
    a.other = q.b;
    a.codes = q.codes;
    a.scale = q.scale;
    a.stride = q.stride;
    a.dim = q.dim;
    return q.b ? launch_rows<kRowSilu>(a, q.rows, stream) : launch_rows<kRowPlain>(a, q.rows, stream);
}

}  // namespace gsp
