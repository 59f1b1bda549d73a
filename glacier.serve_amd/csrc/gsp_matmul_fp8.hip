// Projections of 8-bit activations by 4-bit weights (gsp_matmul_batch_fp8):
// y[b][o] = x_scale[b] * sum_i W[o][i] * e4m3(x[b][i]) with Q4_0, Q4_1 or Q4_K
// rows in their GGUF bytes.
//
// Products run on the fp16 matrix cores.  e4m3 activations are fp16 values,
// converted two at a time; a nibble q at bits 4 to 7 of a 16-bit lane is the fp16
// subnormal q * 2^-20, so a shift and a mask make two weights ready.  Both choices
// are about bits, as probed on the cores: eight neighbouring terms are aligned to
// the largest exponent among them and cut 24 bits below it, a subnormal counting as
// exponent -14 whatever its value.  A product's last bit is 2^-9 * 2^-20 and the
// largest exponent 8 - 14, so every bit is kept (at bits 0 to 3, q * 2^-24, the last
// four are not).  The fp8 instruction cuts 13 bits below the largest term (448 * 8 +
// 0.125 loses the second), which is less than a sum is to hold.  The 32 terms of one
// instruction (16 x 16 x 32) are one group of weights under one scale, whose fp32 sum
// enters the output's fp32 sum with that scale:
//   Q4_0  d (q - 8): the sum starts at -8 * 2^-20 * sum x, a product of x with a
//         constant operand.
//   Q4_1  d q + m and Q4_K  d sc q - dmin m: the sum of x, a product with ones,
//         enters with the group's minimum.
//
// Operand layout.  Lane (n, j) = (lane % 16, lane / 16) of the instruction
// holds 8 of its column's 32 terms.  Which 8 does not matter as long as both
// operands agree, so lanes load long contiguous pieces (64 weights of a row,
// 16 activations) and a 4 x 4 transposition among the four lanes of a column
// (four register swaps, no LDS) deals every lane its dword of each piece.
#include <type_traits>

#include "gsp_internal.h"
#include "../../include/glacier_paged.h"

namespace gsp {
namespace {

typedef float f4 __attribute__((ext_vector_type(4)));
typedef uint32_t u2 __attribute__((ext_vector_type(2)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));
typedef u4 u4_al4 __attribute__((aligned(4)));

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));

constexpr uint32_t kNib = 0x00f000f0u;
constexpr float kCode = 1048576.0f;  // a nibble's fp16 value is q / kCode

__device__ inline void swap32(uint32_t& a, uint32_t& b) {
    const auto r = __builtin_amdgcn_permlane32_swap(a, b, false, false);
    a = r[0], b = r[1];
}
__device__ inline void swap16(uint32_t& a, uint32_t& b) {
    const auto r = __builtin_amdgcn_permlane16_swap(a, b, false, false);
    a = r[0], b = r[1];
}

// Register t of lane (n, j) becomes what register j of lane (n, t) was.
__device__ inline void transpose4(uint32_t& a, uint32_t& b, uint32_t& c, uint32_t& d) {
    swap32(a, c);
    swap32(b, d);
    swap16(a, b);
    swap16(c, d);
}

// r[t] becomes lane (n, t)'s v in all four lanes of the column.
__device__ inline void spread4(uint32_t v, uint32_t* r) {
    uint32_t a = v, b = v;
    swap32(a, b);
    r[0] = a, r[1] = a;
    swap16(r[0], r[1]);
    r[2] = b, r[3] = b;
    swap16(r[2], r[3]);
}

__device__ inline float half_lo(uint32_t w) { return (float)__builtin_bit_cast(_Float16, (uint16_t)w); }
__device__ inline float half_hi(uint32_t w) { return (float)__builtin_bit_cast(_Float16, (uint16_t)(w >> 16)); }

// One lane's 8 terms of a group: activations 4j .. 4j + 3 and 16 + 4j .. + 3 of
// it, and the quants of the same weights.
struct Terms {
    uint32_t r[4];
};

__device__ inline f4 mfma(const Terms& a, const Terms& b, f4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
}

// The e4m3 bytes of a lane's two dwords of a group as fp16.
__device__ inline Terms x_terms(uint32_t lo, uint32_t hi) {
    const auto two = [](uint32_t w, auto high) {
        return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, decltype(high)::value));
    };
    return Terms{{two(lo, std::false_type{}), two(hi, std::false_type{}), two(lo, std::true_type{}),
                  two(hi, std::true_type{})}};
}

// The same fp16 weight beside every activation.
__device__ inline Terms splat_terms(uint32_t half) {
    const uint32_t w = half * 0x10001u;
    return Terms{{w, w, w, w}};
}
constexpr uint32_t kOne = 0x3c00, kMinus8 = 0x8080;  // 1, -8 / kCode

// Bytes 0 2 1 3 of a dword: the two 16-bit lanes of a mask then hold neighbours.
__device__ inline uint32_t deal_bytes(uint32_t w) { return __builtin_amdgcn_perm(w, w, 0x03010200u); }

// A unit is 256 weights of each of 16 rows: lane (n, j) holds the j-th 64 of
// row n as they lie in memory.
template <int WT>
struct Unit;

template <>
struct Unit<GSP_WTYPE_Q4_0> {
    static constexpr int kPairBytes = 36;
    static constexpr bool kMins = false;
    uint32_t w[9];
    __device__ inline void load(const uint8_t* row, int64_t pair) {
        const uint8_t* p = row + pair * kPairBytes;
        const u4 a = *reinterpret_cast<const u4_al4*>(p);
        const u4 b = *reinterpret_cast<const u4_al4*>(p + 16);
        w[8] = *reinterpret_cast<const uint32_t*>(p + 32);
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = a[i], w[4 + i] = b[i];
    }
};

template <>
struct Unit<GSP_WTYPE_Q4_1> {
    static constexpr int kPairBytes = 40;
    static constexpr bool kMins = true;
    uint32_t w[10];
    __device__ inline void load(const uint8_t* row, int64_t pair) {
        const uint8_t* p = row + pair * kPairBytes;
        const u4 a = *reinterpret_cast<const u4_al4*>(p);
        const u4 b = *reinterpret_cast<const u4_al4*>(p + 16);
        w[8] = *reinterpret_cast<const uint32_t*>(p + 32);
        w[9] = *reinterpret_cast<const uint32_t*>(p + 36);
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = a[i], w[4 + i] = b[i];
    }
};

template <>
struct Unit<GSP_WTYPE_Q4_K> {
    static constexpr bool kMins = true;
    uint32_t w[12];  // d | dmin, 12 bytes of scales and mins, the quarter's 32 bytes of quants
    __device__ inline void load(const uint8_t* row, int64_t pair) {
        const uint8_t* p = row + (pair >> 2) * 144;
        const u4 h = *reinterpret_cast<const u4_al4*>(p);
        const u4 a = *reinterpret_cast<const u4_al4*>(p + 16 + 32 * (pair & 3));
        const u4 b = *reinterpret_cast<const u4_al4*>(p + 32 + 32 * (pair & 3));
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = h[i], w[4 + i] = a[i], w[8 + i] = b[i];
    }
};

// A unit dealt out for the matrix instruction: dwords of quants with bytes in
// the order 0 2 1 3, and the scales of every group.  Group 2t + h of the unit's
// eight is q[h][t] (Q4_K: the low or the high halves of q[0][t] and q[1][t]).
template <int WT>
struct Dealt {
    uint32_t q[2][4];
    uint32_t s[2][4];
    float d, dmin;  // Q4_K: of the super-block, d times kCode

    __device__ inline void deal(const Unit<WT>& u) {
        if constexpr (WT == GSP_WTYPE_Q4_0) {
            // d0 and 16 bytes of quants, then d1 and 16: the first block's quants lie two bytes off.
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                q[0][i] = __builtin_amdgcn_perm(u.w[i + 1], u.w[i], 0x05030402u);
                q[1][i] = deal_bytes(u.w[5 + i]);
            }
            spread4((u.w[0] & 0xffffu) | (u.w[4] & 0xffff0000u), s[0]);
        } else if constexpr (WT == GSP_WTYPE_Q4_1) {
#pragma unroll
            for (int i = 0; i < 4; ++i) q[0][i] = deal_bytes(u.w[1 + i]), q[1][i] = deal_bytes(u.w[6 + i]);
            spread4(u.w[0], s[0]);
            spread4(u.w[5], s[1]);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) q[0][i] = deal_bytes(u.w[4 + i]), q[1][i] = deal_bytes(u.w[8 + i]);
            d = half_lo(u.w[0]) * kCode;
            dmin = half_hi(u.w[0]);
            // Groups 2j and 2j + 1: two 6-bit scales and two 6-bit mins into one dword.
            const int j = (threadIdx.x >> 4) & 3;
            const int sh = (j & 1) * 16;
            const uint32_t h1 = u.w[1] >> sh, h2 = u.w[2] >> sh, h3 = u.w[3] >> sh;
            const uint32_t sc = j < 2 ? h1 & 0x3f3fu : (h3 & 0x0f0fu) | (h1 & 0xc0c0u) >> 2;
            const uint32_t mn = j < 2 ? h2 & 0x3f3fu : (h3 >> 4 & 0x0f0fu) | (h2 & 0xc0c0u) >> 2;
            spread4(sc | mn << 16, s[0]);
        }
        transpose4(q[0][0], q[0][1], q[0][2], q[0][3]);
        transpose4(q[1][0], q[1][1], q[1][2], q[1][3]);
    }
    __device__ inline Terms terms(int t, int h) const {
        if constexpr (WT == GSP_WTYPE_Q4_K) {
            // 4j .. 4j + 3 from q[0], 16 + 4j .. from q[1].
            const uint32_t a = q[0][t], b = q[1][t];
            if (h) return Terms{{a & kNib, b & kNib, (a >> 8) & kNib, (b >> 8) & kNib}};
            return Terms{{(a << 4) & kNib, (b << 4) & kNib, (a >> 4) & kNib, (b >> 4) & kNib}};
        }
        const uint32_t a = q[h][t];
        return Terms{{(a << 4) & kNib, a & kNib, (a >> 4) & kNib, (a >> 8) & kNib}};
    }
    // The group's scale, times kCode, and what the sum of x enters with.
    __device__ inline float scale(int t, int h) const {
        if constexpr (WT == GSP_WTYPE_Q4_0) return (h ? half_hi(s[0][t]) : half_lo(s[0][t])) * kCode;
        if constexpr (WT == GSP_WTYPE_Q4_1) return half_lo(s[h][t]) * kCode;
        return d * (float)((s[0][t] >> (8 * h)) & 0xffu);
    }
    __device__ inline float least(int t, int h) const {
        if constexpr (WT == GSP_WTYPE_Q4_1) return half_hi(s[h][t]);
        if constexpr (WT == GSP_WTYPE_Q4_K) return -dmin * (float)((s[0][t] >> (16 + 8 * h)) & 0xffu);
        return 0.f;
    }
};

// One workgroup: 16 * NT weight rows by 16 * MT batch rows.  Its waves share
// the units of K, each with sums of its own, which are added in the order of
// the waves at the end.
template <int WT, int MT, int NT>
__global__ __launch_bounds__(1024) void matmul_fp8_kernel(MatmulFp8Args a) {
    extern __shared__ float part[];  // [waves][NT][MT][256]
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
    const int n = lane & 15, j = lane >> 4;
    const int tiles_b = (a.batch + 16 * MT - 1) / (16 * MT);
    const int row0 = blockIdx.x / tiles_b * (16 * NT), b0 = blockIdx.x % tiles_b * (16 * MT);
    const int pairs = a.in_dim >> 6, units = (pairs + 3) >> 2;
    const uint8_t* wrow[NT];
#pragma unroll
    for (int i = 0; i < NT; ++i)
        wrow[i] = static_cast<const uint8_t*>(a.w) + (int64_t)min(row0 + 16 * i + n, a.out_dim - 1) * a.row_bytes;
    const uint8_t* xrow[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) xrow[m] = a.x + (int64_t)min(b0 + 16 * m + n, a.batch - 1) * a.in_dim + 16 * j;

    f4 acc[NT][MT];
#pragma unroll
    for (int i = 0; i < NT; ++i) {
#pragma unroll
        for (int m = 0; m < MT; ++m) acc[i][m] = f4{0.f, 0.f, 0.f, 0.f};
    }
    Unit<WT> next[NT];
    if (wave < units) {
#pragma unroll
        for (int i = 0; i < NT; ++i) next[i].load(wrow[i], min(4 * wave + j, pairs - 1));
    }
    for (int u = wave; u < units; u += waves) {
        Dealt<WT> w[NT];
#pragma unroll
        for (int i = 0; i < NT; ++i) w[i].deal(next[i]);
        if (u + waves < units) {
#pragma unroll
            for (int i = 0; i < NT; ++i) next[i].load(wrow[i], min(4 * (u + waves) + j, pairs - 1));
        }
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            if (4 * u + t < pairs) {
                uint32_t x[MT][4];
#pragma unroll
                for (int m = 0; m < MT; ++m) {
                    const u4 v = *reinterpret_cast<const u4*>(xrow[m] + (int64_t)(4 * u + t) * 64);
#pragma unroll
                    for (int i = 0; i < 4; ++i) x[m][i] = v[i];
                    transpose4(x[m][0], x[m][1], x[m][2], x[m][3]);
                }
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    Terms xt[MT];
                    f4 sx[MT];
#pragma unroll
                    for (int m = 0; m < MT; ++m) {
                        xt[m] = x_terms(x[m][2 * h], x[m][2 * h + 1]);
                        sx[m] = mfma(xt[m], splat_terms(Unit<WT>::kMins ? kOne : kMinus8), f4{0.f, 0.f, 0.f, 0.f});
                    }
#pragma unroll
                    for (int i = 0; i < NT; ++i) {
                        const Terms q = w[i].terms(t, h);
                        const float sc = w[i].scale(t, h), mn = w[i].least(t, h);
#pragma unroll
                        for (int m = 0; m < MT; ++m) {
                            const f4 s = mfma(xt[m], q, Unit<WT>::kMins ? f4{0.f, 0.f, 0.f, 0.f} : sx[m]);
#pragma unroll
                            for (int r = 0; r < 4; ++r) {
                                acc[i][m][r] = fmaf(sc, s[r], acc[i][m][r]);
                                if constexpr (Unit<WT>::kMins) acc[i][m][r] = fmaf(mn, sx[m][r], acc[i][m][r]);
                            }
                        }
                    }
                }
            }
        }
    }
    // Lane (n, j) holds batch rows 4j .. 4j + 3 of weight row n.
#pragma unroll
    for (int i = 0; i < NT; ++i) {
#pragma unroll
        for (int m = 0; m < MT; ++m) {
#pragma unroll
            for (int r = 0; r < 4; ++r)
                part[((wave * NT + i) * MT + m) * 256 + (4 * j + r) * 16 + n] = acc[i][m][r];
        }
    }
    __syncthreads();
    for (int e = threadIdx.x; e < NT * MT * 256; e += blockDim.x) {
        float s = 0.f;
        for (int v = 0; v < waves; ++v) s += part[v * (NT * MT * 256) + e];
        const int i = e / (MT * 256), m = e / 256 % MT;
        const int b = b0 + 16 * m + (e >> 4) % 16, o = row0 + 16 * i + (e & 15);
        if (b < a.batch && o < a.out_dim) a.y[(int64_t)b * a.out_dim + o] = s * a.x_scale[b];
    }
}

template <int WT, int MT, int NT>
hipError_t launch_form(MatmulFp8Args a, hipStream_t stream) {
    const int units = (a.in_dim + 255) / 256;
    const int most = std::min(16, 65536 / (NT * MT * 1024));
    const int per = (units + most - 1) / most;
    const int waves = (units + per - 1) / per;
    // A launch holds fewer than 2^32 threads: very large batches take several.
    const int64_t tiles = ((int64_t)a.out_dim + 16 * NT - 1) / (16 * NT);
    const int64_t most_rows = std::max<int64_t>(1, (1 << 21) / tiles) * (16 * MT);
    for (int64_t left = a.batch; left > 0; left -= most_rows) {
        a.batch = (int32_t)std::min(left, most_rows);
        const uint32_t grid = (uint32_t)(tiles * ((a.batch + 16 * MT - 1) / (16 * MT)));
        hipLaunchKernelGGL((matmul_fp8_kernel<WT, MT, NT>), dim3(grid), dim3(64 * waves), waves * NT * MT * 1024, stream,
                           a);
        a.x += (int64_t)a.batch * a.in_dim;
        a.x_scale += a.batch;
        a.y += (int64_t)a.batch * a.out_dim;
    }
    return hipGetLastError();
}

template <int WT>
hipError_t launch_type(const MatmulFp8Args& a, hipStream_t stream) {
    if (a.batch <= 16) return launch_form<WT, 1, 1>(a, stream);
    if (a.batch <= 32) return launch_form<WT, 2, 1>(a, stream);
    return launch_form<WT, 4, 1>(a, stream);
}

}  // namespace

int64_t matmul_fp8_row_bytes(int32_t w_type, int32_t in_dim) {
    return (int64_t)(in_dim / 64) * (w_type == GSP_WTYPE_Q4_1 ? 40 : 36);
}

hipError_t launch_matmul_fp8(int32_t w_type, const MatmulFp8Args& a, hipStream_t stream) {
    if (w_type == GSP_WTYPE_Q4_0) return launch_type<GSP_WTYPE_Q4_0>(a, stream);
    if (w_type == GSP_WTYPE_Q4_1) return launch_type<GSP_WTYPE_Q4_1>(a, stream);
    return launch_type<GSP_WTYPE_Q4_K>(a, stream);
}

}  // namespace gsp
