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
typedef float f16v __attribute__((ext_vector_type(16)));
typedef uint32_t u2 __attribute__((ext_vector_type(2)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

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
    return Terms{{two(lo, std::false_type{}), two(lo, std::true_type{}), two(hi, std::false_type{}),
                  two(hi, std::true_type{})}};
}

// The same fp16 weight beside every activation.
__device__ inline Terms splat_terms(uint32_t half) {
    const uint32_t w = half * 0x10001u;
    return Terms{{w, w, w, w}};
}
constexpr uint32_t kOne = 0x0010, kMinus8 = 0x8080;  // 1 / kCode, -8 / kCode

// Bytes 0 2 1 3 of a dword: the two 16-bit lanes of a mask then hold neighbours.
__device__ inline uint32_t deal_bytes(uint32_t w) { return __builtin_amdgcn_perm(w, w, 0x03010200u); }

// A unit is 256 weights of each of 16 rows, as they lie in memory: 128 or 160
// bytes a row and its scales.  Lane (n, j) reads the j-th 64 of row n from LDS.
template <int WT>
struct Unit {
    static constexpr bool kMins = WT != GSP_WTYPE_Q4_0;
    static constexpr int kRow = WT == GSP_WTYPE_Q4_1 ? 160 : 144;
    // Q4_0, Q4_1: a pair of blocks.  Q4_K: d | dmin, 12 bytes of scales and mins, 32 bytes of quants.
    static constexpr int kWords = WT == GSP_WTYPE_Q4_0 ? 9 : WT == GSP_WTYPE_Q4_1 ? 10 : 12;
    uint32_t w[kWords];

    __device__ inline void read(const uint8_t* rows, int n, int j) {
        const uint8_t* p = rows + n * kRow;
        if constexpr (WT == GSP_WTYPE_Q4_K) {
            const u4 h = *reinterpret_cast<const u4*>(p);
            const u4 a = *reinterpret_cast<const u4*>(p + 16 + 32 * j);
            const u4 b = *reinterpret_cast<const u4*>(p + 32 + 32 * j);
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = h[i], w[4 + i] = a[i], w[8 + i] = b[i];
        } else {
#pragma unroll
            for (int i = 0; i < kWords; ++i) w[i] = *reinterpret_cast<const uint32_t*>(p + 4 * kWords * j + 4 * i);
        }
    }
};

// A unit dealt out for the matrix instruction: dwords of quants with bytes in
// the order 0 2 1 3, and the scales of every group.  Group 2t + h of the unit's
// eight is q[h][t] (Q4_K: the low or the high halves of q[0][t] and q[1][t]).
template <int WT>
struct Dealt {
    uint32_t q[2][4];
    uint32_t s[2][4];
    float d, dmin;  // Q4_K: of the super-block

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
            d = half_lo(u.w[0]);
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
    // Quants times 1 / kCode.
    __device__ inline Terms terms(int t, int h) const {
        if constexpr (WT == GSP_WTYPE_Q4_K) {
            const uint32_t a = q[0][t], b = q[1][t];
            if (h) return Terms{{a & kNib, (a >> 8) & kNib, b & kNib, (b >> 8) & kNib}};
            return Terms{{(a << 4) & kNib, (a >> 4) & kNib, (b << 4) & kNib, (b >> 4) & kNib}};
        }
        const uint32_t a = q[h][t];
        return Terms{{(a << 4) & kNib, (a >> 4) & kNib, a & kNib, (a >> 8) & kNib}};
    }
    // What the tile form multiplies activations by, as normal fp16 numbers formed from 1024 + 16 q in one fused
    // step: q - 8 (Q4_0), q (Q4_1), or q times the group's 6-bit scale, an exact integer up to 945 (Q4_K).  mask:
    // kNib in a register, for one instruction with the or.
    __device__ inline Terms operand(int t, int h, uint32_t mask) const {
        h2 f = {0.0625f16, 0.0625f16}, c = {-64.f16, -64.f16};
        if constexpr (WT == GSP_WTYPE_Q4_0) c = h2{-72.f16, -72.f16};
        if constexpr (WT == GSP_WTYPE_Q4_K) {
            const float sc = (float)((s[0][t] >> (8 * h)) & 0xffu) * 0.0625f;
            f = __builtin_bit_cast(h2, __builtin_amdgcn_cvt_pkrtz(sc, sc));
            c = f * h2{-1024.f16, -1024.f16};
        }
        const auto make = [&](uint32_t w) {
            return __builtin_bit_cast(
                uint32_t, __builtin_elementwise_fma(__builtin_bit_cast(h2, (w & mask) | 0x64006400u), f, c));
        };
        const uint32_t a = WT == GSP_WTYPE_Q4_K ? q[0][t] : q[h][t], b = WT == GSP_WTYPE_Q4_K ? q[1][t] : a;
        if (WT == GSP_WTYPE_Q4_K && h) return Terms{{make(a), make(a >> 8), make(b), make(b >> 8)}};
        if (WT == GSP_WTYPE_Q4_K) return Terms{{make(a << 4), make(a >> 4), make(b << 4), make(b >> 4)}};
        return Terms{{make(a << 4), make(a >> 4), make(a), make(a >> 8)}};
    }
    // The unit's eight minimums as fp16, m (Q4_1) or the 6-bit integer (Q4_K), for the lanes where keep is all ones.
    __device__ inline Terms minimums(uint32_t keep) const {
        Terms t;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (WT == GSP_WTYPE_Q4_K) {
                const float lo = (float)((s[0][i] >> 16) & 0xffu), hi = (float)(s[0][i] >> 24);
                t.r[i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(lo, hi)) & keep;
            } else {
                t.r[i] = __builtin_amdgcn_perm(s[1][i], s[0][i], 0x07060302u) & keep;
            }
        }
        return t;
    }
    // The group's scale, and what the sum of x enters with.
    __device__ inline float scale(int t, int h) const {
        if constexpr (WT == GSP_WTYPE_Q4_0) return h ? half_hi(s[0][t]) : half_lo(s[0][t]);
        if constexpr (WT == GSP_WTYPE_Q4_1) return half_lo(s[h][t]);
        return d * (float)((s[0][t] >> (8 * h)) & 0xffu);
    }
    __device__ inline float least(int t, int h) const {
        if constexpr (WT == GSP_WTYPE_Q4_1) return half_hi(s[h][t]);
        if constexpr (WT == GSP_WTYPE_Q4_K) return -dmin * (float)((s[0][t] >> (16 + 8 * h)) & 0xffu);
        return 0.f;
    }
};

// BYTES of every lane into LDS, one lane's behind the other's from `to` on.
template <int BYTES>
__device__ inline void load_to_lds(const uint8_t* from, uint8_t* to) {
    const auto f = (const __attribute__((address_space(1))) void*)from;
    const auto t = (__attribute__((address_space(3))) void*)to;
    if constexpr (BYTES == 16)
        __builtin_amdgcn_global_load_lds(f, t, 16, 0, 0);
    else
        __builtin_amdgcn_global_load_lds(f, t, 4, 0, 0);
}

// One workgroup: 16 * NT weight rows by 4 * R * MT batch rows.  Its waves share
// the units of K, each with sums of its own, which are added in the order of
// the waves at the end.
//
// Each wave has a slot of LDS for one unit of weights and of activations.  Loads
// go straight there, with neighbouring lanes on neighbouring bytes: a lane that
// loaded what it multiplies would put each 16 bytes of an instruction on another
// row, one cache access a lane.  The wave takes the landed unit into registers and
// sends for the next one before it computes (a second slot, two units ahead, gained
// nothing).  AL: rows of weights are 16-byte aligned and whole units; otherwise they
// are loaded 4 bytes a lane.
//
// R of the four sums that a lane has of a product are used: batch row 4 R m + R j + r
// is row 4 j + r of the m-th operand, so that up to four batch rows (R 1) cost one
// multiply-add an output tile and group, and their activations a quarter of the slot.
//
// One row of 3584 x 37888 (Q4_0) takes 17.4 us, 4.4 TB/s of weights; from some eight rows
// on the vector unit's issue bounds it (16 rows 21 us), and small products the launch and
// the first loads (Q4_1, 8 rows of 896 x 1152, 4.4 us).
template <int WT, int MT, int R, int NT, int W, bool AL>
__global__ __launch_bounds__(64 * W) void matmul_fp8_kernel(MatmulFp8Args a) {
    constexpr int kRow = Unit<WT>::kRow, kTile = 16 * kRow, kX = 4 * R * 256, kSlot = NT * kTile + MT * kX;
    constexpr int kWide = AL ? kTile / 1024 * 1024 : 0;  // of a tile, loaded 16 bytes a lane
    static_assert(kSlot >= NT * MT * R * 256, "the partial sums take the slots' place");
    __shared__ __attribute__((aligned(16))) uint8_t lds[W * kSlot];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    const int n = lane & 15, j = lane >> 4;
    const int tiles_b = (a.batch + 4 * R * MT - 1) / (4 * R * MT);
    const int row0 = blockIdx.x / tiles_b * (16 * NT), b0 = blockIdx.x % tiles_b * (4 * R * MT);
    const int pairs = a.in_dim >> 6, units = (pairs + 3) >> 2;
    uint8_t* slot = lds + wave * kSlot;

    // Where a lane's bytes of a tile lie: the tile's LDS image is 16 rows of kRow bytes, filled in the lanes' order.
    // Bytes past a row's end are its last ones again and meet no product.
    const uint8_t* w0 = static_cast<const uint8_t*>(a.w);
    const auto weight_at = [&](int i, int byte, int u) {
        const int r = byte / kRow, c = byte % kRow;
        const int64_t row = (int64_t)min(row0 + 16 * i + r, a.out_dim - 1) * a.row_bytes;
        int64_t col = (int64_t)u * kRow + c;
        if constexpr (!AL) col = min(col, a.row_bytes - 4);
        return w0 + row + col;
    };
    // Piece p (16 bytes) of row r of activations goes to place p ^ (4 r and on) of the row, so that the reads below
    // spread over the banks.
    const auto turn = [](int r) { return R == 1 ? 4 * r : R == 2 ? 2 * r : r; };
    const auto x_at = [&](int m, int i, int u) {
        const int r = 4 * i + (lane >> 4), p = (lane & 15) ^ turn(r);
        const int64_t row = (int64_t)min(b0 + 4 * R * m + r, a.batch - 1) * a.in_dim;
        return a.x + row + min(u * 256 + p * 16, a.in_dim - 16);
    };
    const auto send = [&](int u) {
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            uint8_t* to = slot + i * kTile;
#pragma unroll
            for (int at = 0; at < kWide; at += 1024) load_to_lds<16>(weight_at(i, at + 16 * lane, u), to + at);
#pragma unroll
            for (int at = kWide; at < kTile; at += 256) load_to_lds<4>(weight_at(i, at + 4 * lane, u), to + at);
        }
#pragma unroll
        for (int m = 0; m < MT; ++m) {
#pragma unroll
            for (int i = 0; i < R; ++i) load_to_lds<16>(x_at(m, i, u), slot + NT * kTile + m * kX + i * 1024);
        }
    };
    // Lane (n, j)'s row of the m-th operand: row n is batch row R (n / 4) + n % 4 where that is below R.
    const int xr = R * (n >> 2) + min(n & 3, R - 1);

    float acc[NT][MT][R];
#pragma unroll
    for (int i = 0; i < NT; ++i) {
#pragma unroll
        for (int m = 0; m < MT; ++m) {
#pragma unroll
            for (int r = 0; r < R; ++r) acc[i][m][r] = 0.f;
        }
    }
    if (wave < units) send(wave);
    for (int u = wave; u < units; u += waves) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the unit has landed
        Unit<WT> raw[NT];
        u4 xq[4][MT];
#pragma unroll
        for (int i = 0; i < NT; ++i) raw[i].read(slot + i * kTile, n, j);
#pragma unroll
        for (int t = 0; t < 4; ++t) {
#pragma unroll
            for (int m = 0; m < MT; ++m)
                xq[t][m] = *reinterpret_cast<const u4*>(slot + NT * kTile + m * kX + xr * 256 + ((4 * t + j) ^ turn(xr)) * 16);
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // and is in registers: the slot may be overwritten
        if (u + waves < units) send(u + waves);
        Dealt<WT> w[NT];
#pragma unroll
        for (int i = 0; i < NT; ++i) w[i].deal(raw[i]);
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            if (!AL && 4 * u + t >= pairs) continue;
            uint32_t x[MT][4];
#pragma unroll
            for (int m = 0; m < MT; ++m) {
#pragma unroll
                for (int i = 0; i < 4; ++i) x[m][i] = xq[t][m][i];
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
                        for (int r = 0; r < R; ++r) {
                            acc[i][m][r] = fmaf(sc, s[r], acc[i][m][r]);
                            if constexpr (Unit<WT>::kMins) acc[i][m][r] = fmaf(mn, sx[m][r], acc[i][m][r]);
                        }
                    }
                }
            }
        }
    }
    __syncthreads();  // every wave is done with its slots
    float* part = reinterpret_cast<float*>(lds);  // [waves][NT][MT][4 R][16]
#pragma unroll
    for (int i = 0; i < NT; ++i) {
#pragma unroll
        for (int m = 0; m < MT; ++m) {
#pragma unroll
            for (int r = 0; r < R; ++r) part[(((wave * NT + i) * MT + m) * 4 * R + R * j + r) * 16 + n] = acc[i][m][r];
        }
    }
    __syncthreads();
    for (int e = threadIdx.x; e < NT * MT * R * 64; e += blockDim.x) {
        float s = 0.f;
        for (int v = 0; v < waves; ++v) s += part[v * (NT * MT * R * 64) + e];
        const int i = e / (MT * R * 64), b = b0 + e / 16 % (MT * R * 4), o = row0 + 16 * i + (e & 15);
        if (b < a.batch && o < a.out_dim) a.y[(int64_t)b * a.out_dim + o] = s * kCode * a.x_scale[b];
    }
}

// Waves for `units` of K, at most `most`, with the units spread evenly.
int even_waves(int units, int most) {
    const int per = (units + most - 1) / most;
    return (units + per - 1) / per;
}

// Rows of weights are whole units and 16-byte aligned.
bool wide_loads(const MatmulFp8Args& a) { return a.in_dim % 256 == 0 && reinterpret_cast<uintptr_t>(a.w) % 16 == 0; }

template <int WT, int MT, int R, int NT, int W>
hipError_t launch_form(MatmulFp8Args a, hipStream_t stream) {
    const int waves = even_waves(a.in_dim / 256 + (a.in_dim % 256 != 0), W);  // in_dim may be close to 2^31
    const bool aligned = wide_loads(a);
    // A launch holds fewer than 2^32 threads: very large batches take several.
    const int64_t tiles = ((int64_t)a.out_dim + 16 * NT - 1) / (16 * NT);
    const int64_t most_rows = std::max<int64_t>(1, (1 << 21) / tiles) * (4 * R * MT);
    for (int64_t left = a.batch; left > 0; left -= most_rows) {
        a.batch = (int32_t)std::min(left, most_rows);
        const uint32_t grid = (uint32_t)(tiles * ((a.batch + 4 * R * MT - 1) / (4 * R * MT)));
        if (aligned)
            hipLaunchKernelGGL((matmul_fp8_kernel<WT, MT, R, NT, W, true>), dim3(grid), dim3(64 * waves), 0, stream, a);
        else
            hipLaunchKernelGGL((matmul_fp8_kernel<WT, MT, R, NT, W, false>), dim3(grid), dim3(64 * waves), 0, stream, a);
        a.x += (int64_t)a.batch * a.in_dim;
        a.x_scale += a.batch;
        a.y += (int64_t)a.batch * a.out_dim;
    }
    return hipGetLastError();
}

// Keeps a value's computation from being moved behind this point, or folded into its uses.
__device__ inline void pin(f4& v) { asm volatile("" : "+v"(v)); }
__device__ inline void pin(f16v& v) { asm volatile("" : "+v"(v)); }
__device__ inline void pin(float& v) { asm volatile("" : "+v"(v)); }

// LDS traffic of the wave is done; the other waves' too after the barrier.
// Loads to LDS stay in flight, which __syncthreads() would wait for.
__device__ inline void lds_barrier() {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// The tile form, for batches that use an expanded weight many times: 16 * MT
// batch rows by 16 * WN weight rows a workgroup.  Each converts its activations to
// fp16 in LDS, in the order the instruction's operands take, 128 of K at a time in
// two buffers.  Each wave has its own 16 weight rows, in a slot as above.
//
// The matrix and the vector units work beside each other: while the products of one
// group run, the previous group's sums are scaled into the outputs' (Q4_0 and Q4_1: one
// fused multiply-add an output and group is the vector unit's main work) and the next
// group's weights are expanded.  Q4_K's scales are integers within the operand, so that
// its sums run over the eight groups of a super-block in the matrix unit alone.
// Minimums meet the sums of x in one more product a unit: staging adds up each group,
// and leaves its sum as two fp16 numbers, the nearest and what that leaves, which hold
// every such sum: it is a multiple of 2^-9 below 2^14, and the rest, of either sign, at
// most half a step of the nearest.
//
// Two heights: 64 rows by 128 (Q4_0, 3584 x 3584 at 512 rows 31.6 us, 416 TFLOP/s) and
// 32 by 64 where that fills the chip better (896 x 4864 at 65 rows 7.8 us).
template <int WT, int MT, int WN, bool AL>
__global__ __launch_bounds__(64 * WN) void matmul_fp8_tile_kernel(MatmulFp8Args a) {
    constexpr int kRow = Unit<WT>::kRow, kTile = 16 * kRow;
    constexpr int G = 4, kSteps = 8 / G;                       // steps of a unit, G groups of 32 each
    constexpr int kStep = MT * G * 1024;                     // LDS bytes of a step's activations
    constexpr int kRowPieces = 2 * G;                        // 16-byte pieces of a row in a step
    constexpr int kPieces = MT * 16 * kRowPieces / (64 * WN);  // pieces a thread stages
    static_assert(kPieces * 64 * WN == MT * 16 * kRowPieces, "even shares");
    __shared__ __attribute__((aligned(16))) uint8_t xs0[kStep];
    __shared__ __attribute__((aligned(16))) uint8_t xs1[kStep];
    const auto x_buf = [&](int step) { return step % 2 ? xs1 : xs0; };
    __shared__ __attribute__((aligned(16))) uint8_t ws[WN][kTile];
    constexpr bool kMins = Unit<WT>::kMins;
    __shared__ __attribute__((aligned(16))) _Float16 gs[kMins ? 2 : 1][kMins ? MT : 1][2][16][8];  // group sums of two units
    __shared__ __attribute__((aligned(16))) float scales[16 * MT];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n = lane & 15, j = lane >> 4;
    const int tiles_b = (a.batch + 16 * MT - 1) / (16 * MT), tiles_n = (a.out_dim + 16 * WN - 1) / (16 * WN);
    // Workgroups go to the eight XCDs in turn: each XCD gets a run of tiles that share weight rows.
    const int tiles = tiles_b * tiles_n;
    const int split = blockIdx.x / tiles;
    int tile = blockIdx.x % tiles;
    const int per_xcd = tiles / 8;
    if (tile < per_xcd * 8) tile = tile % 8 * per_xcd + tile / 8;
    const int row0 = (tile / tiles_b * WN + wave) * 16, b0 = tile % tiles_b * (16 * MT);
    // This split's units of K.
    const int pairs = a.in_dim >> 6;
    const int units = (pairs + 3) >> 2, u0 = split * a.units_per_split, u1 = min(u0 + a.units_per_split, units);

    // Weights: 16 rows' offsets fit 32 bits.  Rows behind the last are the last again.
    const auto send = [&](int u) {
        const int first = min(row0, a.out_dim - 1), rows = a.out_dim - 1 - first;
        const uint8_t* base = static_cast<const uint8_t*>(a.w) + (int64_t)first * a.row_bytes + (int64_t)u * kRow;
        const uint32_t left = (uint32_t)(a.row_bytes - (int64_t)u * kRow - 4);
        const auto at_byte = [&](int byte) {
            const int r = byte / kRow;
            uint32_t col = byte % kRow;
            if constexpr (!AL) col = min(col, left);
            return base + (uint64_t)((uint32_t)min(r, rows) * (uint32_t)a.row_bytes + col);
        };
        constexpr int kWide = AL ? kTile / 1024 * 1024 : 0;
#pragma unroll
        for (int at = 0; at < kWide; at += 1024) load_to_lds<16>(at_byte(at + 16 * lane), ws[wave] + at);
#pragma unroll
        for (int at = kWide; at < kTile; at += 256) load_to_lds<4>(at_byte(at + 4 * lane), ws[wave] + at);
    };
    // Piece i of a thread: 16 bytes of a row, neighbouring lanes on neighbouring pieces.
    u4 piece[kPieces];
    const int b_last = min(16 * MT, a.batch - b0) - 1;
    const auto fetch_x = [&](int step) {
        const uint8_t* base = a.x + (int64_t)b0 * a.in_dim;
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            const int p = i * (64 * WN) + (int)threadIdx.x, r = p / kRowPieces;
            const int c = min(step * (32 * G) + p % kRowPieces * 16, a.in_dim - 16);
            piece[i] = *reinterpret_cast<const u4*>(base + (uint64_t)((uint32_t)min(r, b_last) * (uint32_t)a.in_dim + c));
        }
    };
    // Half of group g of row r is 8 bytes of each of the four lanes (r, j) of the operand; odd groups' rows are turned by
    // eight, so that a wave's writes meet all banks.
    const auto stage_x = [&](int step, uint8_t* buf) {
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            const int p = i * (64 * WN) + (int)threadIdx.x, r = p / kRowPieces, g = p % kRowPieces / 2, half = p & 1;
            uint8_t* to = buf + ((r >> 4) * G + g) * 1024 + ((r & 15) ^ (8 * (g & 1))) * 16 + half * 8;
            float total = 0.f;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const Terms t = x_terms(piece[i][k], 0u);
                *reinterpret_cast<u2*>(to + k * 256) = u2{t.r[0], t.r[1]};
                if constexpr (kMins) {
                    const h2 one = {1.f16, 1.f16};
                    total = __builtin_amdgcn_fdot2(__builtin_bit_cast(h2, t.r[0]), one, total, false);
                    total = __builtin_amdgcn_fdot2(__builtin_bit_cast(h2, t.r[1]), one, total, false);
                }
            }
            if constexpr (kMins) {
                total += __shfl_xor(total, 1);  // the group's other half is the next lane's
                const _Float16 hi = (_Float16)total;
                gs[step / kSteps % 2][r >> 4][half][r & 15][step % kSteps * G + g] =
                    half ? (_Float16)(total - (float)hi) : hi;
            }
        }
    };
    // The operands of one group and of the next.
    Terms xt[2][MT];
    const int read_at[2] = {lane * 16, (lane ^ 8) * 16};
    const auto read_x = [&](const uint8_t* buf, int g) {
#pragma unroll
        for (int m = 0; m < MT; ++m)
            xt[g % 2][m] =
                __builtin_bit_cast(Terms, *reinterpret_cast<const u4*>(buf + (m * G + g) * 1024 + read_at[g % 2]));
    };

    constexpr bool kWholeBlock = WT == GSP_WTYPE_Q4_K;
    f4 acc[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) acc[m] = f4{0.f, 0.f, 0.f, 0.f};
    const f4 zero = {0.f, 0.f, 0.f, 0.f};
    uint32_t mask = kNib;
    asm volatile("" : "+v"(mask));
    f4 sum[kWholeBlock ? 1 : 2][MT];  // Q4_K: the super-block's sums; else the last two groups'
    const uint32_t keep = j < 2 ? 0xffffffffu : 0u;
    Dealt<WT> w;
    send(u0);
    if (threadIdx.x < 16 * MT) scales[threadIdx.x] = a.x_scale[min(b0 + (int)threadIdx.x, a.batch - 1)];
    fetch_x(kSteps * u0);
    stage_x(kSteps * u0, x_buf(0));
    fetch_x(kSteps * u0 + 1);
    lds_barrier();
    read_x(x_buf(0), 0);
    float sc_last = 0.f;
    if constexpr (!kWholeBlock) {
#pragma unroll
        for (int m = 0; m < MT; ++m) sum[1][m] = zero;
    }
    for (int u = u0; u < u1; ++u) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the unit's weights have landed
        Unit<WT> raw;
        raw.read(ws[wave], n, j);
        w.deal(raw);
        Terms q = w.operand(0, 0, mask);
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            // The buffer written here was last read before the barrier below, in the step before.  At the end the last
            // step and unit are loaded again, for nobody.
            stage_x(kSteps * u + s + 1, x_buf(s + 1));
            fetch_x(min(kSteps * u + s + 2, kSteps * u1 - 1));
            if (s == 0) {
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the unit's weights are in registers
                send(min(u + 1, u1 - 1));
            }
#pragma unroll
            for (int g = 0; g < G; ++g) {
                const int ug = s * G + g, t = ug / 2, h = ug % 2;
                if (g == G - 1) lds_barrier();  // the next step's activations are staged, this step's in registers
                read_x(x_buf(g < G - 1 ? s : s + 1), (g + 1) % G);
                float sc = 0.f;
                if constexpr (!kWholeBlock) sc = AL || 4 * u + t < pairs ? w.scale(t, h) : 0.f;
#pragma unroll
                for (int m = 0; m < MT; ++m) {
                    if constexpr (kWholeBlock) {
                        sum[0][m] = mfma(xt[g % 2][m], q, ug == 0 ? zero : sum[0][m]);
                    } else {
                        sum[g % 2][m] = mfma(xt[g % 2][m], q, zero);
#pragma unroll
                        for (int r = 0; r < 4; ++r) acc[m][r] = fmaf(sc_last, sum[(g + 1) % 2][m][r], acc[m][r]);
                    }
                }
                if (ug < 7) q = w.operand((ug + 1) / 2, (ug + 1) % 2, mask);
                sc_last = sc;
                pin(sc_last);
#pragma unroll
                for (int m = 0; m < MT; ++m) pin(acc[m]);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        if constexpr (kMins) {
            Terms mn = w.minimums(keep);
#pragma unroll
            for (int t = 0; t < 4; ++t)
                if (!AL && 4 * u + t >= pairs) mn.r[t] = 0;
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                const Terms ms = __builtin_bit_cast(Terms, *reinterpret_cast<const u4*>(&gs[u % 2][m][j & 1][n][0]));
                if constexpr (kWholeBlock) {
                    const f4 low = mfma(ms, mn, zero);
#pragma unroll
                    for (int r = 0; r < 4; ++r) acc[m][r] = fmaf(w.d, sum[0][m][r], fmaf(-w.dmin, low[r], acc[m][r]));
                    pin(acc[m]);
                } else {
                    acc[m] = mfma(ms, mn, acc[m]);
                }
            }
        }
    }
    if constexpr (!kWholeBlock) {
#pragma unroll
        for (int m = 0; m < MT; ++m) {
#pragma unroll
            for (int r = 0; r < 4; ++r) acc[m][r] = fmaf(sc_last, sum[1][m][r], acc[m][r]);
        }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // no load outlives the loop
    float* y = a.partials ? a.partials + (int64_t)split * a.batch * a.out_dim : a.y;
    const bool whole = b0 + 16 * MT <= a.batch && row0 + 16 <= a.out_dim;
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        const f4 f = *reinterpret_cast<const f4*>(&scales[16 * m + 4 * j]);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int b = b0 + 16 * m + 4 * j + r;
            if (whole || (b < a.batch && row0 + n < a.out_dim)) y[(int64_t)b * a.out_dim + row0 + n] = acc[m][r] * f[r];
        }
    }
}

// 256 weights of each of 32 rows for the 32 x 32 x 16 instruction (two a group of 32
// weights: lane (n, h) = (lane % 32, lane / 32) holds dwords 2h + p of
// row n in the p-th).  A lane reads half a row's blocks from LDS and trades every
// second register with the lane of the other half.
template <int WT>
struct Rows {
    uint32_t q[16];  // bytes in the order 0 2 1 3; Q4_0, Q4_1: group g's p-th at 2 g + p; Q4_K: a pair of groups' at 4, + 2 p
    uint32_t s[8];   // Q4_0: two groups' d each; Q4_1: a group's d and m; Q4_K: four scales, four, four minimums, four
    float d, dmin;   // Q4_K: of the super-block

    __device__ inline void read(const uint8_t* rows, int n, int h) {
        const uint8_t* p = rows + n * Unit<WT>::kRow;
        if constexpr (WT == GSP_WTYPE_Q4_K) {
            const u4 head = *reinterpret_cast<const u4*>(p);
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const u4 a = *reinterpret_cast<const u4*>(p + 16 + 64 * h + 32 * c);
                const u4 b = *reinterpret_cast<const u4*>(p + 32 + 64 * h + 32 * c);
                // Dword i of a byte row belongs to lane half i / 2.
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    uint32_t a0 = deal_bytes(a[i]), a1 = deal_bytes(a[2 + i]), b0 = deal_bytes(b[i]), b1 = deal_bytes(b[2 + i]);
                    swap32(a0, a1);
                    swap32(b0, b1);
                    q[4 * c + 2 * i] = a0, q[4 * c + 2 * i + 1] = b0;
                    q[8 + 4 * c + 2 * i] = a1, q[8 + 4 * c + 2 * i + 1] = b1;
                }
            }
            d = half_lo(head[0]);
            dmin = half_hi(head[0]);
            s[0] = head[1] & 0x3f3f3f3fu;
            s[1] = (head[3] & 0x0f0f0f0fu) | (head[1] & 0xc0c0c0c0u) >> 2;
            s[2] = head[2] & 0x3f3f3f3fu;
            s[3] = (head[3] >> 4 & 0x0f0f0f0fu) | (head[2] & 0xc0c0c0c0u) >> 2;
        } else {
            constexpr int kWords = Unit<WT>::kRow / 8;
            uint32_t w[kWords];
#pragma unroll
            for (int i = 0; i < kWords; i += 2) {
                const u2 two = *reinterpret_cast<const u2*>(p + 4 * kWords * h + 4 * i);
                w[i] = two[0], w[i + 1] = two[1];
            }
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                uint32_t e[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if constexpr (WT == GSP_WTYPE_Q4_1)
                        e[i] = deal_bytes(w[5 * b + 1 + i]);
                    else if (b % 2)
                        e[i] = deal_bytes(w[9 * (b / 2) + 5 + i]);
                    else  // between two dwords
                        e[i] = __builtin_amdgcn_perm(w[9 * (b / 2) + i + 1], w[9 * (b / 2) + i], 0x05030402u);
                }
                swap32(e[0], e[2]);
                swap32(e[1], e[3]);
                q[2 * b] = e[0], q[2 * b + 1] = e[1], q[8 + 2 * b] = e[2], q[8 + 2 * b + 1] = e[3];
            }
            constexpr int kScales = WT == GSP_WTYPE_Q4_1 ? 4 : 2;  // dwords a lane
#pragma unroll
            for (int i = 0; i < kScales; ++i) {
                uint32_t a = WT == GSP_WTYPE_Q4_1 ? w[5 * i] : (w[9 * i] & 0xffffu) | (w[9 * i + 4] & 0xffff0000u), b = a;
                swap32(a, b);
                s[i] = a, s[kScales + i] = b;
            }
        }
    }
    // Quants of group g times 1 / kCode (Q4_0, Q4_1).
    __device__ inline Terms quants(int g, int p, uint32_t mask) const {
        const uint32_t a = q[2 * g + p];
        return Terms{{(a << 4) & mask, (a >> 4) & mask, a & mask, (a >> 8) & mask}};
    }
    // The p-th operand of group g: q - 8 (Q4_0) and q times the group's 6-bit scale, an exact integer up to 945 (Q4_K),
    // formed from 1024 + 16 q in one fused step, or q times 1 / kCode (Q4_1).  mask: kNib in a register.
    __device__ inline Terms operand(int g, int p, uint32_t mask) const {
        if constexpr (WT == GSP_WTYPE_Q4_1) return quants(g, p, mask);
        h2 f = {0.0625f16, 0.0625f16}, c = {-72.f16, -72.f16};
        if constexpr (WT == GSP_WTYPE_Q4_K) {
            const float sc = (float)((s[g / 4] >> (8 * (g % 4))) & 0xffu) * 0.0625f;
            f = __builtin_bit_cast(h2, __builtin_amdgcn_cvt_pkrtz(sc, sc));
            c = f * h2{-1024.f16, -1024.f16};
        }
        const auto make = [&](uint32_t w) {
            return __builtin_bit_cast(
                uint32_t, __builtin_elementwise_fma(__builtin_bit_cast(h2, (w & mask) | 0x64006400u), f, c));
        };
        const uint32_t a = WT == GSP_WTYPE_Q4_K ? q[g / 2 * 4 + 2 * p] : q[2 * g + p];
        const uint32_t b = WT == GSP_WTYPE_Q4_K ? q[g / 2 * 4 + 2 * p + 1] : a;
        if (WT == GSP_WTYPE_Q4_K && g % 2) return Terms{{make(a), make(a >> 8), make(b), make(b >> 8)}};
        if (WT == GSP_WTYPE_Q4_K) return Terms{{make(a << 4), make(a >> 4), make(b << 4), make(b >> 4)}};
        return Terms{{make(a << 4), make(a >> 4), make(a), make(a >> 8)}};
    }
    // What a group's sum of products enters with.
    __device__ inline float scale(int g) const {
        if constexpr (WT == GSP_WTYPE_Q4_1) return half_lo(s[g]) * kCode;
        return g % 2 ? half_hi(s[g / 2]) : half_lo(s[g / 2]);
    }
    // What the eight groups' sums of x enter with, as fp16: m (Q4_1) or the 6-bit minimum (Q4_K).
    __device__ inline Terms minimums() const {
        Terms t;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (WT == GSP_WTYPE_Q4_K) {
                const uint32_t two = s[2 + i / 2] >> (16 * (i % 2));
                t.r[i] = __builtin_bit_cast(uint32_t,
                                            __builtin_amdgcn_cvt_pkrtz((float)(two & 0xffu), (float)(two >> 8 & 0xffu)));
            } else {
                t.r[i] = __builtin_amdgcn_perm(s[2 * i + 1], s[2 * i], 0x07060302u);
            }
        }
        return t;
    }
};

__device__ inline f16v mfma32(const Terms& a, const Terms& b, f16v c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
}

// The stream form of more rows: 32 weight rows by 32 batch rows a workgroup, in the
// 32 x 32 x 16 instruction, its waves sharing the units of K as above.  A lane's
// activations of a group are two pieces of 8 bytes of its row, which LDS gives it as
// they are.  A unit's sums of x by group are products as well, with ones in row g for
// group g: they arrive as [group][batch row], four groups a lane half, and meet the
// minimums as two fp16 numbers each in one product.  Rows of weights are whole units,
// 16-byte aligned.  us, 64 rows of 18944 x 3584: Q4_0 22.9, Q4_1 24.1, Q4_K 24.5, with
// 16 x 16 x 32 products 26.7, 33.3 and 31.9: fewer of them, no swaps of activations, and
// minimums and Q4_K's scales without the vector unit, whose issue bounds both.
template <int WT, int W>
__global__ __launch_bounds__(64 * W) void matmul_fp8_stream32_kernel(MatmulFp8Args a) {
    constexpr int kRow = Unit<WT>::kRow, kTile = 32 * kRow, kX = 32 * 256, kSlot = kTile + kX;
    constexpr int kWide = kTile / 1024 * 1024;  // of the weights, loaded 16 bytes a lane
    constexpr bool kMins = Unit<WT>::kMins, kWholeBlock = WT == GSP_WTYPE_Q4_K;
    // Q4_0's sums start at -8 / kCode times the sum of x: two products instead of eight instructions an operand.
    constexpr bool kStart = WT == GSP_WTYPE_Q4_0;
    constexpr float kOut = kStart ? kCode : 1.f;
    static_assert(kSlot >= 4096, "the partial sums take the slots' place");
    __shared__ __attribute__((aligned(16))) uint8_t lds[W * kSlot];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    const int n = lane & 31, h = lane >> 5;
    const int tiles_b = (a.batch + 31) / 32;
    const int row0 = blockIdx.x / tiles_b * 32, b0 = blockIdx.x % tiles_b * 32;
    const int units = a.in_dim >> 8;
    uint8_t* slot = lds + wave * kSlot;

    const auto weight_at = [&](int byte, int u) {
        const int r = byte / kRow, c = byte % kRow;
        const int64_t row = (int64_t)min(row0 + r, a.out_dim - 1) * a.row_bytes;
        return static_cast<const uint8_t*>(a.w) + row + (int64_t)u * kRow + c;
    };
    // Piece p (16 bytes) of row r of activations goes to place p ^ r of the row, so that the reads below spread over the
    // banks.
    const auto send = [&](int u) {
#pragma unroll
        for (int at = 0; at < kWide; at += 1024) load_to_lds<16>(weight_at(at + 16 * lane, u), slot + at);
#pragma unroll
        for (int at = kWide; at < kTile; at += 256) load_to_lds<4>(weight_at(at + 4 * lane, u), slot + at);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int r = 4 * i + (lane >> 4), p = (lane & 15) ^ (r & 15);
            const int64_t row = (int64_t)min(b0 + r, a.batch - 1) * a.in_dim;
            load_to_lds<16>(a.x + row + u * 256 + p * 16, slot + kTile + i * 1024);
        }
    };

    const f16v zero = {};
    f16v acc = zero, sum[2] = {zero, zero};
    float sc_last = 0.f;
    uint32_t mask = kNib;
    asm volatile("" : "+v"(mask));
    if (wave < units) send(wave);
    for (int u = wave; u < units; u += waves) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the unit has landed
        Rows<WT> w;
        w.read(slot, n, h);
        u2 x[8][2];
#pragma unroll
        for (int g = 0; g < 8; ++g) {
#pragma unroll
            for (int i = 0; i < 2; ++i)
                x[g][i] = *reinterpret_cast<const u2*>(slot + kTile + n * 256 + ((2 * g + i) ^ (n & 15)) * 16 + 8 * h);
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // and is in registers: the slot may be overwritten
        if (u + waves < units) send(u + waves);
        f16v sx = zero;
#pragma unroll
        for (int g = 0; g < 8; ++g) {
            Terms xt[2];
#pragma unroll
            for (int p = 0; p < 2; ++p) xt[p] = x_terms(x[g][0][p], x[g][1][p]);
            const int at = kWholeBlock ? 0 : g % 2;
            if constexpr (kStart) {
#pragma unroll
                for (int p = 0; p < 2; ++p) sum[at] = mfma32(xt[p], splat_terms(kMinus8), p ? sum[at] : zero);
#pragma unroll
                for (int p = 0; p < 2; ++p) sum[at] = mfma32(xt[p], w.quants(g, p, mask), sum[at]);
            } else {
#pragma unroll
                for (int p = 0; p < 2; ++p)
                    sum[at] = mfma32(xt[p], w.operand(g, p, mask), p || (kWholeBlock && g) ? sum[at] : zero);
            }
            if constexpr (kMins) {
                const Terms ones = splat_terms(n == g ? 0x3c00u : 0u);
#pragma unroll
                for (int p = 0; p < 2; ++p) sx = mfma32(ones, xt[p], sx);
            }
            if constexpr (!kWholeBlock) {
#pragma unroll
                for (int r = 0; r < 16; ++r) acc[r] = fmaf(sc_last, sum[1 - at][r], acc[r]);
                sc_last = w.scale(g);
            }
        }
        if constexpr (kMins) {
            Terms mn = w.minimums(), ms;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const float s0 = sx[2 * i], s1 = sx[2 * i + 1];
                const h2 first = {(_Float16)s0, (_Float16)s1};
                const h2 rest = {(_Float16)(s0 - (float)first[0]), (_Float16)(s1 - (float)first[1])};
                ms.r[i] = __builtin_bit_cast(uint32_t, first);
                ms.r[2 + i] = __builtin_bit_cast(uint32_t, rest);
                mn.r[i] = h ? mn.r[2 + i] : mn.r[i];
                mn.r[2 + i] = mn.r[i];
            }
            if constexpr (kWholeBlock) {
                const f16v low = mfma32(ms, mn, zero);
#pragma unroll
                for (int r = 0; r < 16; ++r) acc[r] = fmaf(w.d, sum[0][r], fmaf(-w.dmin, low[r], acc[r]));
            } else {
                acc = mfma32(ms, mn, acc);
            }
        }
    }
    if constexpr (!kWholeBlock) {
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[r] = fmaf(sc_last, sum[1][r], acc[r]);
    }
    __syncthreads();  // every wave is done with its slots
    float* part = reinterpret_cast<float*>(lds);  // [waves][16][lane]
#pragma unroll
    for (int r = 0; r < 16; ++r) part[(wave * 16 + r) * 64 + lane] = acc[r];
    __syncthreads();
    for (int e = threadIdx.x; e < 1024; e += blockDim.x) {
        float s = 0.f;
        for (int v = 0; v < waves; ++v) s += part[v * 1024 + e];
        const int r = e >> 6, b = b0 + (r & 3) + 8 * (r >> 2) + 4 * (e >> 5 & 1), o = row0 + (e & 31);
        if (b < a.batch && o < a.out_dim) a.y[(int64_t)b * a.out_dim + o] = s * kOut * a.x_scale[b];
    }
}

// The wide tile form: 128 batch rows by 256 weight rows a workgroup, 128 by 32 a wave,
// in the 32 x 32 x 16 instruction, of which half as many are issued for the same terms.
// Beside a multiply-add for each output it takes 9.3 ns a SIMD for 16 x 16 x 32 terms,
// the other one 11.2.  With Q4_0 and Q4_1 the vector unit issues three quarters of the
// time (3584 x 18944 at 2048 rows), with 512 multiply-adds, 176 instructions of expansion
// (Q4_0), 64 products and 63 others a wave and unit; the matrix unit is busy 45 %.  Q4_K,
// whose scales are in its operands, has 35 % fewer instructions and takes 3 % less: both
// units are busy half of the time, and waves wait to issue a third of it.  LDS leaves room
// for one workgroup a CU, two waves a SIMD to cover each other's products.  Activations
// come converted from matmul_fp8_convert_kernel (9 us there), as converting them in every
// workgroup took 4 % longer.  us at 2048 rows (TFLOP/s), 3584 x 18944 and 18944 x 3584:
// Q4_0 331 (840) and 326, Q4_1 338 and 330, Q4_K 324 and 315; another card took 4 % less.
// Q4_1 with 4-byte loads is short of registers and spills 13 of them (896 x 9728 at 2048
// rows 92 us, Q4_0 78).
//
// Measured without gain: the loads to LDS sent one by one between the products, the
// weights read before their unit begins, activations through registers, the barrier
// behind a product, and 32 x 32 x 16 tiles of 64 or 32 rows (3584 x 3584 at 512 rows
// 40 us instead of 32: too few waves a SIMD).
constexpr int kWideRows = kMatmulFp8WideRows, kWideWaves = kMatmulFp8WideCols / 32;
template <int WT, bool AL>
__global__ __launch_bounds__(64 * kWideWaves) void matmul_fp8_wide_kernel(MatmulFp8Args a) {
    constexpr int kRow = Unit<WT>::kRow, kTile = 16 * kRow;
    constexpr int MT = kWideRows / 32, WN = kWideWaves, G = 4, kSteps = 8 / G;  // steps of a unit, G groups of 32 each
    constexpr int kStep = MT * G * 2048;      // LDS bytes of a step's activations
    constexpr int kBlocks = 2 * MT * G / WN;  // KB that a wave loads of them
    static_assert(MT == 4 && kBlocks * WN == 2 * MT * G && 2 * MT == WN, "even shares");
    // Two arrays, so that the compiler sees that loads into one do not concern reads of the other.
    __shared__ __attribute__((aligned(16))) uint8_t xs0[kStep];
    __shared__ __attribute__((aligned(16))) uint8_t xs1[kStep];
    const auto x_buf = [&](int step) { return step % 2 ? xs1 : xs0; };
    __shared__ __attribute__((aligned(16))) uint8_t ws[WN][2 * kTile];
    constexpr bool kMins = Unit<WT>::kMins;
    __shared__ __attribute__((aligned(16))) _Float16 gs[kMins ? 2 : 1][kMins ? MT : 1][2][32][8];  // group sums of two units
    __shared__ __attribute__((aligned(16))) float scales[32 * MT];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n = lane & 31, h = lane >> 5;
    const int tiles_b = (a.batch + 32 * MT - 1) / (32 * MT), tiles_n = (a.out_dim + 32 * WN - 1) / (32 * WN);
    // Workgroups go to the eight XCDs in turn: each XCD gets a run of tiles that share weight rows.
    const int tiles = tiles_b * tiles_n;
    const int split = blockIdx.x / tiles;
    int tile = blockIdx.x % tiles;
    const int per_xcd = tiles / 8;
    if (tile < per_xcd * 8) tile = tile % 8 * per_xcd + tile / 8;
    const int row0 = (tile / tiles_b * WN + wave) * 32, b0 = tile % tiles_b * (32 * MT);
    // This split's units of K.
    const int pairs = a.in_dim >> 6;
    const int units = (pairs + 3) >> 2, u0 = split * a.units_per_split, u1 = min(u0 + a.units_per_split, units);

    // Weights: 16 rows' offsets fit 32 bits.  Rows behind the last are the last again.
    constexpr int kWide16 = AL ? kTile / 1024 : 0, kTileLoads = kWide16 + (kTile - 1024 * kWide16) / 256;
    constexpr int kLoads = 2 * kTileLoads;  // of a unit's weights
    const auto send_w = [&](int u, int load) {
        const int i = load / kTileLoads, k = load % kTileLoads;
        const int first = min(row0 + 16 * i, a.out_dim - 1), rows = a.out_dim - 1 - first;
        const uint8_t* base = static_cast<const uint8_t*>(a.w) + (int64_t)first * a.row_bytes + (int64_t)u * kRow;
        const uint32_t left = (uint32_t)(a.row_bytes - (int64_t)u * kRow - 4);
        const int at = k < kWide16 ? 1024 * k : 1024 * kWide16 + 256 * (k - kWide16);
        const int byte = at + (k < kWide16 ? 16 : 4) * lane, r = byte / kRow;
        uint32_t col = byte % kRow;
        if constexpr (!AL) col = min(col, left);
        const uint8_t* from = base + (uint64_t)((uint32_t)min(r, rows) * (uint32_t)a.row_bytes + col);
        if (k < kWide16)
            load_to_lds<16>(from, &ws[wave][i * kTile + at]);
        else
            load_to_lds<4>(from, &ws[wave][i * kTile + at]);
    };
    // Converted activations: a step's KB of half the operands of 32 rows and a group each, and a unit's group sums, half
    // of 32 rows a wave.
    const auto send_x = [&](int step, uint8_t* to, int load) {
        const int kb = wave * kBlocks + load, m = kb / (2 * G), half = kb % (2 * G);
        const int64_t at = (((int64_t)(b0 / 32 + m) * units * 8 + step * G) * 2 + half) * 1024;
        load_to_lds<16>(a.xf + at + 16 * lane, to + kb * 1024);
    };
    const auto send_sums = [&](int u) {
        if (lane < 32)
            load_to_lds<16>(a.sums + (((int64_t)(b0 / 32 + wave / 2) * units + u) * 2 + wave % 2) * 512 + 16 * lane,
                            reinterpret_cast<uint8_t*>(&gs[kMins ? u % 2 : 0][kMins ? wave / 2 : 0][wave % 2][0][0]));
    };
    // A group's operands, replaced in place by the next group's behind the products that use them.
    Terms xt[MT][2];
    const auto read_x = [&](const uint8_t* buf, int g, int m) {
        const uint8_t* from = buf + (m * G + g) * 2048 + h * 512 + n * 16;
#pragma unroll
        for (int p = 0; p < 2; ++p) xt[m][p] = __builtin_bit_cast(Terms, *reinterpret_cast<const u4*>(from + p * 1024));
    };

    constexpr bool kWholeBlock = WT == GSP_WTYPE_Q4_K;
    // Sums of a super-block, or of the last products, all but one of them on the way (two instead of four: 2 % longer).
    constexpr int kBuf = MT, kBehind = kBuf - 1;
    const f16v zero = {};
    f16v acc[MT], sum[kBuf];
#pragma unroll
    for (int m = 0; m < MT; ++m) acc[m] = zero;
    uint32_t mask = kNib;
    asm volatile("" : "+v"(mask));
    Rows<WT> w;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) send_w(u0, i);
    if (threadIdx.x < 32 * MT) scales[threadIdx.x] = a.x_scale[min(b0 + (int)threadIdx.x, a.batch - 1)];
    if constexpr (kMins) send_sums(u0);
#pragma unroll
    for (int i = 0; i < kBlocks; ++i) send_x(kSteps * u0, x_buf(0), i);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    lds_barrier();
#pragma unroll
    for (int m = 0; m < MT; ++m) read_x(x_buf(0), 0, m);
    float sc_last = 0.f;
    if constexpr (!kWholeBlock) {
#pragma unroll
        for (int i = 0; i < kBuf; ++i) sum[i] = zero;
    }
    const auto add = [&](int m, float sc, const f16v& s, int from) {
#pragma unroll
        for (int r = from; r < from + 8; ++r) acc[m][r] = fmaf(sc, s[r], acc[m][r]);
    };
    for (int u = u0; u < u1; ++u) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the unit's weights have landed
        w.read(ws[wave], n, h);
        Terms q[2] = {w.operand(0, 0, mask), w.operand(0, 1, mask)};
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            // The buffer written in this step was last read before the barrier below, in the step before.  At the end the
            // last step and unit are loaded again, for nobody, so that the waits' counts hold.
#pragma unroll
            for (int i = 0; i < kBlocks; ++i) send_x(min(kSteps * u + s + 1, kSteps * u1 - 1), x_buf(s + 1), i);
            if (s == 0) {
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the unit's weights are in registers
#pragma unroll
                for (int i = 0; i < kLoads; ++i) send_w(min(u + 1, u1 - 1), i);
            }
#pragma unroll
            for (int g = 0; g < G; ++g) {
                const int ug = s * G + g;
                Terms next[2];
                float sc = 0.f;
                if constexpr (!kWholeBlock) sc = AL || 4 * u + ug / 2 < pairs ? w.scale(ug) : 0.f;
#pragma unroll
                for (int m = 0; m < MT; ++m) {
                    if (g == G - 1 && m == 0) {
                        // The next step's activations have landed, this step's are in registers.  Loads complete in order,
                        // and behind the next step's only the next unit's weights were sent for, in a unit's first step.
                        asm volatile("s_waitcnt vmcnt(%0)" ::"n"(s == 0 ? kLoads : 0) : "memory");
                        lds_barrier();
                        if constexpr (kMins)
                            if (s == 0) send_sums(min(u + 1, u1 - 1));  // every wave is past the sums of the unit before
                    }
                    // Half of an operand of the next group beside each pair of products.  The order matters: scheduled by
                    // the compiler, with whole operands beside every other pair, 18944 x 3584 takes 318 us instead of 305
                    // (Q4_0, 2048 rows).
                    const auto expand = [&] {
                        if (ug == 7) return;
                        const Terms whole = w.operand(ug + 1, m / 2, mask);
                        for (int i = 0; i < 2; ++i) next[m / 2].r[m % 2 * 2 + i] = whole.r[m % 2 * 2 + i];
                    };
                    const uint8_t* next_x = x_buf(g < G - 1 ? s : s + 1);
                    if constexpr (kWholeBlock) {
                        sum[m] = mfma32(xt[m][0], q[0], ug == 0 ? zero : sum[m]);
                        __builtin_amdgcn_sched_barrier(0);
                        expand();
                        __builtin_amdgcn_sched_barrier(0);
                        sum[m] = mfma32(xt[m][1], q[1], sum[m]);
                        __builtin_amdgcn_sched_barrier(0);
                        read_x(next_x, (g + 1) % G, m);
                    } else {
                        const int at = (g * MT + m) % kBuf, then = (at + 1) % kBuf, tm = (m + MT - kBehind) % MT;
                        const float ts = m >= kBehind ? sc : sc_last;
                        sum[at] = mfma32(xt[m][0], q[0], zero);
                        __builtin_amdgcn_sched_barrier(0);
                        add(tm, ts, sum[then], 0);
                        __builtin_amdgcn_sched_barrier(0);
                        sum[at] = mfma32(xt[m][1], q[1], sum[at]);
                        __builtin_amdgcn_sched_barrier(0);
                        read_x(next_x, (g + 1) % G, m);
                        add(tm, ts, sum[then], 8);
                        pin(acc[tm]);
                        expand();
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
                if (ug < 7) q[0] = next[0], q[1] = next[1];
                sc_last = sc;
                pin(sc_last);
            }
        }
        if constexpr (kMins) {
            Terms mn = w.minimums();
#pragma unroll
            for (int t = 0; t < 4; ++t)
                if (!AL && 4 * u + t >= pairs) mn.r[t] = 0;
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                const Terms ms = __builtin_bit_cast(Terms, *reinterpret_cast<const u4*>(&gs[u % 2][m][h][n][0]));
                if constexpr (kWholeBlock) {
                    const f16v low = mfma32(ms, mn, zero);
#pragma unroll
                    for (int r = 0; r < 16; ++r) acc[m][r] = fmaf(w.d, sum[m][r], fmaf(-w.dmin, low[r], acc[m][r]));
                    pin(acc[m]);
                } else {
                    acc[m] = mfma32(ms, mn, acc[m]);
                }
            }
        }
    }
    if constexpr (!kWholeBlock) {
#pragma unroll
        for (int i = 1; i <= kBehind; ++i) {
            const int m = MT - 1 - kBehind + i, at = i % kBuf;  // the last products' places, as the step's count is 0 mod kBuf
            add(m, sc_last, sum[at], 0);
            add(m, sc_last, sum[at], 8);
        }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // no load outlives the loop
    float* y = a.partials ? a.partials + (int64_t)split * a.batch * a.out_dim : a.y;
    const bool whole = b0 + 32 * MT <= a.batch && row0 + 32 <= a.out_dim;
#pragma unroll
    for (int m = 0; m < MT; ++m) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const f4 f = *reinterpret_cast<const f4*>(&scales[32 * m + 8 * i + 4 * h]);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int b = b0 + 32 * m + 8 * i + 4 * h + r;
                if (whole || (b < a.batch && row0 + n < a.out_dim))
                    y[(int64_t)b * a.out_dim + row0 + n] = acc[m][4 * i + r] * f[r];
            }
        }
    }
}

// Activations for the wide tile form: fp16 in the operands' order, [32 rows][group]
// of 2 KB, in it [p][h][row] 16 bytes, and each group's sum as two fp16 numbers,
// [32 rows][unit][2][row][group].  Rows and groups past the end are 0.  A thread
// converts one group of a row.
__global__ __launch_bounds__(256) void matmul_fp8_convert_kernel(const uint8_t* x, uint8_t* xf, _Float16* sums, int in_dim,
                                                                 int batch, int units) {
    const int n = threadIdx.x & 31, g = threadIdx.x >> 5;
    const int64_t tile = blockIdx.x / units;
    const int u = blockIdx.x % units;
    const int64_t row = tile * 32 + n;
    const int k = u * 256 + g * 32;
    u4 lo = {0, 0, 0, 0}, hi = lo;
    if (row < batch && k < in_dim) {
        const uint8_t* p = x + row * in_dim + k;
        lo = *reinterpret_cast<const u4*>(p);
        hi = *reinterpret_cast<const u4*>(p + 16);
    }
    uint8_t* to = xf + ((tile * units + u) * 8 + g) * 2048 + n * 16;
    float total = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const Terms t = x_terms(lo[j], hi[j]);
        *reinterpret_cast<u4*>(to + (j % 2 * 2 + j / 2) * 512) = __builtin_bit_cast(u4, t);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            total = __builtin_amdgcn_fdot2(__builtin_bit_cast(h2, t.r[i]), h2{1.f16, 1.f16}, total, false);
    }
    if (sums) {
        _Float16* s = sums + (tile * units + u) * 512 + n * 8 + g;
        const _Float16 first = (_Float16)total;
        s[0] = first;
        s[256] = (_Float16)(total - (float)first);
    }
}

// The splits' sums, in their order.
__global__ __launch_bounds__(256) void add_splits_kernel(const float* part, float* y, int64_t n, int splits) {
    for (int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x; at < n; at += (int64_t)gridDim.x * 256) {
        float s = part[at];
        for (int i = 1; i < splits; ++i) s += part[i * n + at];
        y[at] = s;
    }
}

template <int WT, int W>
hipError_t launch_stream32(const MatmulFp8Args& a, hipStream_t stream) {
    const uint32_t grid = (uint32_t)((a.out_dim + 31) / 32 * ((a.batch + 31) / 32));
    hipLaunchKernelGGL((matmul_fp8_stream32_kernel<WT, W>), dim3(grid), dim3(64 * even_waves(a.in_dim / 256, W)), 0, stream, a);
    return hipGetLastError();
}

// Rows of a launch, which holds fewer than 2^32 threads: very large batches take several.
int64_t launch_rows(int64_t others, int rows) { return std::max<int64_t>(1, (1 << 21) / others) * rows; }

void add_splits(const MatmulFp8Args& a, int splits, hipStream_t stream) {
    const int64_t n = (int64_t)a.batch * a.out_dim;
    hipLaunchKernelGGL(add_splits_kernel, dim3((uint32_t)std::min<int64_t>((n + 255) / 256, 2048)), dim3(256), 0, stream,
                       a.partials, a.y, n, splits);
}

// The tile forms: `rows` x `cols` a workgroup, `launch` of them a piece of the batch.
template <class Launch>
hipError_t launch_tiles(MatmulFp8Args a, int splits, int rows, int cols, int64_t most_rows, hipStream_t stream, Launch launch) {
    a.units_per_split = ((a.in_dim + 255) / 256 + splits - 1) / splits;
    if (splits == 1) a.partials = nullptr;
    const int64_t tiles_n = ((int64_t)a.out_dim + cols - 1) / cols;
    most_rows = std::min(most_rows, launch_rows(tiles_n, rows));
    for (int64_t left = a.batch; left > 0; left -= most_rows) {
        a.batch = (int32_t)std::min(left, most_rows);
        launch(a, dim3((uint32_t)(tiles_n * ((a.batch + rows - 1) / rows) * splits)));
        if (splits > 1) add_splits(a, splits, stream);
        a.x += (int64_t)a.batch * a.in_dim;
        a.x_scale += a.batch;
        a.y += (int64_t)a.batch * a.out_dim;
    }
    return hipGetLastError();
}

template <int WT, int MT, int WN>
hipError_t launch_tile(const MatmulFp8Args& all, int splits, hipStream_t stream) {
    return launch_tiles(all, splits, 16 * MT, 16 * WN, all.batch, stream, [&](const MatmulFp8Args& a, dim3 grid) {
        if (wide_loads(a))
            hipLaunchKernelGGL((matmul_fp8_tile_kernel<WT, MT, WN, true>), grid, dim3(64 * WN), 0, stream, a);
        else
            hipLaunchKernelGGL((matmul_fp8_tile_kernel<WT, MT, WN, false>), grid, dim3(64 * WN), 0, stream, a);
    });
}

template <int WT>
hipError_t launch_wide(const MatmulFp8Args& all, int splits, hipStream_t stream) {
    const int units = (all.in_dim + 255) / 256;
    const int64_t most = std::min(matmul_fp8_converted_rows(units), launch_rows(units, kWideRows));
    return launch_tiles(all, splits, kWideRows, 32 * kWideWaves, most, stream, [&](MatmulFp8Args a, dim3 grid) {
        const int64_t tiles = ((int64_t)a.batch + kWideRows - 1) / kWideRows * (kWideRows / 32);
        a.sums = Unit<WT>::kMins ? a.xf + tiles * units * 16384 : nullptr;
        hipLaunchKernelGGL(matmul_fp8_convert_kernel, dim3((uint32_t)(tiles * units)), dim3(256), 0, stream, a.x, a.xf,
                           reinterpret_cast<_Float16*>(a.sums), a.in_dim, a.batch, units);
        if (wide_loads(a))
            hipLaunchKernelGGL((matmul_fp8_wide_kernel<WT, true>), grid, dim3(64 * kWideWaves), 0, stream, a);
        else
            hipLaunchKernelGGL((matmul_fp8_wide_kernel<WT, false>), grid, dim3(64 * kWideWaves), 0, stream, a);
    });
}

template <int WT>
hipError_t launch_type(const MatmulFp8Args& a, const MatmulFp8Plan& p, hipStream_t stream) {
    switch (p.form) {
        case MatmulFp8Plan::kWide: return launch_wide<WT>(a, p.splits, stream);
        case MatmulFp8Plan::kTile64: return launch_tile<WT, 4, 8>(a, p.splits, stream);
        case MatmulFp8Plan::kTile32: return launch_tile<WT, 2, 4>(a, p.splits, stream);
        case MatmulFp8Plan::kStream32: return p.waves == 8 ? launch_stream32<WT, 8>(a, stream) : launch_stream32<WT, 4>(a, stream);
        default: break;
    }
    // The stream form.  With many outputs two tiles share a workgroup's activations; with few, more waves share a tile's
    // K.  us, Q4_0: 4096 x 14336 at 1 row 9.6 with two tiles and 4 waves, 12.8 with one tile and 16; 3584 x 4608 6.3 and
    // 6.9; 18944 x 3584 at 1 row 10.7 with one tile and 16 waves, 15 with two tiles.
    const bool wide = a.out_dim > 4096;
    if (a.batch <= 4)
        return wide ? launch_form<WT, 1, 1, 2, 4>(a, stream) : launch_form<WT, 1, 1, 1, 16>(a, stream);
    if (a.batch <= 8)
        return wide ? launch_form<WT, 1, 2, 2, 8>(a, stream) : launch_form<WT, 1, 2, 1, 16>(a, stream);
    if (a.batch <= 16)
        return wide ? launch_form<WT, 1, 4, 2, 8>(a, stream) : launch_form<WT, 1, 4, 1, 8>(a, stream);
    // More rows: 32 a workgroup while its workgroups, one a CU, run in one round (18944 x 3584 at 32 rows 18.9 us with
    // one tile); else 16 a workgroup (3584 x 4608 at 37 rows 11.3, 13 with 32).
    const int64_t tiles_b = (a.batch + 31) / 32;
    if (a.out_dim >= 16384 && a.batch <= 32) return launch_form<WT, 2, 4, 2, 4>(a, stream);
    if ((a.out_dim + 15) / 16 * tiles_b <= p.cus) return launch_form<WT, 2, 4, 1, 8>(a, stream);
    if ((a.out_dim + 31) / 32 * tiles_b <= p.cus) return launch_form<WT, 2, 4, 2, 8>(a, stream);
    return launch_form<WT, 1, 4, 2, 8>(a, stream);
}

}  // namespace

int64_t matmul_fp8_row_bytes(int32_t w_type, int32_t in_dim) {
    return (int64_t)(in_dim / 64) * (w_type == GSP_WTYPE_Q4_1 ? 40 : 36);
}

hipError_t launch_matmul_fp8(int32_t w_type, const MatmulFp8Args& a, const MatmulFp8Plan& plan, hipStream_t stream) {
    if (w_type == GSP_WTYPE_Q4_0) return launch_type<GSP_WTYPE_Q4_0>(a, plan, stream);
    if (w_type == GSP_WTYPE_Q4_1) return launch_type<GSP_WTYPE_Q4_1>(a, plan, stream);
    return launch_type<GSP_WTYPE_Q4_K>(a, plan, stream);
}

}  // namespace gsp
