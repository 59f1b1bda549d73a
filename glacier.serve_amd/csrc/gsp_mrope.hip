// Rotary positions of several axes with the packed step's K/V write
// (gsp_mrope_write_step, gfx950).
#include "gsp_internal.h"
#include "gsp_rope.h"
#include "../../include/glacier_paged.h"

namespace gsp {
namespace {

// The axis whose position turns pair j.
__device__ inline int axis_of_pair(const MropeWriteArgs& a, int j) {
    if (a.interleaved) {
        const int m = j % a.n_axes;
        return j < a.n_axes * a.sections[m] ? m : 0;
    }
    int axis = 0, end = a.sections[0];
    while (axis + 1 < a.n_axes && j >= end) end += a.sections[++axis];
    return axis;
}

template <int VEC>
struct Floats {
    float v[VEC];
};

template <int VEC>
__device__ inline Floats<VEC> load_floats(const float* p) {
    Floats<VEC> r;
    if constexpr (VEC == 4) {
        const float4 f = *reinterpret_cast<const float4*>(p);
        r.v[0] = f.x, r.v[1] = f.y, r.v[2] = f.z, r.v[3] = f.w;
    } else {
        r.v[0] = *p;
    }
    return r;
}
template <int VEC, typename KT>
__device__ inline void store_floats(KT* p, const Floats<VEC>& r) {
    if constexpr (VEC == 4)
        store4(p, make_float4(r.v[0], r.v[1], r.v[2], r.v[3]));
    else
        *p = static_cast<KT>(r.v[0]);
}

// A token's work is a list of items of 2 VEC values: per Q head and per K head
// head_dim / (2 VEC), the first rope_dim / (2 VEC) of VEC rotation pairs and the
// rest of dims past rope_dim, which pass through; then per V head v_head_dim /
// VEC of VEC values.  Workgroup (token, y) takes items [256 y, 256 y + 256), one
// a thread, whose loads are issued before the angle table is built.  VEC 4
// needs head_dim and rope_dim in eights, v_head_dim and strides in fours and
// 16-byte aligned buffers; VEC 1 takes everything.
template <typename KT, int VEC>
__global__ __launch_bounds__(256) void mrope_write_kernel(MropeWriteArgs a) {
    __shared__ float cs[kRopeMaxHalf][2];
    const int64_t i = blockIdx.x;
    const int d = a.head_dim, dv = a.v_head_dim;
    const int half = a.rope_dim >> 1;
    const int rot_items = half / VEC, per_head = d / (2 * VEC), per_v = dv / VEC;
    const int nq = a.n_heads * per_head, nk = a.n_kv * per_head, nv = a.n_kv * per_v;
    const int t = blockIdx.y * 256 + threadIdx.x;

    int kind = 3, h = 0, m = 0;  // 0 Q, 1 K, 2 V, 3 none
    if (t < nq) {
        kind = 0;
        h = t / per_head;
        m = t - h * per_head;
    } else if (t < nq + nk) {
        kind = 1;
        h = (t - nq) / per_head;
        m = (t - nq) - h * per_head;
    } else if (t < nq + nk + nv) {
        kind = 2;
        h = (t - nq - nk) / per_v;
        m = (t - nq - nk) - h * per_v;
    }
    const bool turn = m < rot_items;
    const bool near = a.style == GSP_ROPE_PAIRS || !turn;  // the item's values lie side by side
    const int e0 = near ? 2 * VEC * m : VEC * m;
    const int e1 = near ? e0 + VEC : e0 + half;
    Floats<VEC> x0{}, x1{};
    if (kind < 2) {
        const float* src = kind == 0 ? a.q + i * a.q_stride + h * d : a.k + i * a.k_stride + h * d;
        x0 = load_floats<VEC>(src + e0);
        x1 = load_floats<VEC>(src + e1);
    } else if (kind == 2) {
        x0 = load_floats<VEC>(a.v + i * a.v_stride + h * dv + VEC * m);
    }
    const int64_t blk = a.block_ids[i];
    const int64_t slot = a.slots[i];
    for (int j = threadIdx.x; j < half; j += 256)
        rope_angle(a, (double)a.positions[(int64_t)axis_of_pair(a, j) * a.n + i], j, &cs[j][0], &cs[j][1]);
    __syncthreads();

    if (kind == 3 || (kind != 0 && blk < 0)) return;
    if (kind == 2) {
        store_floats<VEC>(static_cast<KT*>(a.v_pool) + blk * a.v_block_stride + a.v_layer_offset +
                              (int64_t)h * a.v_head_stride + slot * dv + VEC * m,
                          x0);
        return;
    }
    if (turn) {
        const Floats<VEC> y0 = x0, y1 = x1;
#pragma unroll
        for (int p = 0; p < VEC; ++p) {
            const float c = cs[VEC * m + p][0], s = cs[VEC * m + p][1];
            if (near) {  // pair p is values 2p and 2p + 1 of the item
                const float u = VEC == 1 ? y0.v[0] : p < VEC / 2 ? y0.v[2 * p % VEC] : y1.v[2 * p % VEC];
                const float w = VEC == 1 ? y1.v[0] : p < VEC / 2 ? y0.v[(2 * p + 1) % VEC] : y1.v[(2 * p + 1) % VEC];
                float u2, w2;
                rope_turn(u, w, c, s, &u2, &w2);
                if constexpr (VEC == 1) {
                    x0.v[0] = u2, x1.v[0] = w2;
                } else {
                    (p < VEC / 2 ? x0 : x1).v[2 * p % VEC] = u2;
                    (p < VEC / 2 ? x0 : x1).v[(2 * p + 1) % VEC] = w2;
                }
            } else {
                rope_turn(y0.v[p], y1.v[p], c, s, &x0.v[p], &x1.v[p]);
            }
        }
    }
    if (kind == 0) {
        float* q = a.q_out + (i * a.n_heads + h) * d;
        store_floats<VEC>(q + e0, x0);
        store_floats<VEC>(q + e1, x1);
    } else {
        KT* kd = static_cast<KT*>(a.k_pool) + blk * a.block_stride + a.layer_offset + (int64_t)h * a.head_stride +
                 slot * d;
        store_floats<VEC>(kd + e0, x0);
        store_floats<VEC>(kd + e1, x1);
    }
}

template <typename KT, int VEC>
void launch_form(const MropeWriteArgs& a, hipStream_t stream) {
    const int items = (a.n_heads + a.n_kv) * (a.head_dim / (2 * VEC)) + a.n_kv * (a.v_head_dim / VEC);
    hipLaunchKernelGGL((mrope_write_kernel<KT, VEC>), dim3(a.n, (items + 255) / 256), dim3(256), 0, stream, a);
}

}  // namespace

hipError_t launch_mrope_write(int kv_f16, const MropeWriteArgs& a, hipStream_t stream) {
    if (a.n <= 0) return hipSuccess;
    const auto al16 = [](const void* p) { return ((uintptr_t)p & 15) == 0; };
    const bool vec = a.head_dim % 8 == 0 && a.rope_dim % 8 == 0 && a.v_head_dim % 4 == 0 && a.q_stride % 4 == 0 &&
                     a.k_stride % 4 == 0 && a.v_stride % 4 == 0 && al16(a.q) && al16(a.q_out) && al16(a.k) &&
                     al16(a.v) && al16(a.k_pool) && al16(a.v_pool);
    if (vec && kv_f16)
        launch_form<_Float16, 4>(a, stream);
    else if (vec)
        launch_form<float, 4>(a, stream);
    else if (kv_f16)
        launch_form<_Float16, 1>(a, stream);
    else
        launch_form<float, 1>(a, stream);
    return hipGetLastError();
}

}  // namespace gsp
