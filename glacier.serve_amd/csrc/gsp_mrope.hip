// Rotary positions of several axes with the packed step's K/V write
// (gsp_mrope_write_step, gfx950).  Bound by memory: Q is read and written once,
// K and V read once and written into their slots.  The angles' rates come with
// the launch's arguments (made on the host, 64 powers in fp64 that would else
// cost every workgroup a third of its time), so that no table has to be on the device.
// Sixteen prompts, 7700 tokens of 28 + 4 heads of 128, take 58.6 us with other buffers
// than the call before, 4.8 TB/s as a large copy, and 51 where part of them is still in
// the last-level cache; a decode step of 64 rows is bound by the launch.
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
// VEC of VEC values.  Workgroup (token, y) takes items [256 I y, 256 I (y + 1)),
// I a thread, whose loads are issued before the angle table is built.  VEC 4
// needs head_dim and rope_dim in eights, v_head_dim and strides in fours and
// 16-byte aligned buffers; VEC 1 takes everything.
template <typename KT, int VEC, int I>
__global__ __launch_bounds__(256) void mrope_write_kernel(MropeWriteArgs a) {
    __shared__ float cs[kRopeMaxHalf][2];
    const int64_t i = blockIdx.x;
    const int d = a.head_dim, dv = a.v_head_dim;
    const int half = a.rope_dim >> 1;
    const int rot_items = half / VEC, per_head = d / (2 * VEC), per_v = dv / VEC;
    const int nq = a.n_heads * per_head, nk = a.n_kv * per_head, nv = a.n_kv * per_v;

    struct Item {
        int kind, h, m;  // 0 Q, 1 K, 2 V, 3 none
        Floats<VEC> x0, x1;
    } item[I];
    // The item's values lie side by side, or half a rotation apart.
    const auto near = [&](int m) { return a.style == GSP_ROPE_PAIRS || m >= rot_items; };
    const auto first = [&](int m) { return near(m) ? 2 * VEC * m : VEC * m; };
    const auto second = [&](int m) { return near(m) ? 2 * VEC * m + VEC : VEC * m + half; };
#pragma unroll
    for (int k = 0; k < I; ++k) {
        Item& it = item[k];
        const int t = (blockIdx.y * I + k) * 256 + threadIdx.x;
        it.kind = t < nq ? 0 : t < nq + nk ? 1 : t < nq + nk + nv ? 2 : 3;
        const int at = it.kind == 0 ? t : it.kind == 1 ? t - nq : t - nq - nk;
        const int per = it.kind == 2 ? per_v : per_head;
        it.h = at / per;
        it.m = at - it.h * per;
        if (it.kind < 2) {
            const float* src = it.kind == 0 ? a.q + i * a.q_stride + it.h * d : a.k + i * a.k_stride + it.h * d;
            it.x0 = load_floats<VEC>(src + first(it.m));
            it.x1 = load_floats<VEC>(src + second(it.m));
        } else if (it.kind == 2) {
            it.x0 = load_floats<VEC>(a.v + i * a.v_stride + it.h * dv + VEC * it.m);
        }
    }
    const int64_t blk = a.block_ids[i];
    const int64_t slot = a.slots[i];
    for (int j = threadIdx.x; j < half; j += 256)
        rope_angle((double)a.positions[(int64_t)axis_of_pair(a, j) * a.n + i], a.rates[j], a.mscale, &cs[j][0], &cs[j][1]);
    __syncthreads();

#pragma unroll
    for (int k = 0; k < I; ++k) {
        Item& it = item[k];
        if (it.kind == 3 || (it.kind != 0 && blk < 0)) continue;
        if (it.kind == 2) {
            store_floats<VEC>(static_cast<KT*>(a.v_pool) + blk * a.v_block_stride + a.v_layer_offset +
                                  (int64_t)it.h * a.v_head_stride + slot * dv + VEC * it.m,
                              it.x0);
            continue;
        }
        if (it.m < rot_items) {
            const Floats<VEC> y0 = it.x0, y1 = it.x1;
            const float* c = cs[VEC * it.m];
#pragma unroll
            for (int p = 0; p < VEC; ++p) {
                if (!near(it.m)) {
                    rope_turn(y0.v[p], y1.v[p], c[2 * p], c[2 * p + 1], &it.x0.v[p], &it.x1.v[p]);
                } else if constexpr (VEC == 1) {
                    rope_turn(y0.v[0], y1.v[0], c[0], c[1], &it.x0.v[0], &it.x1.v[0]);
                } else {  // pair p is values 2p and 2p + 1 of the item
                    const Floats<VEC>& y = p < VEC / 2 ? y0 : y1;
                    Floats<VEC>& x = p < VEC / 2 ? it.x0 : it.x1;
                    rope_turn(y.v[2 * p % VEC], y.v[2 * p % VEC + 1], c[2 * p], c[2 * p + 1], &x.v[2 * p % VEC],
                              &x.v[2 * p % VEC + 1]);
                }
            }
        }
        if (it.kind == 0) {
            float* q = a.q_out + (i * a.n_heads + it.h) * d;
            store_floats<VEC>(q + first(it.m), it.x0);
            store_floats<VEC>(q + second(it.m), it.x1);
        } else {
            KT* kd = static_cast<KT*>(a.k_pool) + blk * a.block_stride + a.layer_offset + (int64_t)it.h * a.head_stride +
                     slot * d;
            store_floats<VEC>(kd + first(it.m), it.x0);
            store_floats<VEC>(kd + second(it.m), it.x1);
        }
    }
}

template <typename KT, int VEC>
void launch_form(const MropeWriteArgs& a, hipStream_t stream) {
    const int items = (a.n_heads + a.n_kv) * (a.head_dim / (2 * VEC)) + a.n_kv * (a.v_head_dim / VEC);
    // One item a thread spreads a decode tick over more workgroups; with many tokens three let a workgroup share its
    // angles among more loads (7966 tokens of 28/4 heads, d 128, fp32 pages: 57.6 us with one, 53.9 with three, launches
    // of two streams overlapping).
    constexpr int kMany = 3;
    if (a.n < 512)
        hipLaunchKernelGGL((mrope_write_kernel<KT, VEC, 1>), dim3(a.n, (items + 255) / 256), dim3(256), 0, stream, a);
    else
        hipLaunchKernelGGL((mrope_write_kernel<KT, VEC, kMany>), dim3(a.n, (items + 256 * kMany - 1) / (256 * kMany)),
                           dim3(256), 0, stream, a);
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
