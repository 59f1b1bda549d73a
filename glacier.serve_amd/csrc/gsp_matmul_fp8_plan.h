// Which kernel a projection of 8-bit activations takes (gsp_matmul_fp8.hip),
// without HIP: from its sizes, its weights' alignment and the CU count alone.
#pragma once

#include <algorithm>
#include <cstdint>

namespace gsp {

// A workgroup of the wide tile form.
constexpr int kMatmulFp8WideRows = 128, kMatmulFp8WideCols = 256;

// The kernel that a product takes, and the ranges of K that share an output (several only with a tile form).
struct MatmulFp8Plan {
    enum { kStream = 0, kWide, kTile64, kTile32, kStream32 };
    int32_t form = kStream;
    int32_t splits = 1;
    int32_t waves = 0;  // kStream32: of a workgroup
    int32_t cus = 1;
};

// aligned: rows of weights are whole units of 256, 16-byte aligned.
MatmulFp8Plan plan_matmul_fp8(int32_t in_dim, int32_t out_dim, int32_t batch, bool aligned, int cus);

// Workspace of the wide tile form, its converted activations: the most that a call keeps, the rows that a piece of the
// batch holds (0: K too long for the form), and the bytes of a product.
constexpr int64_t kMatmulFp8MostConverted = 1 << 30;
int64_t matmul_fp8_converted_rows(int units);
int64_t matmul_fp8_x_bytes(int32_t in_dim, int32_t batch, const MatmulFp8Plan& plan);

}  // namespace gsp
