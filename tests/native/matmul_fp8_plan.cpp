// Prints, for every line "in_dim out_dim batch aligned cus" of the standard input, the form, the K ranges, the units
// of 256 of a range, the waves (32 x 32 stream) and the bytes of converted activations that gsp_matmul_batch_fp8 plans.
#include <cstdio>

#include "gsp_matmul_fp8_plan.h"

int main() {
    static const char* const kForms[] = {"stream", "wide", "tile64", "tile32", "stream32"};
    int in, out, batch, aligned, cus;
    while (std::scanf("%d %d %d %d %d", &in, &out, &batch, &aligned, &cus) == 5) {
        const gsp::MatmulFp8Plan p = gsp::plan_matmul_fp8(in, out, batch, aligned != 0, cus);
        const int units = in / 256 + (in % 256 != 0);
        std::printf("%s %d %d %d %lld\n", kForms[p.form], p.splits, (units + p.splits - 1) / p.splits, p.waves,
                    (long long)gsp::matmul_fp8_x_bytes(in, batch, p));
    }
    return 0;
}
