#include "gsp_matmul_fp8_plan.h"

#include <cmath>

namespace gsp {

// Converted activations of 32 rows take 16 KB a unit and 1 KB of sums.  A call keeps at most 1 GB of them: more rows
// are multiplied piece by piece, each of many more workgroups than the chip holds.
constexpr int64_t kConverted = 16384 + 1024;
int64_t matmul_fp8_converted_rows(int units) {
    return kMatmulFp8MostConverted / (units * kConverted) / (kMatmulFp8WideRows / 32) * kMatmulFp8WideRows;
}

// Which form a product takes: the one whose modelled time is least.  A tile's
// workgroup takes a time per unit of K that depends on how many share its CU;
// workgroups run in rounds of what the chip holds; splits of K add the partial
// sums' traffic and a launch.
static MatmulFp8Plan least_time(int32_t in_dim, int32_t out_dim, int32_t batch, bool aligned, int cus) {
    MatmulFp8Plan best{};
    best.cus = cus;
    // Tile offsets are 32-bit; a longer K is streamed.  Up to 64 rows only wide outputs repay the conversion.
    if (in_dim > (1 << 24) || batch <= (out_dim >= 16384 ? 32 : 64)) return best;
    struct Form {
        int form, rows, cols;
        double us[4];   // a unit's time with one to four workgroups on a CU; 0: they do not fit
        double around;  // a round's time before and behind its units
    };
    // Measured on 3584 and 18944 of K, Q4_0, at 65 to 2048 rows.
    constexpr Form kForms[] = {{MatmulFp8Plan::kWide, kMatmulFp8WideRows, kMatmulFp8WideCols, {4.3, 0, 0, 0}, 10},
                               {MatmulFp8Plan::kTile64, 64, 128, {2.05, 3.7, 0, 0}, 4},
                               {MatmulFp8Plan::kTile32, 32, 64, {1.33, 1.75, 2.5, 3.25}, 4}};
    const int units = (in_dim + 255) / 256;
    double least = 0;
    if (batch <= 64 && aligned) {
        // The stream's 32 x 32 tiles, three a CU with Q4_0, whose times stand for all three types (registers leave two of
        // Q4_1's and Q4_K's: 3584 x 18944 at 64 rows 28.3, 31.2 and 29.5 us): 3584 x 18944 at 48 rows 27.7 us against 31.9 in tiles of 64, 4096 x 32768
        // 43.7 and 37.4, 1024 x 65536 33 and 20.
        const double tiles = (double)(((int64_t)out_dim + 31) / 32 * ((batch + 31) / 32));
        least = 7 + tiles / (3 * cus) * (1.2 + 0.86 * units);
    }
    for (const Form& f : kForms) {
        // K past 3.9 million: the activations of one workgroup's rows would not fit.
        if (f.form == MatmulFp8Plan::kWide && matmul_fp8_converted_rows(units) == 0) continue;
        if (batch <= f.rows / 2) continue;  // half of it empty: the next one takes less, and no workspace up to 64 rows
        const double tiles = (double)(((int64_t)batch + f.rows - 1) / f.rows) * (((int64_t)out_dim + f.cols - 1) / f.cols);
        int fit = 4;
        while (fit > 1 && f.us[fit - 1] == 0) --fit;
        for (int splits = 1; splits <= (batch > 64 ? 16 : 1) && splits * 2 <= std::max(2, units); ++splits) {
            if (splits > 1 && tiles * splits > (double)cus * fit) break;
            const int per = (units + splits - 1) / splits;
            if ((units + per - 1) / per != splits) continue;
            const double on_cu = std::ceil(tiles * splits / cus);
            const double full = std::floor(on_cu / fit);
            const int rest = (int)(on_cu - full * fit);
            double t = (full * f.us[fit - 1] + (rest ? f.us[rest - 1] : 0)) * per;
            t += f.around * (fit == 1 ? on_cu : 1);
            if (splits > 1) t += 3.5 + (double)batch * out_dim * 4 * 2 * splits / 4e6;
            if (least == 0 || t < least) {
                least = t;
                best.form = f.form;
                best.splits = splits;
            }
        }
    }
    return best;
}

MatmulFp8Plan plan_matmul_fp8(int32_t in_dim, int32_t out_dim, int32_t batch, bool aligned, int cus) {
    MatmulFp8Plan plan = least_time(in_dim, out_dim, batch, aligned, cus);
    if (plan.form != MatmulFp8Plan::kStream) return plan;
    // Streamed products of 17 to 64 rows, in 32 x 32 tiles where these fill more than half of the CUs: in one round with 8
    // waves each (3584 x 4608 at 32 rows Q4_0 8.2 against 9.3, Q4_K 8.4 and 10.4; 3584 x 3584, on 112 CUs, 8.2 and 7.5),
    // in several with 4, three a CU (Q4_1 and Q4_K two; Q4_0 4096 x 14336 at 32 rows 14.6 against 17.5, at 64 24.6 and 28.2), unless a second
    // round would be short and much of the last rows' tile is empty (3584 x 4608 at 37 rows 14.1 and 11.3, 3584 x 8192
    // 15.0 and 15.2).
    const int64_t tiles = ((int64_t)out_dim + 31) / 32 * ((batch + 31) / 32);
    if (batch > 16 && batch <= 64 && aligned && tiles > cus / 2) {
        plan.waves = tiles <= cus ? 8 : batch <= 32 || batch > 48 || tiles >= 2 * cus ? 4 : 0;
        if (plan.waves) plan.form = MatmulFp8Plan::kStream32;
    }
    return plan;
}

int64_t matmul_fp8_x_bytes(int32_t in_dim, int32_t batch, const MatmulFp8Plan& plan) {
    if (plan.form != MatmulFp8Plan::kWide) return 0;
    const int units = (in_dim + 255) / 256;
    const int64_t rows = std::min<int64_t>(batch, matmul_fp8_converted_rows(units));
    return (rows + kMatmulFp8WideRows - 1) / kMatmulFp8WideRows * (kMatmulFp8WideRows / 32) * units * kConverted;
}

}  // namespace gsp
