// Launchers of products with 4-bit weights (q4_matmul.cu). All asynchronous on the context's stream.
#pragma once

#include <cstddef>
#include <cstdint>

#include "../internal.hpp"

namespace csdr {

// How a weight lies on the device: units of sixteen rows and kCols columns, a row tile's units one behind the
// other. A unit: codes, for each pair of 32-column groups and each lane (g = lane / 4, t = lane % 4) the words
// (row g, group 0), (row g + 8, group 0), (row g, group 1), (row g + 8, group 1), columns 8 t + 0 .. 3 of the
// group in a word's low half, + 4 .. 7 in its high half (pack_codes, codes4.cuh); then for g < 8 the steps of rows g and g + 8:
//   q4_0   128 columns; fp16 steps [g][row g, row g + 8][4 groups]
//   q4_k   256 columns; 6-bit (step, minimum) as bytes [g][row][8 groups], then fp16 (d, dmin) [g][row]
// so that a lane finds what its matrix fragments take in 128-bit pieces and a row tile is read front to
// back. Rows and columns behind the matrix hold zero steps.
struct Q4View {
    const uint8_t* base;
    uint32_t rows, cols, n_units;   // units of a row tile
    int format;                     // 0: q4_0, 1: q4_k
};
constexpr uint32_t q4_unit_cols(int format) { return format ? 256u : 128u; }
constexpr uint32_t q4_unit_bytes(int format) { return format ? 2048u + 256u + 64u : 1024u + 128u; }

void launch_q4_relay(csdr_context* ctx, const uint8_t* payload, const Q4View& w, uint8_t* out);

struct Q4Args {
    const void* x;
    int x_dtype;
    size_t x_token, x_col;          // elements between tokens and between columns
    size_t batch;
    float* y;
    size_t y_token, y_row;
    const float* bias;
};
void launch_q4_matmul(csdr_context* ctx, const Q4View& w, const Q4Args& a);

}  // namespace csdr

struct csdr_q4_weight {
    csdr_context* ctx = nullptr;
    csdr::Q4View view{};
    csdr::DevPtr data;
};
