// A 4-bit microscaled matrix in device memory, shared by its quantisation and its product.
#pragma once

#include "tftq_tile.h"

constexpr int64_t MX_MOST = (1ll << 31) - 1024;  // rows or columns

struct MxMatrix {
    uint8_t *panels;
    uint8_t *scales;
};

// The parts of a buffer of tftq_mx_bytes(rows, cols) bytes; two null pointers for none.
__attribute__((visibility("hidden"))) MxMatrix mx_matrix(void *buffer, int64_t rows, int64_t cols);
