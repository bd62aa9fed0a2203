// Where the tensor cores' kernels read an operand of the projection of many requests: where it
// stands, or laid out anew in a call's scratch. Plain C++, checked without a GPU.
#pragma once

#include <cstdint>

namespace bsml {

// planes x rows x cols of 16-bit numbers, rows `ld` numbers apart
struct Operand {
    const void* p = nullptr;
    int64_t ld = 0, rows = 0, planes = 1;
    int cols = 0;
    bool moved = false;       // laid out in scratch
    int64_t bytes = 0;        // of scratch
};

// f32: three bf16 planes; 16-bit numbers are read where they stand if their rows are on 16-byte
// boundaries. A single row may then be read a TMA box or a guarded vector at a time, but no
// further than its end: with `whole` (the operand is read in pieces of up to 8 numbers without a
// guard) it has to be whole pieces long.
inline Operand operand(const void* p, int64_t ld, int64_t rows, int cols, bool f32, bool whole) {
    const int64_t padded = ((int64_t)cols + 7) / 8 * 8;
    Operand o;
    o.p = p;
    o.rows = rows;
    o.cols = cols;
    o.ld = rows > 1 ? ld : padded;
    o.moved = f32 || (reinterpret_cast<uintptr_t>(p) & 15) != 0 || o.ld % 8 != 0 ||
              (whole && rows == 1 && padded != cols);
    if (o.moved) {
        o.ld = padded;
        o.planes = f32 ? 3 : 1;
        o.bytes = (o.planes * o.rows * o.ld * 2 + 255) / 256 * 256;
    }
    return o;
}

}  // namespace bsml
