// The projection of multilora.h on the tensor cores (csrc/multilora_tc.cu).
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

#include "philox.cuh"

namespace bsml {

// What the wide product needs to know of 16 rows, made with their numbers.
constexpr int kPartSlots = 3;
struct alignas(32) RowGroup {
    int slot[kPartSlots];        // the adapter of each slot (LowParts), -1 for none
    uint32_t rows;               // bit j: row j is read and written (id >= -1); bit 16 + j: it is padding
    uint32_t many;               // rows of later runs than there are slots
    uint32_t without;            // live rows without an adapter
    uint32_t pad[2];
};

// The rank numbers of every row between the two low-rank products: `t` as they are, and
// `parts` as the 16-bit operand of the tensor cores (LowParts below).
struct LowRank {
    float* t = nullptr;              // (rows, rank)
    void* parts = nullptr;           // (rows, kPartSlots * cols of low_parts(rank, dtype)), 16-bit
    RowGroup* groups = nullptr;      // (rows / 32 rounded up, 2)
    // (rows), fp16 only: the parts are the row's numbers over the power of two of this biased exponent
    uint8_t* power = nullptr;
};

// Layout of LowRank::parts. A row has kPartSlots pieces of `cols` columns; its numbers are in the
// piece of its slot, the other pieces are zero. The slot is the ordinal of the row's run (rows
// in a row with one adapter) among the runs that begin in, or reach into, its 32 rows (32 i ..
// 32 i + 31); the parts of a row of a later run than kPartSlots are not used. In a piece: number r
// of part i in column i * pitch + r, zero up to the pitch; the parts sum to the number. bf16
// and fp32 hold three bf16 parts (24 bits), fp16 two of its own (22). fp16's are of the row's numbers over
// a power of two that brings the largest to 2^14 .. 2^15: as they are, a number beyond 65504 would have no
// parts, and one below 1/8 (gradients are below 1e-4) fewer than 22 bits.
struct LowParts {
    int n = 0, pitch = 0, cols = 0;
};
LowParts low_parts(int rank, int dtype);

// out[m][f] = sum_k z[m][k] W(f, k) + bias[f] + keep(m, f) * sum_r t[m][r] Q_a(f, r), a = ids[m],
// with W(f, k) at W[f * width + k] and Q_a(f, r) at Q[(a * feats + f) * rank + r], or
// transposed: W[k * feats + f] and Q[(a * rank + r) * feats + f].
struct ProjectTc {
    int dtype = 0;
    bool transposed = false;
    int rows = 0, width = 0, feats = 0, rank = 0, adapters = 0;
    const void* z = nullptr;
    int64_t ldz = 0;
    const void *W = nullptr, *Q = nullptr, *bias = nullptr;
    // the thin operand of the product that makes `low`, where that reads the tensor cores'
    // layout (nullptr where it does not): (adapters, rank, width), transposed (adapters, width, rank)
    const void* P = nullptr;
    LowRank low;
    const int* ids = nullptr;
    DropProb drop;
    const uint64_t* rng = nullptr;
    bool zero_padding = false;
    void* out = nullptr;
    int64_t ldo = 0;
};

// Scratch of one call (operands laid out for the tensor cores), in bytes; 0 where every
// operand is read where it stands.
int64_t project_tc_scratch(const ProjectTc& p);
// Lays the operands out (one launch, none where they can be read where they stand) and
// says where z and P are: 16-bit rows on 16-byte boundaries, fp32 as three bf16 planes.
struct LaidOut {
    const void *z = nullptr, *P = nullptr;
    int64_t ldz = 0, ldp = 0, z_plane = 0, p_plane = 0;
};
LaidOut project_tc_prepare(const ProjectTc& p, void* scratch, cudaStream_t st);
// The product itself; the kernel before it on the stream is the one that made p.low, which
// called launch_dependents().
void project_tc(const ProjectTc& p, void* scratch, cudaStream_t st);

// Reads and clears the error word of this file's bounded waits.
int multilora_error_flag();
// A wait that runs out, on a barrier that nothing completes.
void multilora_wait_selftest(cudaStream_t st);

}  // namespace bsml
