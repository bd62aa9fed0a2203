// One shared projection and each row's own low-rank adapter (see multilora.h):
//   h[m] = s_a / (1 - p) A_a (keep * x[m])            (rank numbers a row, fp32)
//   y[m] = W x[m] + bias + B_a h[m]
// and the backward
//   g[m] = s_a / (1 - p) B_a^T dy[m]
//   dx[m] = W^T dy[m] + keep * (A_a^T g[m])
//   dA_a = sum_{m of a} g[m] (keep * x[m])^T,  dB_a = sum_{m of a} dy[m] h[m]^T
// This file has the thin products (h, g, dA, dB) and the order of a call; the wide ones are
// csrc/multilora_tc.cu.
#include "multilora.h"

#include <algorithm>
#include <mutex>
#include <type_traits>

#include "common.cuh"
#include "multilora_tc.h"
#include "philox.cuh"
#include "scalar.cuh"
#include "tc_ptx.cuh"

namespace bsml {

namespace {

constexpr int kThreads = 256;
constexpr int kMaxRank = 128;

// ── h and g: rows times an adapter's thin matrix
// A number as the parts of LowParts: three bf16 numbers, or two fp16 ones. Each part is the rounded
// remainder of those before it, a number that is not finite has no remainder. bf16's three hold an fp32
// number whole (below 2^-110 less); fp16's two, of `v` over its row's power of two, 22 bits or steps of
// 2^-39 of the row's largest number: a third would add 2^-23 of it, where h itself is off by more after its
// sum, and an output by 2^-11.
template <class T>
__device__ __forceinline__ void put_parts(uint16_t* row, const LowParts& lp, int r, float v) {
    if constexpr (!std::is_same<T, __half>::value) {
        for (int i = 0; i < lp.n; ++i) {
            __nv_bfloat16 b = __float2bfloat16_rn(v);
            if (isinf(__bfloat162float(b)) && isfinite(v)) b = __float2bfloat16_rz(v);
            row[i * lp.pitch + r] = __bfloat16_as_ushort(b);
            v = isfinite(v) ? v - __bfloat162float(b) : 0.f;
        }
    } else {
        const __half hi = __float2half_rn(v);
        row[r] = __half_as_ushort(hi);
        row[lp.pitch + r] = __half_as_ushort(__float2half_rn(isfinite(v) ? v - __half2float(hi) : 0.f));
    }
}
// The biased exponent of the power of two over which the numbers of an fp16 row are held, `most` being the largest
// finite magnitude of them, and the factor that brings them there (most: to 2^14 .. 2^15, numbers
// below 2^-112 no further than times 2^126).
__device__ __forceinline__ int row_power(float most) { return max((int)(__float_as_uint(most) >> 23) - 14, 1); }
__device__ __forceinline__ float row_factor(int power) { return __uint_as_float((uint32_t)(254 - power) << 23); }
__device__ __forceinline__ float finite_size(float v) { return isfinite(v) ? fabsf(v) : 0.f; }
__device__ __forceinline__ float warp_max(float v) {   // of numbers >= 0
    return __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(v)));
}

struct ShrinkArgs {
    const void* z;            // (rows, width), the type's own numbers
    int64_t ldz;
    const void* P;            // adapters x rank x width (row stride ldp), or adapters x width x rank
    int64_t ldp;
    const void *zt, *Pt;      // the operands of the tensor cores: the same, or bf16 planes of fp32
    int64_t ldzt, ldpt, zt_plane, pt_plane;
    int z_vec, p_vec;         // 16-byte rows of z and P
    const float* scale;
    const int* ids;
    int rows, width, rank, adapters;
    int block;                // ranks a CTA (shrink_rows_kernel): a multiple of 8
    int splits;               // CTAs a tile (shrink_tile_kernel), a cluster
    DropProb drop;
    const uint64_t* rng;
    LowRank low;
    LowParts lp;
};

// The slots of 32 rows (LowParts), by a whole warp: lane l has row l's adapter `ad`, -1 for none.
__device__ __forceinline__ int row_slot(int ad, int lane) {
    const int before = __shfl_up_sync(0xffffffffu, ad, 1);
    const uint32_t starts = __ballot_sync(0xffffffffu, ad >= 0 && (lane == 0 || before != ad));
    return __popc(starts & ((2u << lane) - 1)) - 1;
}
// 32 rows from m0 (lane l: row l): the adapter of each, -1 for none, and its slot. Whole warp.
struct Rows32 {
    int ad, slot;
    bool live, pad;
};
__device__ __forceinline__ Rows32 rows32(const ShrinkArgs& a, int64_t m0, int lane) {
    const bool in = m0 + lane < a.rows;
    const int id = in ? a.ids[m0 + lane] : -1;
    Rows32 r;
    r.live = in && id >= -1;
    r.pad = in && id < -1;
    r.ad = id >= 0 && id < a.adapters ? id : -1;
    r.slot = row_slot(r.ad, lane);
    return r;
}
__device__ __forceinline__ void put_groups(const ShrinkArgs& a, int64_t m0, const Rows32& r, int lane) {
    const uint32_t all = 0xffffffffu, half = lane < 16 ? 0x0000FFFFu : 0xFFFF0000u;
    RowGroup g = {};
#pragma unroll
    for (int k = 0; k < kPartSlots; ++k) {
        const uint32_t in = __ballot_sync(all, r.ad >= 0 && r.slot == k) & half;
        const int ad = __shfl_sync(all, r.ad, in ? __ffs(in) - 1 : 0);
        g.slot[k] = in ? ad : -1;
    }
    const int at = lane & 16;
    g.rows = (__ballot_sync(all, r.live) >> at & 0xFFFFu) | __ballot_sync(all, r.pad) >> at << 16;
    g.many = __ballot_sync(all, r.ad >= 0 && r.slot >= kPartSlots) & half;
    g.without = __ballot_sync(all, r.live && r.ad < 0) & half;
    if ((lane & 15) == 0) a.low.groups[m0 / 16 + (lane >> 4)] = g;
}
__device__ __forceinline__ uint16_t* parts_row(const ShrinkArgs& a, int64_t m) {
    return (uint16_t*)a.low.parts + m * (kPartSlots * a.lp.cols);
}
// The numbers of a row without an adapter.
__device__ __forceinline__ void put_none(const ShrinkArgs& a, int64_t m, int tid, int n) {
    for (int r = tid; r < a.rank; r += n) a.low.t[m * a.rank + r] = 0.f;
    if (a.low.power && tid == 0) a.low.power[m] = 127;
}
// Zeros of a row without an adapter (slot < 0), or around the numbers of the parts in `slot`.
__device__ __forceinline__ void put_zeros(const ShrinkArgs& a, int64_t m, int slot, int tid, int n) {
    uint16_t* parts = parts_row(a, m);
    const int lo = slot < 0 ? 0 : slot * a.lp.cols, used = a.lp.n * a.lp.pitch;
    for (int c = tid; c < kPartSlots * a.lp.cols; c += n) {
        const int in = c - lo;
        if (slot < 0 || in < 0 || in >= used || in % a.lp.pitch >= a.rank) parts[c] = 0;
    }
    if (slot < 0) put_none(a, m, tid, n);
}

// 8 numbers of a row from column k as they lie in memory
template <class T>
struct Raw8 {
    uint4 q[sizeof(T) / 2];
    __device__ __forceinline__ void load(const T* p) {
#pragma unroll
        for (int i = 0; i < (int)(sizeof(T) / 2); ++i) q[i] = __ldg(reinterpret_cast<const uint4*>(p) + i);
    }
    // element by element, zero from `width` on
    __device__ __forceinline__ void load(const T* row, int k, int width) {
        T* e = reinterpret_cast<T*>(q);
#pragma unroll
        for (int j = 0; j < 8; ++j) e[j] = k + j < width ? row[k + j] : from_f<T>(0.f);
    }
    __device__ __forceinline__ float operator[](int j) const { return to_f(reinterpret_cast<const T*>(q)[j]); }
};

// One CTA a row and block of ranks, for few rows: h[r] = f sum_k z[k] P(r, k) on the CUDA
// cores. What counts is the time of one pass over the adapter, so loads go out in batches that
// nothing waits in between. Not transposed: a warp takes one rank or two at a time, its lanes
// 8 columns each. Transposed: a thread takes 8 ranks of every (256 / vectors a row)-th row of P.
// Bound by the latency of that pass and of the launch: one row of 4096 bf16 columns, 16 ranks, 4.5 us
// (5.7 cold), 64 rows 6.3.
template <class T, bool TR>
__global__ void __launch_bounds__(kThreads, 4) shrink_rows_kernel(const __grid_constant__ ShrinkArgs a) {
    tc::launch_dependents();
    __shared__ float sums[8][kMaxRank];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int64_t m = blockIdx.x;
    const int r0 = blockIdx.y * a.block, r1 = min(a.rank, r0 + a.block);
    // every warp works the row's slot out from the ids of its 32 rows
    const Rows32 r32 = rows32(a, m & ~31, lane);
    const int at = (int)(m & 31), ad = __shfl_sync(0xffffffffu, r32.ad, at);
    const int slot = __shfl_sync(0xffffffffu, r32.slot, at);
    if (at == 0 && blockIdx.y == 0 && warp == 0) put_groups(a, m, r32, lane);
    if (ad < 0) {
        if (blockIdx.y == 0) put_zeros(a, m, -1, tid, kThreads);
        return;
    }
    const T* z = (const T*)a.z + m * a.ldz;
    const float f = a.drop.scale * (a.scale ? a.scale[ad] : 1.f);
    if constexpr (!TR) {
        const RngKey key = a.drop.thr ? load_rng(a.rng) : RngKey{};
        const T* P = (const T*)a.P + (int64_t)ad * a.rank * a.ldp;
        const bool vec = a.z_vec && a.p_vec;
        auto sum = [&](int r, auto n) {
            constexpr int N = decltype(n)::value, U = (sizeof(T) == 4 ? 2 : 4) / N;
            const T* p[N];
            float s[N];
#pragma unroll
            for (int i = 0; i < N; ++i) {
                p[i] = P + (int64_t)(r + 8 * i) * a.ldp;
                s[i] = 0.f;
            }
            auto add = [&](const Raw8<T>& v, const Raw8<T>(&w)[N], int k) {
                const uint32_t keep = a.drop.thr ? keep_bits(k >> 3, (uint32_t)m, key, a.drop.thr) : 0xFFu;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float x = keep >> j & 1 ? v[j] : 0.f;
#pragma unroll
                    for (int i = 0; i < N; ++i) s[i] = fmaf(x, w[i][j], s[i]);
                }
            };
            int k = lane * 8;
            if (vec)
                for (; k + 256 * (U - 1) + 8 <= a.width; k += 256 * U) {
                    Raw8<T> v[U], w[U][N];
#pragma unroll
                    for (int u = 0; u < U; ++u) {
                        v[u].load(z + k + 256 * u);
#pragma unroll
                        for (int i = 0; i < N; ++i) w[u][i].load(p[i] + k + 256 * u);
                    }
#pragma unroll
                    for (int u = 0; u < U; ++u) add(v[u], w[u], k + 256 * u);
                }
            for (; k < a.width; k += 256) {
                Raw8<T> v, w[N];
                const bool whole = vec && k + 8 <= a.width;
                if (whole) v.load(z + k);
                else v.load(z, k, a.width);
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    if (whole) w[i].load(p[i] + k);
                    else w[i].load(p[i], k, a.width);
                }
                add(v, w, k);
            }
#pragma unroll
            for (int i = 0; i < N; ++i) {
                for (int o = 16; o > 0; o >>= 1) s[i] += __shfl_xor_sync(0xffffffffu, s[i], o);
                if (lane == 0) sums[0][r + 8 * i] = s[i];
            }
        };
        int r = r0 + warp;
        for (; r + 8 < r1; r += 16) sum(r, std::integral_constant<int, 2>{});
        if (r < r1) sum(r, std::integral_constant<int, 1>{});
        __syncthreads();
    } else {
        // vectors of 8 ranks, a power of two of them a row of threads
        constexpr int U = sizeof(T) == 4 ? 4 : 8;
        const int nv = (r1 - r0 + 7) / 8;
        int vp = 1;
        while (vp < nv) vp *= 2;
        const int v = tid % vp, rv = r0 + v * 8, step = kThreads / vp;
        const T* P = (const T*)a.P + (int64_t)ad * a.width * a.ldp;
        float s[8] = {};
        if (v < nv) {
            int k = tid / vp;
            if (a.p_vec)
                for (; k + (U - 1) * step < a.width; k += U * step) {
                    Raw8<T> w[U];
                    T x[U];
#pragma unroll
                    for (int u = 0; u < U; ++u) {
                        w[u].load(P + (int64_t)(k + u * step) * a.ldp + rv);
                        x[u] = z[k + u * step];
                    }
#pragma unroll
                    for (int u = 0; u < U; ++u)
#pragma unroll
                        for (int j = 0; j < 8; ++j) s[j] = fmaf(to_f(x[u]), w[u][j], s[j]);
                }
            for (; k < a.width; k += step) {
                Raw8<T> w;
                const T* p = P + (int64_t)k * a.ldp;
                if (a.p_vec) w.load(p + rv);
                else w.load(p, rv, a.rank);
                const float x = to_f(z[k]);
#pragma unroll
                for (int j = 0; j < 8; ++j) s[j] = fmaf(x, w[j], s[j]);
            }
        }
#pragma unroll
        for (int j = 0; j < 8; ++j)
            for (int o = 16; o >= vp; o >>= 1) s[j] += __shfl_xor_sync(0xffffffffu, s[j], o);
        if (lane < vp && v < nv)
#pragma unroll
            for (int j = 0; j < 8; ++j) sums[warp][rv + j] = s[j];
        __syncthreads();
        if (const int r = r0 + tid; r < r1) {
            float t = 0.f;
            for (int w = 0; w < 8; ++w) t += sums[w][r];
            sums[0][r] = t;
        }
    }
    const int r = r0 + tid;
    float h = r < r1 ? f * sums[0][r] : 0.f;
    if (r < r1) a.low.t[m * a.rank + r] = h;
    if constexpr (std::is_same<T, __half>::value) {
        // the row's largest number: of the first warp, or over the warps, and the cluster of the row's CTAs
        __shared__ float most[4];
        const int ctas = (int)gridDim.y;
        float all = warp < 4 ? warp_max(finite_size(h)) : 0.f;
        if (a.rank > 32 || ctas > 1) {
            if (warp < 4 && lane == 0) most[warp] = all;
            if (ctas > 1) tc::cluster_sync();
            else __syncthreads();
            all = fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3]));
            if (ctas > 1) {
                float v = 0.f;   // lane: warp (lane & 3) of CTA lane / 4
                if (lane < 4 * ctas) v = tc::ld_cluster(tc::map_shared(tc::smem_u32(&most[lane & 3]), lane >> 2));
                all = warp_max(v);
                tc::cluster_sync();   // no CTA ends before the others have read it
            }
        }
        const int power = row_power(all);
        h *= row_factor(power);
        if (blockIdx.y == 0 && tid == 0) a.low.power[m] = (uint8_t)power;
    }
    if (r < r1 && slot < kPartSlots) put_parts<T>(parts_row(a, m) + slot * a.lp.cols, a.lp, r, h);
    if (blockIdx.y == 0) put_zeros(a, m, slot, tid, kThreads);
}

// Copies from global to shared memory that nothing waits for until copy_async_wait.
// 16 bytes, of which the first `bytes` are read and the others zero
__device__ __forceinline__ void copy_async16(uint32_t to, const void* from, int bytes = 16) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copy_async4(uint32_t to, const void* from) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ void copy_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_async_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

template <bool F16>
__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&x)[4], uint32_t b0, uint32_t b1) {
    if constexpr (F16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(x[0]), "r"(x[1]), "r"(x[2]), "r"(x[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(x[0]), "r"(x[1]), "r"(x[2]), "r"(x[3]), "r"(b0), "r"(b1));
}

// 8x8 transpose of 16-bit numbers over a warp
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}

// 8 16-bit numbers of a row from column k; at the row's end (TAIL) zero from `width` on
template <bool TAIL>
__device__ __forceinline__ uint4 vec8(const uint16_t* row, int k, int width) {
    if constexpr (TAIL) {
        if (k + 8 > width) {
            uint16_t e[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) e[j] = k + j < width ? row[k + j] : (uint16_t)0;
            return make_uint4(e[0] | e[1] << 16, e[2] | e[3] << 16, e[4] | e[5] << 16, e[6] | e[7] << 16);
        }
    }
    return __ldg(reinterpret_cast<const uint4*>(row + k));
}
// Many rows: a CTA has MT * 16 of them and splits the contraction over its warps, 64 columns
// a turn. Each warp reads its part of z straight into MMA operands, 16 bytes a lane and load (a
// ring of asynchronous copies in shared memory was no faster): an MMA sums over its 16 columns in
// any order, so lane t of a row takes columns 8t .. 8t+7 of 32 as the operand's slots (2t, 2t+1,
// 2t+8, 2t+9) of two MMAs, and P's operand uses the same order. P transposed is read in pairs of
// ranks and turned by movmatrix. PL planes of fp32 (z, P) give the products of significance 2^-16
// and above. A tile whose rows have several adapters takes a pass for each (z is then in L1 or
// L2). NT: blocks of 8 ranks, up to 64 ranks a pass.
// What bounds it is the chain of a tile, 1.2 us a turn of 512 columns (dropped 3, the generator's
// instructions; 64 ranks 2.5, transposed 6), not the reading of z: bf16, 16 ranks, 8192 rows x 4096
// columns 26 us (2.6 TB/s), dropped 44, transposed 29.
constexpr int kMaxSplits = 8;
template <class T, bool TR, int NT>
__global__ void __launch_bounds__(kThreads) shrink_tile_kernel(const __grid_constant__ ShrinkArgs a) {
    tc::launch_dependents();
    constexpr int PL = sizeof(T) == 4 ? 3 : 1, MT = PL == 1 ? 2 : 1, TM = MT * 16;
    constexpr bool F16 = std::is_same<T, __half>::value;
    constexpr int RP = NT * 8 + 4;   // row of the partial sums, padded against bank conflicts
    __shared__ float sums[4][TM][RP];
    __shared__ int sid[TM], sslot[TM];   // adapter (-1 for none) and slot of each row
    __shared__ int sad[TM], n_ad;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    // With few tiles, a cluster shares one: each CTA sums over its part of the columns, and writes
    // the numbers of every splits-th row.
    const int splits = a.splits, split = (int)blockIdx.x % splits;
    const int64_t m0 = (int64_t)(blockIdx.x / splits) * TM;
    if (warp == 0) {
        // the ids of the tile's 32 rows (of its half of them, with 16 rows a tile)
        const int64_t m32 = m0 & ~(int64_t)31;
        const Rows32 r32 = rows32(a, m32, lane);
        const int mine = r32.ad, row = lane - (int)(m0 - m32);
        const bool in = row >= 0 && row < TM;
        if (in) {
            sid[row] = mine;
            sslot[row] = r32.slot;
        }
        if (m0 == m32 && split == 0) put_groups(a, m32, r32, lane);
        // the tile's adapters, each where its first row stands
        const int id = in ? mine : -1;
        const uint32_t same = __match_any_sync(0xffffffffu, id);   // by every lane, whatever its row
        const bool first = id >= 0 && __ffs(same) - 1 == lane;
        const uint32_t firsts = __ballot_sync(0xffffffffu, first);
        if (first) sad[__popc(firsts & ((1u << lane) - 1))] = id;
        if (lane == 0) n_ad = __popc(firsts);
    }
    __syncthreads();
    const RngKey key = a.drop.thr ? load_rng(a.rng) : RngKey{};
    // the parts' columns beside the numbers (all of them: the numbers follow), and rows without
    for (int i = warp; i < TM; i += 8) {
        if (m0 + i >= a.rows) break;
        if (i % splits != split) continue;
        uint4* parts = reinterpret_cast<uint4*>(parts_row(a, m0 + i));
        for (int c = lane; c < kPartSlots * a.lp.cols / 8; c += 32) parts[c] = make_uint4(0, 0, 0, 0);
        if (sid[i] < 0) put_none(a, m0 + i, lane, 32);
    }

    for (int pass = 0; pass < n_ad; ++pass) {
        const int ad = sad[pass];
        const float f = a.drop.scale * (a.scale ? a.scale[ad] : 1.f);
        for (int rb = 0; rb < a.rank; rb += NT * 8) {
            float acc[MT][NT][4] = {}, sum[MT][NT][4] = {};
            // Lane pointers at this warp's first chunk of 64 columns; a turn advances them by 512
            // (a CTA).
            // (Rows of other adapters, or the last row again past the end, are read and their
            // sums dropped: no load waits for a test.)
            const int first = split * 8 + warp, turn = splits * 512;
            const uint16_t* zp[MT][2];
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int u = 0; u < 2; ++u)
                    zp[i][u] = (const uint16_t*)a.zt + min(m0 + i * 16 + u * 8 + g, (int64_t)a.rows - 1) * a.ldzt +
                               first * 64 + t * 8;
            const uint16_t* P = (const uint16_t*)a.Pt + (int64_t)ad * (TR ? a.width : a.rank) * a.ldpt;
            const int ldp = (int)a.ldpt;
            // transposed: matrix row g of block s is contraction slot g: column 8 * (g / 2) + 2s + (g & 1)
            const uint16_t* pp = TR ? P + (int64_t)(first * 64 + (g >> 1) * 8 + (g & 1)) * ldp : P + first * 64 + t * 8;
            int po[NT];   // of rank block n
#pragma unroll
            for (int n = 0; n < NT; ++n)
                po[n] = TR ? min(rb + n * 8 + t * 2, ldp - 2) : min(rb + n * 8 + g, a.rank - 1) * ldp;
            // 32 columns from column k0 (of the row) at `at` (from the lane pointers)
            auto step = [&](int k0, int at, auto tail) {
                constexpr bool TAIL = decltype(tail)::value;
                const int k = k0 + t * 8, room = a.width - k;   // columns left for this lane
                uint4 x[PL][MT][2], b[PL][NT];
#pragma unroll
                for (int q = 0; q < PL; ++q)
#pragma unroll
                    for (int i = 0; i < MT; ++i)
#pragma unroll
                        for (int u = 0; u < 2; ++u) x[q][i][u] = vec8<TAIL>(zp[i][u] + q * a.zt_plane + at, 0, room);
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int q = 0; q < PL; ++q) {
                        const uint16_t* e = pp + q * a.pt_plane + po[n];
                        if constexpr (!TR) {
                            b[q][n] = vec8<TAIL>(e + at, 0, room);
                        } else {
                            uint32_t w[4];
#pragma unroll
                            for (int s = 0; s < 4; ++s)
                                w[s] = !TAIL || k0 + (g >> 1) * 8 + 2 * s + (g & 1) < a.width
                                           ? __ldg(reinterpret_cast<const uint32_t*>(e + (at + 2 * s) * ldp))
                                           : 0u;
                            b[q][n] = make_uint4(w[0], w[1], w[2], w[3]);
                        }
                    }
                if (a.drop.thr)
#pragma unroll
                    for (int i = 0; i < MT; ++i)
#pragma unroll
                        for (int u = 0; u < 2; ++u) {
                            const uint4 w = philox4x32_10(k >> 3, (uint32_t)(m0 + i * 16 + u * 8 + g), key);
#pragma unroll
                            for (int q = 0; q < PL; ++q) x[q][i][u] = drop_group(x[q][i][u], w, a.drop.thr);
                        }
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    uint32_t c[PL][4];
#pragma unroll
                    for (int q = 0; q < PL; ++q) {
                        c[q][0] = b[q][n].x; c[q][1] = b[q][n].y; c[q][2] = b[q][n].z; c[q][3] = b[q][n].w;
                        if (TR)
#pragma unroll
                            for (int s = 0; s < 4; ++s) c[q][s] = transpose8(c[q][s]);
                    }
#pragma unroll
                    for (int i = 0; i < MT; ++i)
#pragma unroll
                        for (int qz = PL - 1; qz >= 0; --qz)
#pragma unroll
                            for (int qp = PL - 1 - qz; qp >= 0; --qp) {
                                const uint4 u0 = x[qz][i][0], u1 = x[qz][i][1];
                                const uint32_t f0[4] = {u0.x, u1.x, u0.y, u1.y}, f1[4] = {u0.z, u1.z, u0.w, u1.w};
                                mma_16816<F16>(acc[i][n], f0, c[qp][0], c[qp][1]);
                                mma_16816<F16>(acc[i][n], f1, c[qp][2], c[qp][3]);
                            }
                }
            };
            // The sums of kTurns turns, rounded to nearest. (An MMA truncates its sum, always towards zero.)
            auto gather = [&]() {
#pragma unroll
                for (int i = 0; i < MT; ++i)
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            sum[i][n][j] += acc[i][n][j];
                            acc[i][n][j] = 0.f;
                        }
            };
            constexpr int kTurns = PL == 1 ? 8 : 1;
            int k0 = first * 64, left = kTurns;
#pragma unroll 1
            for (; k0 + 64 <= a.width; k0 += turn) {
                if (left-- == 0) {
                    gather();
                    left = kTurns - 1;
                }
                step(k0, 0, std::false_type{});
                step(k0 + 32, 32, std::false_type{});
#pragma unroll
                for (int i = 0; i < MT; ++i)
#pragma unroll
                    for (int u = 0; u < 2; ++u) zp[i][u] += turn;
                pp += TR ? turn * (int64_t)ldp : turn;
            }
            // a last piece of fewer than 64 columns
            if (k0 < a.width) {
                step(k0, 0, std::true_type{});
                if (k0 + 32 < a.width) step(k0 + 32, 32, std::true_type{});
            }
            gather();
            // the warps' sums, in a fixed order: w + (w + 4), then the four; then the CTAs'
            auto at = [&](int i, int n, int j) -> float& {
                return sums[warp & 3][i * 16 + (j >> 1) * 8 + g][n * 8 + t * 2 + (j & 1)];
            };
            if (warp >= 4)
#pragma unroll
                for (int i = 0; i < MT; ++i)
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int j = 0; j < 4; ++j) at(i, n, j) = sum[i][n][j];
            __syncthreads();
            if (warp < 4)
#pragma unroll
                for (int i = 0; i < MT; ++i)
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int j = 0; j < 4; ++j) at(i, n, j) += sum[i][n][j];
            __syncthreads();
            auto four = [&](int row, int c) {
                return (sums[0][row][c] + sums[1][row][c]) + (sums[2][row][c] + sums[3][row][c]);
            };
            if (splits > 1) {
                for (int i = tid; i < TM * NT * 8; i += kThreads) {
                    const int row = i / (NT * 8), c = i % (NT * 8);
                    sums[0][row][c] = four(row, c);
                }
                tc::cluster_sync();
            }
            for (int i = tid; i < TM * NT * 8; i += kThreads) {
                const int row = i / (NT * 8), c = i % (NT * 8), r = rb + c;
                if (sid[row] != ad || r >= a.rank || row % splits != split) continue;
                float s = 0.f;
                if (splits == 1) {
                    s = four(row, c);
                } else {
                    float part[kMaxSplits];
#pragma unroll
                    for (int k = 0; k < kMaxSplits; ++k)
                        part[k] = tc::ld_cluster(tc::map_shared(tc::smem_u32(&sums[0][row][c]), min(k, splits - 1)));
#pragma unroll
                    for (int k = 0; k < kMaxSplits; ++k) s += k < splits ? part[k] : 0.f;
                }
                const float h = f * s;
                a.low.t[(m0 + row) * a.rank + r] = h;
                if (!F16 && sslot[row] < kPartSlots)
                    put_parts<T>(parts_row(a, m0 + row) + sslot[row] * a.lp.cols, a.lp, r, h);
            }
            // the sums are read before the next ones, or the CTA's end
            if (splits > 1) tc::cluster_sync();
            else __syncthreads();
        }
    }
    if constexpr (F16) {   // the parts, now that every number of the rows is known: a warp a row
#pragma unroll
        for (int k = 0; k < TM / 8; ++k) {
            const int i = warp + 8 * k;
            if (m0 + i >= a.rows || i % splits != split || sid[i] < 0) continue;
            float v[kMaxRank / 32], most = 0.f;
#pragma unroll
            for (int j = 0; j < kMaxRank / 32; ++j) {
                const int r = lane + 32 * j;
                v[j] = r < a.rank ? a.low.t[(m0 + i) * a.rank + r] : 0.f;
                most = fmaxf(most, finite_size(v[j]));
            }
            const int power = row_power(warp_max(most));
            const float up = row_factor(power);
            if (lane == 0) a.low.power[m0 + i] = (uint8_t)power;
            if (sslot[i] < kPartSlots)
#pragma unroll
                for (int j = 0; j < kMaxRank / 32; ++j)
                    if (lane + 32 * j < a.rank)
                        put_parts<T>(parts_row(a, m0 + i) + sslot[i] * a.lp.cols, a.lp, lane + 32 * j, v[j] * up);
        }
    }
}

// ── small forward problems in one launch
// 128 features x 32 rows a CTA on the CUDA cores (true fp32 products), with the rows' h made by
// every CTA that needs them: at these sizes a launch costs more than the few products. Not
// worth it beyond: the thin product is repeated for every 128 features, and the wide one runs
// at the CUDA cores' rate. Bound by latency: one clip's 128 x 2048 fp32 projection (rank 8) 9.8 us, 256 clips'
// (4.7 MB, 0.15 GFLOP) 14.4. (Its rule does not look at the rank: at 128 ranks the thin product is as large as a CTA's
// wide one. Not measured there.)
constexpr int kSmallF = 128, kSmallR = 32, kSmallK = 128, kSmallPitch = kSmallK + 4;

struct SmallArgs {
    const void *x, *W, *A, *B, *bias;
    int64_t ldx, ldy;
    const float* scale;
    const int* ids;
    int rows, width, feats, rank, adapters;
    int x_vec, w_vec, a_vec;     // rows on 4-number boundaries
    DropProb drop;
    const uint64_t* rng;
    int zero_padding;
    void* y;
    float* h;                    // nullable
};

// 4 numbers of a row from column k, zero from `width` on
template <class T>
__device__ __forceinline__ float4 row4(const T* row, int k, int width, bool vec) {
    if (vec && k + 4 <= width) {
        if constexpr (sizeof(T) == 4) {
            return __ldg(reinterpret_cast<const float4*>(row + k));
        } else {
            const uint2 q = __ldg(reinterpret_cast<const uint2*>(row + k));
            const T* e = reinterpret_cast<const T*>(&q);
            return make_float4(to_f(e[0]), to_f(e[1]), to_f(e[2]), to_f(e[3]));
        }
    }
    float v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = k + j < width ? to_f(row[k + j]) : 0.f;
    return make_float4(v[0], v[1], v[2], v[3]);
}

template <class T>
__global__ void __launch_bounds__(2 * kThreads) project_small_kernel(const __grid_constant__ SmallArgs a) {
    extern __shared__ float sm[];
    float* ws = sm;                                   // [128][pitch]
    float* xs = ws + kSmallF * kSmallPitch;           // [32][pitch]
    float* hs = xs + kSmallR * kSmallPitch;           // [32][rank]
    __shared__ int sid[kSmallR];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int f0 = blockIdx.y * kSmallF, m0 = blockIdx.x * kSmallR;
    if (warp >= 8) {
        // ── h, beside the shared projection: a warp takes every eighth row, two at a time, 8
        // ranks at a time, its lanes 4 columns each
        const RngKey key = a.drop.thr ? load_rng(a.rng) : RngKey{};
        const int mine = warp - 8;
        const bool keep_h = a.h && blockIdx.y == 0;
        int id4[4];   // ids of this warp's rows, loaded together
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int m = m0 + mine + 8 * i;
            id4[i] = m < a.rows ? __ldg(a.ids + m) : -2;
            if (lane == 0) sid[mine + 8 * i] = id4[i];
        }
#pragma unroll
        for (int i = 0; i < 4; i += 2) {
            bool has[2];
            const T *x[2], *A[2];
            float f[2];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int m = m0 + mine + 8 * (i + u), ad = id4[i + u];
                has[u] = ad >= 0 && ad < a.adapters;
                x[u] = (const T*)a.x + (has[u] ? m : 0) * a.ldx;
                A[u] = (const T*)a.A + (int64_t)(has[u] ? ad : 0) * a.rank * a.width;
                f[u] = a.drop.scale * (a.scale && has[u] ? __ldg(a.scale + ad) : 1.f);
                if (!has[u] && keep_h && m < a.rows)
                    for (int r = lane; r < a.rank; r += 32) a.h[(int64_t)m * a.rank + r] = 0.f;
            }
            if (!has[0] && !has[1]) continue;
            for (int r0 = 0; r0 < a.rank; r0 += 8) {
                float s[2][8] = {};
                for (int k = lane * 4; k < a.width; k += 128) {
                    float4 v[2], w[2][8];
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        v[u] = row4(x[u], k, a.width, a.x_vec);
#pragma unroll
                        for (int r = 0; r < 8; ++r)
                            w[u][r] = row4(A[u] + (int64_t)min(r0 + r, a.rank - 1) * a.width, k, a.width, a.a_vec);
                    }
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        float4& q = v[u];
                        if (a.drop.thr) {
                            const uint32_t keep =
                                keep_bits(k >> 3, (uint32_t)(m0 + mine + 8 * (i + u)), key, a.drop.thr) >> (k & 7);
                            q.x = keep & 1 ? q.x : 0.f;
                            q.y = keep & 2 ? q.y : 0.f;
                            q.z = keep & 4 ? q.z : 0.f;
                            q.w = keep & 8 ? q.w : 0.f;
                        }
#pragma unroll
                        for (int r = 0; r < 8; ++r)
                            s[u][r] = fmaf(q.x, w[u][r].x,
                                           fmaf(q.y, w[u][r].y, fmaf(q.z, w[u][r].z, fmaf(q.w, w[u][r].w, s[u][r]))));
                    }
                }
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int r = 0; r < 8; ++r)
                        for (int o = 16; o > 0; o >>= 1) s[u][r] += __shfl_xor_sync(0xffffffffu, s[u][r], o);
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int r = 0; r < 8; ++r)
                        if (lane == r && has[u] && r0 + r < a.rank) {
                            const int row = mine + 8 * (i + u);
                            hs[row * a.rank + r0 + r] = f[u] * s[u][r];
                            if (keep_h) a.h[(int64_t)(m0 + row) * a.rank + r0 + r] = f[u] * s[u][r];
                        }
            }
        }
    }
    // ── the shared projection: lane: features f0 + lane + 32 i; warp: rows 4 warp .. + 3
    if (warp < 8) {   // and their rows of B towards L2
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int m = m0 + warp * 4 + j, ad = m < a.rows ? __ldg(a.ids + m) : -1;
            if (ad >= 0 && ad < a.adapters)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (f0 + lane + 32 * i < a.feats)
                        tc::prefetch_l2((const T*)a.B + ((int64_t)ad * a.feats + f0 + lane + 32 * i) * a.rank);
        }
    }
    float acc[4][4] = {};
    if (warp < 8)
        for (int k0 = 0; k0 < a.width; k0 += kSmallK) {
            const int c = lane * 4, k = k0 + c;
            float4 x[4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
                x[i] = row4((const T*)a.x + (int64_t)min(m0 + warp + 8 * i, a.rows - 1) * a.ldx, k, a.width, a.x_vec);
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                float4 w[8];
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    w[i] = row4((const T*)a.W + (int64_t)min(f0 + warp + 8 * (i + 8 * half), a.feats - 1) * a.width, k,
                                a.width, a.w_vec);
                if (half == 0) asm volatile("bar.sync 1, 256;" ::: "memory");   // the columns before these are used up
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    *reinterpret_cast<float4*>(&ws[(warp + 8 * (i + 8 * half)) * kSmallPitch + c]) = w[i];
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) *reinterpret_cast<float4*>(&xs[(warp + 8 * i) * kSmallPitch + c]) = x[i];
            asm volatile("bar.sync 1, 256;" ::: "memory");
            const int kn = min(kSmallK, (a.width - k0 + 3) / 4 * 4);
#pragma unroll 2
            for (int k = 0; k < kn; k += 4) {
                float4 u[4], v[4];
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    u[i] = *reinterpret_cast<const float4*>(&ws[(lane + 32 * i) * kSmallPitch + k]);
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    v[i] = *reinterpret_cast<const float4*>(&xs[(warp * 4 + i) * kSmallPitch + k]);
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        acc[i][j] = fmaf(u[i].x, v[j].x, acc[i][j]);
                        acc[i][j] = fmaf(u[i].y, v[j].y, acc[i][j]);
                        acc[i][j] = fmaf(u[i].z, v[j].z, acc[i][j]);
                        acc[i][j] = fmaf(u[i].w, v[j].w, acc[i][j]);
                    }
            }
        }
    __syncthreads();
    if (warp >= 8) return;
    // the adapters' products: the loads of 4 ranks of B for every (feature, row) go out together
    // (a row without an adapter reads the first one's, and does not add it)
    const bool b_vec = a.rank % 4 == 0 && reinterpret_cast<uintptr_t>(a.B) % (4 * sizeof(T)) == 0;
    float low[4][4] = {};
    const T* B[4];
    bool has[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int ad = sid[warp * 4 + j];
        has[j] = ad >= 0 && ad < a.adapters;
        B[j] = (const T*)a.B + (int64_t)(has[j] ? ad : 0) * a.feats * a.rank;
    }
    if (has[0] | has[1] | has[2] | has[3])
        for (int r = 0; r < a.rank; r += 4) {
            float4 w[4][4];
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    w[i][j] = row4(B[j] + (int64_t)min(f0 + lane + 32 * i, a.feats - 1) * a.rank, r, a.rank, b_vec);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float h[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) h[e] = has[j] && r + e < a.rank ? hs[(warp * 4 + j) * a.rank + r + e] : 0.f;
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    low[i][j] = fmaf(h[0], w[i][j].x,
                                     fmaf(h[1], w[i][j].y, fmaf(h[2], w[i][j].z, fmaf(h[3], w[i][j].w, low[i][j]))));
            }
        }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int f = f0 + lane + 32 * i;
        if (f >= a.feats) continue;
        const float bias = a.bias ? to_f(((const T*)a.bias)[f]) : 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int m = m0 + warp * 4 + j, id = sid[warp * 4 + j];
            if (m >= a.rows) continue;
            T* y = (T*)a.y + m * a.ldy + f;
            if (id >= -1) *y = from_f<T>(acc[i][j] + bias + (has[j] ? low[i][j] : 0.f));
            else if (a.zero_padding) *y = from_f<T>(0.f);
        }
    }
}

// ── dA and dB: out_a(c, r) = sum_{m of a} keep(m, c) z[m][c] t[m][r]
struct OuterArgs {
    const void* z;
    int64_t ldz;
    int width, vec;
    const float* t;
    DropProb drop;
    void* out;                // adapters x (width x rank or rank x width) numbers
    int64_t oc, orr;          // strides of c and r in out
    float* part;              // [adapter][window][width][rank16]
    int blocks;               // of 128 columns
};
struct OuterPair {
    OuterArgs o[2];
    const int* ids;
    const uint64_t* rng;
    int rows, rank, adapters, windows, window;   // rows a window
    int slices;                                  // CTAs over the adapters of a window
    int* seen;                                   // [tensor][adapter][window]: rows of it
};

constexpr int kColumns = 128, kList = 1024;
// The join's rows of columns, spread so that lanes 8 columns (or 2 rows) apart, and neighbours, fall
// into different banks.
constexpr int kJoinPitch = 145;
__device__ __forceinline__ int join_at(int row, int c) { return row * kJoinPitch + c + (c >> 3); }

__device__ __forceinline__ uint32_t tf32_hi(float v) {
    uint32_t r;
    asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(r) : "f"(v));
    return r;
}
// v = hi + lo in tf32, off by at most 2^-23 (fp32 itself: 2^-24; a third part would be another MMA for every
// two); a number that is not finite has no remainder, and one that rounds over the range's end is cut
__device__ __forceinline__ void tf32_split(float v, uint32_t& hi, uint32_t& lo) {
    hi = tf32_hi(v);
    if (isinf(__uint_as_float(hi)) && isfinite(v)) hi = __float_as_uint(v) & 0xFFFFE000u;
    lo = isfinite(v) ? tf32_hi(v - __uint_as_float(hi)) : 0u;
}
__device__ __forceinline__ void mma_1688(float (&d)[4], const uint32_t (&x)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(x[0]), "r"(x[1]), "r"(x[2]), "r"(x[3]), "r"(b0), "r"(b1));
}

template <class T>
struct OuterCfg {
    static constexpr bool F32 = sizeof(T) == 4;
    static constexpr int V = 16 / sizeof(T), NB = kColumns / (8 * V);   // columns a vector, vectors a row and lane
    static constexpr int kAhead = F32 ? 2 : 4;                          // steps in flight a warp
    static constexpr int kStep = (2 * NB + 1) * 512;                    // bytes of a step: [vector | t][lane][16]
    static constexpr int kRing = 8 * kAhead * kStep, kJoin = 8 * 16 * kJoinPitch * 4;
    static constexpr int kSmem = kRing > kJoin ? kRing : kJoin;
};

// One CTA per (128 columns, slice of the adapters, window of rows). In a window of up to kList
// rows it goes through the adapters of its slice that occur there (the others cost nothing, so
// windows may be short and CTAs alike, however the rows are ordered); in a longer one it has one adapter.
// It lists the adapter's rows, then takes 8 of them a step as the contraction of tf32 MMAs
// (16-bit numbers are tf32 numbers; t is a tf32 pair, fp32 z too). A lane's 16 bytes of a row are 8
// (fp32: 4) neighbouring columns, which go to the same slot of as many MMAs, so z goes
// to operand registers without a shuffle; each lane copies its own bytes of the next steps into
// its own places in shared memory, so nothing synchronises. Warps share a step's columns and
// divide the ranks (16 a warp) and the steps; their sums join in shared memory in warp order.
// Bound by instructions (operands unpacked, and with dropout the generator's, a third of the time) and
// the start and join of a CTA's adapters, not by z: 8192 rows, bf16, 16 ranks, dA and dB of 4096
// columns each (134 MB) 91 us with dropout, 71 without.
template <class T>
__global__ void __launch_bounds__(kThreads, sizeof(T) == 4 ? 1 : 2)
    outer_kernel(const __grid_constant__ OuterPair P) {
    using C = OuterCfg<T>;
    constexpr bool F32 = C::F32;
    constexpr int V = C::V, NB = C::NB;
    __shared__ __align__(16) int list[kList], wids[kList];       // rows of an adapter; the window's adapters
    __shared__ int wcount[8];
    extern __shared__ __align__(16) uint8_t dyn[];               // the warps' rings; then their sums
    float* joined = reinterpret_cast<float*>(dyn);               // [warps][16][128]: join_at
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int which = (int)blockIdx.x >= P.o[0].blocks;
    const OuterArgs& o = P.o[which];
    const int c0 = ((int)blockIdx.x - (which ? P.o[0].blocks : 0)) * kColumns;
    const int win = blockIdx.z;
    const bool one = P.slices == P.adapters;                     // adapter blockIdx.y alone
    const int rblocks = (P.rank + 15) / 16;
    int rgroups = 1;                                             // warps over ranks: a power of two
    while (rgroups < rblocks) rgroups *= 2;
    const int sgroups = 8 / rgroups, rg = warp % rgroups, sg = warp / rgroups, r0 = rg * 16;
    const RngKey key = o.drop.thr ? load_rng(P.rng) : RngKey{};
    const uint32_t ring = tc::smem_u32(dyn) + (uint32_t)(warp * C::kAhead * C::kStep + lane * 16);
    const int begin = win * P.window, end = min(P.rows, begin + P.window);
    const int64_t all = (int64_t)o.width * P.rank;
    if (!one) {
        // the window's adapters of this slice, -1 for the others
        for (int i = tid; i < kList; i += kThreads) {
            const int id = begin + i < end ? __ldg(P.ids + begin + i) : -1;
            wids[i] = id >= 0 && id < P.adapters && id % P.slices == (int)blockIdx.y ? id : -1;
        }
        if (P.windows > 1 && c0 == 0)   // windows without rows of an adapter leave no sums, only the word that says so
            for (int i = blockIdx.y + tid * P.slices; i < P.adapters; i += kThreads * P.slices)
                P.seen[(which * P.adapters + i) * P.windows + win] = 0;
        __syncthreads();
    }
    int ad = one ? (int)blockIdx.y : (int)blockIdx.y - P.slices;
    for (;;) {
        if (!one) {
            // the next adapter that occurs, in order
            int next = P.adapters;
            for (int i = tid; i < kList; i += kThreads)
                if (wids[i] >= 0 && wids[i] > ad) next = min(next, wids[i]);
            next = __reduce_min_sync(0xffffffffu, next);
            __syncthreads();
            if (lane == 0) wcount[warp] = next;
            __syncthreads();
#pragma unroll
            for (int w = 0; w < 8; ++w) next = min(next, wcount[w]);
            if (P.windows == 1)   // zeros of those between
                for (int z = ad + P.slices; z < min(next, P.adapters); z += P.slices)
                    for (int i = tid; i < P.rank * kColumns; i += kThreads) {
                        const int c = o.orr == 1 ? i / P.rank : i % kColumns;
                        const int r = o.orr == 1 ? i % P.rank : i / kColumns;
                        if (c0 + c < o.width) ((T*)o.out)[z * all + (c0 + c) * o.oc + r * o.orr] = from_f<T>(0.f);
                    }
            if (next >= P.adapters) break;
            ad = next;
        }
        // An MMA truncates its sum, always towards zero, so those of kPiece steps go to `kept`, rounded to nearest:
        // fp32's at hand, 16-bit types' (whose long pieces few calls fill) in local memory, having no registers left.
        constexpr int kPiece = F32 ? 8 : 128;
        float acc[V * NB / 2][2][4] = {};
        std::conditional_t<F32, float, volatile float> kept[V * NB / 2][2][4];
        if (F32)
#pragma unroll
            for (int i = 0; i < V * NB; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) kept[i >> 1][i & 1][e] = 0.f;
        int in_piece = 0, pieces = 0;
        int rows_seen = 0;
        for (int base = begin; base < end; base += kList) {
            // the rows of this adapter, in order
            const int stop = min(end, base + kList);
            int have = 0;
            __syncthreads();
            static_assert(kList == 4 * kThreads, "four rows a thread");
            {
                int id[4];
                uint32_t hits = 0;
                if (one) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) id[j] = __ldg(P.ids + min(base + tid * 4 + j, P.rows - 1));
                } else {
                    const int4 q = *reinterpret_cast<const int4*>(&wids[tid * 4]);
                    id[0] = q.x; id[1] = q.y; id[2] = q.z; id[3] = q.w;
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) hits |= (uint32_t)(base + tid * 4 + j < stop && id[j] == ad) << j;
                int at = __popc(hits);   // hits up to this thread's, in the warp
#pragma unroll
                for (int o = 1; o < 32; o *= 2) {
                    const int u = __shfl_up_sync(0xffffffffu, at, o);
                    if (lane >= o) at += u;
                }
                if (lane == 31) wcount[warp] = at;
                at -= __popc(hits);
                __syncthreads();
#pragma unroll
                for (int w = 0; w < 8; ++w) {
                    if (w < warp) at += wcount[w];
                    have += wcount[w];
                }
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (hits >> j & 1) list[at++] = base + tid * 4 + j;
                __syncthreads();
            }
            rows_seen += have;
            if (r0 >= P.rank) continue;
            const int by = sgroups * 8;
            // contraction slots t and t + 4 of step s: past the list's end its last row again, with t = 0
            auto row_of = [&](int s, int u) { return list[min(s + t + 4 * u, have - 1)]; };
            auto fetch = [&](int s, int slot) {   // this lane's bytes of step s into its places
                if (s < have) {
                    const uint32_t to = ring + (uint32_t)(slot * C::kStep);
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        const int m = row_of(s, u);
                        const T* row = (const T*)o.z + (int64_t)m * o.ldz + c0 + g * V;
#pragma unroll
                        for (int n = 0; n < NB; ++n) {
                            // (past the row's end: nothing is read, from an address inside it)
                            const int left = o.width - (c0 + g * V + n * 8 * V);
                            copy_async16(to + (uint32_t)((u * NB + n) * 512),
                                         left > 0 ? row + n * 8 * V : (const T*)o.z,
                                         min(max(left, 0), V) * (int)sizeof(T));
                        }
                        const float* tr = o.t + (int64_t)m * P.rank;
#pragma unroll
                        for (int n = 0; n < 2; ++n)
                            copy_async4(to + (uint32_t)(2 * NB * 512 + (u * 2 + n) * 4),
                                        tr + min(r0 + n * 8 + g, P.rank - 1));
                    }
                }
                copy_async_commit();
            };
            int slot = 0;
            if (o.vec)
#pragma unroll
                for (int i = 0; i < C::kAhead - 1; ++i) fetch(sg * 8 + i * by, i);
#pragma unroll 1
            for (int s = sg * 8; s < have; s += by) {
                if (in_piece++ == kPiece) {
#pragma unroll
                    for (int i = 0; i < V * NB; ++i)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            float& d = acc[i >> 1][i & 1][e];
                            kept[i >> 1][i & 1][e] = F32 || pieces ? kept[i >> 1][i & 1][e] + d : d;
                            d = 0.f;
                        }
                    in_piece = 1;
                    pieces = 1;
                }
                uint4 q[2][NB];
                float tv[2][2];
                if (o.vec) {
                    fetch(s + (C::kAhead - 1) * by, slot == 0 ? C::kAhead - 1 : slot - 1);
                    copy_async_wait<C::kAhead - 1>();
                    const uint8_t* from = dyn + (warp * C::kAhead + slot) * C::kStep + lane * 16;
#pragma unroll
                    for (int u = 0; u < 2; ++u)
#pragma unroll
                        for (int n = 0; n < NB; ++n)
                            q[u][n] = *reinterpret_cast<const uint4*>(from + (u * NB + n) * 512);
                    const float4 f = *reinterpret_cast<const float4*>(from + 2 * NB * 512);
                    tv[0][0] = f.x; tv[0][1] = f.y; tv[1][0] = f.z; tv[1][1] = f.w;
                    slot = slot + 1 == C::kAhead ? 0 : slot + 1;
                } else {
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        const int m = row_of(s, u);
#pragma unroll
                        for (int n = 0; n < 2; ++n)
                            tv[u][n] = o.t[(int64_t)m * P.rank + min(r0 + n * 8 + g, P.rank - 1)];
                        // (columns past the row's end are the last one again: their sums are not stored)
                        const T* row = (const T*)o.z + (int64_t)m * o.ldz;
#pragma unroll
                        for (int n = 0; n < NB; ++n) {
                            T* e = reinterpret_cast<T*>(&q[u][n]);
#pragma unroll
                            for (int j = 0; j < V; ++j)
                                e[j] = __ldg(row + min(c0 + n * 8 * V + g * V + j, o.width - 1));
                        }
                    }
                }
                uint32_t bh[2][2], bl[2][2];
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int n = 0; n < 2; ++n)
                        tf32_split(s + t + 4 * u < have ? tv[u][n] : 0.f, bh[n][u], bl[n][u]);
                if (o.drop.thr)
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        const uint32_t m = (uint32_t)row_of(s, u);
#pragma unroll
                        for (int n = 0; n < NB; ++n) {
                            const int c = c0 + n * 8 * V + g * V;
                            const uint4 w = philox4x32_10(c >> 3, m, key);
                            if constexpr (F32) {   // this lane's half of the group
                                const uint32_t w0 = c & 4 ? w.z : w.x, w1 = c & 4 ? w.w : w.y;
                                q[u][n].x = keep_lo(w0, o.drop.thr) ? q[u][n].x : 0u;
                                q[u][n].y = keep_hi(w0, o.drop.thr) ? q[u][n].y : 0u;
                                q[u][n].z = keep_lo(w1, o.drop.thr) ? q[u][n].z : 0u;
                                q[u][n].w = keep_hi(w1, o.drop.thr) ? q[u][n].w : 0u;
                            } else {
                                q[u][n] = drop_group(q[u][n], w, o.drop.thr);
                            }
                        }
                    }
                // MMA (i, j): column slots g and g + 8 are column j of vectors 2i and 2i + 1
#pragma unroll
                for (int i = 0; i < NB / 2; ++i)
#pragma unroll
                    for (int j = 0; j < V; ++j) {
                        uint32_t f[4], fl[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) {   // operand registers: (slot g | g + 8) + 2 * (row t | t + 4)
                            const float v = to_f(reinterpret_cast<const T*>(&q[e >> 1][2 * i + (e & 1)])[j]);
                            if constexpr (F32) tf32_split(v, f[e], fl[e]);
                            else f[e] = __float_as_uint(v);
                        }
#pragma unroll
                        for (int n = 0; n < 2; ++n) {
                            float(&d)[4] = acc[i * V + j][n];
                            if constexpr (F32) {
                                mma_1688(d, fl, bl[n][0], bl[n][1]);
                                mma_1688(d, fl, bh[n][0], bh[n][1]);
                            }
                            mma_1688(d, f, bl[n][0], bl[n][1]);
                            mma_1688(d, f, bh[n][0], bh[n][1]);
                        }
                    }
            }
            copy_async_wait<0>();
        }
        if (P.windows > 1) {
            if (tid == 0 && c0 == 0) P.seen[(which * P.adapters + ad) * P.windows + win] = rows_seen;
            if (rows_seen == 0) return;   // (in a window of its own adapter alone)
        }
        if (F32 || pieces)
#pragma unroll
            for (int i = 0; i < V * NB; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[i >> 1][i & 1][e] += kept[i >> 1][i & 1][e];
        // join the step groups; then (column, rank) to the output or the window's partial sums
        __syncthreads();
#pragma unroll
        for (int i = 0; i < NB / 2; ++i)
#pragma unroll
            for (int j = 0; j < V; ++j)
#pragma unroll
                for (int n = 0; n < 2; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int c = (2 * i + (e >> 1)) * 8 * V + g * V + j, r = n * 8 + t * 2 + (e & 1);
                        joined[join_at(warp * 16 + r, c)] = acc[i * V + j][n][e];
                    }
        __syncthreads();
        // 128 columns of a rank side by side, or (rank the inner one) 16 ranks of a column
        for (int i = tid; i < rblocks * 16 * kColumns; i += kThreads) {
            int c, r;
            if (o.orr == 1) {
                r = i & 15;
                c = (i >> 4) % kColumns;
                r += (i >> 4) / kColumns * 16;
            } else {
                c = i % kColumns;
                r = i / kColumns;
            }
            if (c0 + c >= o.width || r >= P.rank) continue;
            float s = 0.f;
            for (int k = 0; k < sgroups; ++k) s += joined[join_at((k * rgroups + (r >> 4)) * 16 + (r & 15), c)];
            const int64_t at = (c0 + c) * o.oc + r * o.orr;
            if (P.windows == 1) ((T*)o.out)[ad * all + at] = from_f<T>(s);
            else o.part[((int64_t)ad * P.windows + win) * all + at] = s;
        }
        if (one) break;
    }
}

// The windows' sums of one adapter, in window order.
template <class T>
__global__ void outer_join_kernel(const __grid_constant__ OuterPair P) {
    const int which = blockIdx.z;
    const OuterArgs& o = P.o[which];
    if (!o.out) return;
    const int64_t all = (int64_t)o.width * P.rank;
    const int ad = blockIdx.y;
    const int* seen = P.seen + (which * P.adapters + ad) * P.windows;
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < all; i += (int64_t)gridDim.x * blockDim.x) {
        const float* p = o.part + (int64_t)ad * P.windows * all + i;
        float s = 0.f;
        for (int w = 0; w < P.windows; ++w)
            if (seen[w]) s += p[w * all];
        ((T*)o.out)[ad * all + i] = from_f<T>(s);
    }
}

// ── host side
// One stream-ordered allocation a call, from a pool that keeps what it has been given: the
// default pool returns its memory at every synchronisation, which costs the next call half a
// millisecond. Captured into a graph, the allocation is the graph's own.
struct Scratch {
    cudaStream_t st;
    char* p = nullptr;
    int64_t at = 0;
    explicit Scratch(cudaStream_t s) : st(s) {}
    void reserve(int64_t bytes) {
        if (bytes > 0) BSML_CUDA(cudaMallocFromPoolAsync((void**)&p, bytes, pool(), st));
    }
    void* take(int64_t bytes) {
        char* r = p + at;
        at += bytes;
        return r;
    }
    ~Scratch() {
        if (p) cudaFreeAsync(p, st);
    }
    inline static std::mutex mu;
    inline static cudaMemPool_t pools[64] = {};
    static int device() {
        int dev = 0;
        BSML_CUDA(cudaGetDevice(&dev));
        if (dev >= 64) fail("multilora", "device above 63");
        return dev;
    }
    // What no call uses any more, back to the device (and what graphs that are gone have left)
    static void release() {
        const int dev = device();
        std::lock_guard<std::mutex> lock(mu);
        if (pools[dev]) BSML_CUDA(cudaMemPoolTrimTo(pools[dev], 0));
        BSML_CUDA(cudaDeviceGraphMemTrim(dev));
    }
    static cudaMemPool_t pool() {
        const int dev = device();
        std::lock_guard<std::mutex> lock(mu);
        if (!pools[dev]) {
            cudaMemPoolProps props = {};
            props.allocType = cudaMemAllocationTypePinned;
            props.location.type = cudaMemLocationTypeDevice;
            props.location.id = dev;
            // allowed inside a capture too: a pool's making is not a stream's work
            cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
            BSML_CUDA(cudaThreadExchangeStreamCaptureMode(&mode));
            cudaMemPool_t made = nullptr;
            uint64_t keep = ~0ull;
            cudaError_t e = cudaMemPoolCreate(&made, &props);
            if (e == cudaSuccess) e = cudaMemPoolSetAttribute(made, cudaMemPoolAttrReleaseThreshold, &keep);
            BSML_CUDA(cudaThreadExchangeStreamCaptureMode(&mode));
            BSML_CUDA(e);
            pools[dev] = made;
        }
        return pools[dev];
    }
};

int64_t pad256(int64_t n) { return round_up(n, 256); }

struct LowBytes {
    int64_t t, parts, groups, power, all;
};
LowBytes low_bytes(const MultiLora& p, bool own_t) {
    LowBytes b;
    b.t = own_t ? pad256((int64_t)p.rows * p.rank * 4) : 0;
    b.parts = pad256((int64_t)p.rows * kPartSlots * low_parts(p.rank, p.dtype).cols * 2);
    b.groups = pad256(ceil_div(p.rows, 32) * 2 * (int64_t)sizeof(RowGroup));
    b.power = p.dtype == DT_F16 ? pad256(p.rows) : 0;
    b.all = b.t + b.parts + b.groups + b.power;
    return b;
}

// rows of numbers of `esize` bytes on 16-byte boundaries
bool aligned16(const void* p, int64_t ld, int64_t rows, int esize) {
    return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && (rows <= 1 || (ld * esize) % 16 == 0);
}

template <class T>
constexpr int kTileRows = sizeof(T) == 4 ? 16 : 32;

template <class T, bool TR>
void shrink(const ShrinkArgs& a, bool tiles, cudaStream_t st) {
    ::bsml::count_launch();
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.blockDim = dim3(kThreads);
    cfg.stream = st;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    auto go = [&](void (*kernel)(ShrinkArgs)) { BSML_CUDA(cudaLaunchKernelEx(&cfg, kernel, a)); };
    if (!tiles) {
        cfg.gridDim = dim3((unsigned)a.rows, (unsigned)ceil_div(a.rank, a.block));
        if (std::is_same<T, __half>::value) attr.val.clusterDim.y = cfg.gridDim.y;   // (at most 8: the row's power)
        go(shrink_rows_kernel<T, TR>);
    } else {
        cfg.gridDim = dim3((unsigned)(ceil_div(a.rows, kTileRows<T>) * a.splits));
        attr.val.clusterDim.x = (unsigned)a.splits;
        if (a.rank <= 8) go(shrink_tile_kernel<T, TR, 1>);
        else if (a.rank <= 16) go(shrink_tile_kernel<T, TR, 2>);
        else if (a.rank <= 32) go(shrink_tile_kernel<T, TR, 4>);
        else go(shrink_tile_kernel<T, TR, 8>);
    }
    BSML_LAUNCH("multilora shrink");
}

// Tiles of rows for h and g, or one CTA a row. Measured (us, a row's CTA | tiles): a row's reads its
// adapter from L2, about 10 TB/s in all, and with dropout makes a mask for every two ranks; a
// tile's chain is long however few the rows, longer with many ranks. bf16, 2048 columns, 16 ranks: 256 rows
// 5.0 | 9.7, 512 7.3 | 9.8, 1024 11.1 | 10.3; dropped: 256 9.2 | 11.6, 512 11.1 | 11.5; 64 ranks: 512 rows
// 18.4 | 16.3. From 1024 rows on, the rows' CTAs are two turns of all SMs: 768 columns, 8 ranks
// 7.2 | 6.0 (before it 1021 rows x 1021 columns, 12 ranks, fp16 10.2 | 12.1).
template <class T>
bool shrink_tiles(const MultiLora& p, int width, bool mask) {
    if (p.rows >= 1024) return true;
    const int64_t bytes = (int64_t)p.rows * p.rank * width * (int64_t)sizeof(T) * (mask ? 2 : 1);
    return bytes > (int64_t)(p.rank > 32 ? 128 : 48) << 20;
}
// CTAs a tile: the join costs some 3 us, a turn of 512 columns 1.2 to 6, so only where a CTA is
// spared two turns or more; not more CTAs than SMs (two an SM are no faster).
int shrink_splits(int64_t tiles, int width) {
    const int64_t turns = ceil_div(width, 512);
    const int64_t s = std::max<int64_t>(1, std::min<int64_t>({kMaxSplits, 148 / tiles, turns}));
    return turns - ceil_div(turns, s) >= 2 ? (int)s : 1;
}

template <class T>
struct Call {
    const MultiLora& p;
    cudaStream_t st;

    ProjectTc project_args(bool transposed) const {
        ProjectTc a;
        a.dtype = p.dtype;
        a.transposed = transposed;
        a.rows = p.rows;
        a.width = transposed ? p.cout : p.cin;
        a.feats = transposed ? p.cin : p.cout;
        a.rank = p.rank; a.adapters = p.adapters;
        a.W = p.W;
        a.Q = transposed ? p.A : p.B;
        a.ids = p.ids; a.rng = p.rng;
        a.zero_padding = p.zero_padding;
        if (sizeof(T) == 2 || shrink_tiles<T>(p, a.width, !transposed && p.dropout > 0)) a.P = transposed ? p.B : p.A;
        return a;
    }

    // operands laid out, then the low-rank numbers, then the wide product
    void project(ProjectTc& a, void* ops, DropProb mask, float scale) const {
        const LaidOut l = project_tc_prepare(a, ops, st);
        ShrinkArgs s = {};
        // 16-bit numbers are read where they were laid out, fp32 ones (there they are planes)
        // where they stand unless tiles read them
        const bool laid = sizeof(T) == 2;
        s.z = laid ? l.z : a.z; s.ldz = laid ? l.ldz : a.ldz;
        s.z_vec = aligned16(s.z, s.ldz, a.rows, sizeof(T));
        s.P = laid ? l.P : a.transposed ? p.B : p.A;
        s.ldp = laid ? l.ldp : a.transposed ? p.rank : p.cin;
        // (transposed: vectors of 8 ranks, so its rows have to hold whole ones)
        s.p_vec = aligned16(s.P, s.ldp, 2, sizeof(T)) && (!a.transposed || s.ldp >= round_up(p.rank, 8));
        s.zt = l.z; s.ldzt = l.ldz; s.zt_plane = l.z_plane;
        s.Pt = l.P; s.ldpt = l.ldp; s.pt_plane = l.p_plane;
        s.scale = p.scale; s.ids = p.ids;
        s.rows = p.rows; s.width = a.width; s.rank = p.rank; s.adapters = p.adapters;
        s.drop = mask;
        s.drop.scale = scale;
        s.rng = p.rng;
        s.low = a.low;
        s.lp = low_parts(p.rank, p.dtype);
        // few rows: a CTA for every 8 ranks (fp16, a cluster a row: 8 CTAs at most), while they all run at once
        s.block = (int64_t)p.rows * ceil_div(p.rank, 8) > 592          ? (int)round_up(p.rank, 8)
                  : std::is_same<T, __half>::value && p.rank > 64 ? 16
                                                                       : 8;
        s.splits = shrink_splits(ceil_div(p.rows, kTileRows<T>), a.width);
        const bool tiles = shrink_tiles<T>(p, a.width, mask.thr != 0);
        if (a.transposed) shrink<T, true>(s, tiles, st);
        else shrink<T, false>(s, tiles, st);
        if (a.out) project_tc(a, ops, st);
    }

    // The one-launch kernel against layout, thin product and wide product: while its CUDA-core
    // products are few, and its CTAs' loads of K few turns of 128.
    static bool aligned4(const void* q, int64_t ld, int64_t rows) {   // rows on boundaries of 4 numbers
        return reinterpret_cast<uintptr_t>(q) % (4 * sizeof(T)) == 0 && (rows <= 1 || ld % 4 == 0);
    }
    bool small() const {
        return p.cin <= 4 * kSmallK && (int64_t)p.rows * p.cin * p.cout <= (sizeof(T) == 4 ? 1 << 27 : 1 << 24);
    }
    void forward_small(const void* x, int64_t ldx, const void* bias, void* y, int64_t ldy, float* h) const {
        SmallArgs a = {};
        a.x = x; a.W = p.W; a.A = p.A; a.B = p.B; a.bias = bias;
        a.ldx = ldx; a.ldy = ldy;
        a.scale = p.scale; a.ids = p.ids;
        a.rows = p.rows; a.width = p.cin; a.feats = p.cout; a.rank = p.rank; a.adapters = p.adapters;
        a.x_vec = aligned4(x, ldx, p.rows);
        a.w_vec = aligned4(p.W, p.cin, 2);
        a.a_vec = aligned4(p.A, p.cin, 2);
        a.drop = drop_prob(p.dropout);
        a.rng = p.rng;
        a.zero_padding = p.zero_padding;
        a.y = y; a.h = h;
        auto smem = [](int rank) { return ((kSmallF + kSmallR) * kSmallPitch + kSmallR * rank) * 4; };
        // (the kernel's limit, the same from every call: two host threads may be here at once)
        BSML_CUDA(cudaFuncSetAttribute(project_small_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       smem(kMaxRank)));
        ::bsml::count_launch();
        project_small_kernel<T><<<dim3((unsigned)ceil_div(p.rows, kSmallR), (unsigned)ceil_div(p.cout, kSmallF)),
                                  2 * kThreads, smem(p.rank), st>>>(a);
        BSML_LAUNCH("multilora small");
    }

    void forward(const void* x, int64_t ldx, const void* bias, void* y, int64_t ldy, float* h) const {
        if (small()) return forward_small(x, ldx, bias, y, ldy, h);
        const DropProb dp = drop_prob(p.dropout);
        ProjectTc a = project_args(false);
        a.z = x; a.ldz = ldx; a.bias = bias; a.out = y; a.ldo = ldy;
        const int64_t laid = project_tc_scratch(a);
        const LowBytes lb = low_bytes(p, h == nullptr);
        Scratch s(st);
        s.reserve(laid + lb.all);
        void* ops = s.take(laid);
        take_low(a.low, s, lb, h);
        project(a, ops, dp, dp.scale);
    }

    static void take_low(LowRank& low, Scratch& s, const LowBytes& lb, float* t) {
        low.t = t ? t : (float*)s.take(lb.t);
        low.parts = s.take(lb.parts);
        low.groups = (RowGroup*)s.take(lb.groups);
        if (lb.power) low.power = (uint8_t*)s.take(lb.power);
    }

    void backward(const void* dy, int64_t lddy, const void* x, int64_t ldx, const float* h, void* dx, int64_t lddx,
                  void* dA, void* dB) const {
        const DropProb dp = drop_prob(p.dropout);
        if (p.rows == 0) {
            const size_t n = (size_t)p.adapters * p.rank * sizeof(T);
            if (dA) BSML_CUDA(cudaMemsetAsync(dA, 0, n * p.cin, st));
            if (dB) BSML_CUDA(cudaMemsetAsync(dB, 0, n * p.cout, st));
            return;
        }
        OuterPair o = {};
        o.ids = p.ids; o.rng = p.rng;
        o.rows = p.rows; o.rank = p.rank; o.adapters = p.adapters;
        // Windows of rows divide the adapters' sums: as many as give every SM four blocks, of 128 rows
        // or more (a CTA's rows are one chain), and fewer where many adapters would leave a window
        // few rows of each and much to write. Adapters share CTAs while a window's rows fit their
        // list.
        const int64_t blocks = (dA ? ceil_div(p.cin, kColumns) : 0) + (dB ? ceil_div(p.cout, kColumns) : 0);
        // (and not more than 512 MB of sums)
        const int64_t ctas = 592, sums = (int64_t)p.adapters * p.rank * 4 * ((dA ? p.cin : 0) + (dB ? p.cout : 0));
        const int64_t most =
            std::min(ctas / std::max<int64_t>(blocks, 1), ((int64_t)512 << 20) / std::max<int64_t>(sums, 1));
        o.windows = (int)std::max<int64_t>(
            1, std::min<int64_t>({32, most, p.rows / 128, p.rows / (32 * (int64_t)p.adapters)}));
        o.window = (int)round_up(ceil_div(p.rows, o.windows), 8);
        o.windows = (int)ceil_div(p.rows, o.window);
        const int64_t slices = std::min<int64_t>(p.adapters, ctas / std::max<int64_t>(blocks * o.windows, 1));
        o.slices = o.window > kList ? p.adapters : (int)std::max<int64_t>(1, slices);
        auto outer = [&](OuterArgs& u, const void* z, int64_t ldz, int width, DropProb drop, void* out, int64_t oc,
                         int64_t orr) {
            if (!out) return (int64_t)0;
            u.z = z; u.ldz = ldz; u.width = width; u.vec = aligned16(z, ldz, p.rows, sizeof(T));
            u.drop = drop; u.out = out; u.oc = oc; u.orr = orr;
            u.blocks = (int)ceil_div(width, kColumns);
            return o.windows > 1 ? pad256((int64_t)p.adapters * o.windows * width * p.rank * 4) : 0;
        };
        const int64_t pa = outer(o.o[0], x, ldx, p.cin, dp, dA, 1, p.cin);
        const int64_t pb = outer(o.o[1], dy, lddy, p.cout, DropProb{}, dB, p.rank, 1);
        ProjectTc a = project_args(true);
        a.z = dy; a.ldz = lddy; a.out = dx; a.ldo = lddx; a.drop = dp;
        const bool low = dx || dA;
        const int64_t laid = low ? project_tc_scratch(a) : 0;
        const LowBytes lb = low ? low_bytes(p, true) : LowBytes{};
        Scratch s(st);
        const int64_t ps = o.windows > 1 ? pad256((int64_t)2 * p.adapters * o.windows * 4) : 0;
        s.reserve(laid + lb.all + pa + pb + ps);
        if (low) {
            void* ops = s.take(laid);
            take_low(a.low, s, lb, nullptr);
            project(a, ops, DropProb{}, dp.scale);
        }
        if (!dA && !dB) return;
        o.o[0].t = a.low.t;
        o.o[1].t = h;
        o.o[0].part = (float*)s.take(pa);
        o.o[1].part = (float*)s.take(pb);
        o.seen = (int*)s.take(ps);
        constexpr int smem = OuterCfg<T>::kSmem;
        BSML_CUDA(cudaFuncSetAttribute(outer_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
        ::bsml::count_launch();
        outer_kernel<T><<<dim3(o.o[0].blocks + o.o[1].blocks, o.slices, o.windows), kThreads, smem, st>>>(o);
        BSML_LAUNCH("multilora outer");
        if (o.windows > 1) {
            ::bsml::count_launch();
            const int64_t most = (int64_t)std::max(p.cin, p.cout) * p.rank;
            outer_join_kernel<T><<<dim3((unsigned)std::min<int64_t>(256, ceil_div(most, 256)), p.adapters, 2), 256, 0,
                                   st>>>(o);
            BSML_LAUNCH("multilora join");
        }
    }
};

}  // namespace

void multilora_release_scratch() { Scratch::release(); }

void multilora_forward(const MultiLora& p, const void* x, int64_t ldx, const void* bias, void* y, int64_t ldy,
                       float* h, cudaStream_t st) {
    if (p.rows == 0) return;
    if (p.dtype == DT_F32) Call<float>{p, st}.forward(x, ldx, bias, y, ldy, h);
    else if (p.dtype == DT_BF16) Call<__nv_bfloat16>{p, st}.forward(x, ldx, bias, y, ldy, h);
    else Call<__half>{p, st}.forward(x, ldx, bias, y, ldy, h);
}

void multilora_backward(const MultiLora& p, const void* dy, int64_t lddy, const void* x, int64_t ldx, const float* h,
                        void* dx, int64_t lddx, void* dA, void* dB, cudaStream_t st) {
    if (p.dtype == DT_F32) Call<float>{p, st}.backward(dy, lddy, x, ldx, h, dx, lddx, dA, dB);
    else if (p.dtype == DT_BF16) Call<__nv_bfloat16>{p, st}.backward(dy, lddy, x, ldx, h, dx, lddx, dA, dB);
    else Call<__half>{p, st}.backward(dy, lddy, x, ldx, h, dx, lddx, dA, dB);
}

}  // namespace bsml
