// The shared projection with each row's low-rank adapter on the tensor cores (sm_100a):
//   D[f, m] = sum_k W(f, k) z[m, k] + sum_r Q_a(f, r) t[m, r]
// Features are the 128 (CTA pair: 256) TMEM lanes, rows of z the accumulator's columns. So a
// row's adapter belongs to a column range: the low-rank product is a few more K steps over the
// columns of its rows alone (operand Q_a by TMA; t as 16-bit parts). MMA columns come in groups
// of 16 or 32 rows. Where prompts meet inside a group, each row's parts lie in the columns of
// its slot (the ordinal of its run of rows in 32 rows; zero in the other slots), so one MMA a
// slot adds each adapter to its own rows, and zeros to the others. Zeros times an infinity or
// a NaN of a foreign adapter would be NaN. So such a group keeps its low-rank product in an
// accumulator of its own, where what is not finite is made again alone on the CUDA cores, at the cost of
// its rank numbers and not of the shared product's width. Groups of more runs than slots (single tokens of many requests) get
// their products on the CUDA cores in the epilogue, where a lane owns a feature and reads its
// own contiguous piece of Q_a. Adapters and rows so never meet.
//
// fp32 runs as bf16 planes: an fp32 number is the sum of three bf16 numbers, and the six plane
// products of significance 2^-16 and above are six passes of the same K loop, the smallest
// first: the accumulator's truncations are relative to its value, which stays small until the
// last pass.
// Every MMA truncates the accumulator's sum, always towards zero: positive fp16 numbers lose 6e-9 of
// their sum a column (measured: 4e-4 over 65536 columns; fp32's planes 8e-4 over 131072). So long sums leave
// the accumulator for registers, where fp32 adds round to nearest: fp32's every 512 columns of a pass
// (9e-7), 16-bit types' where an output would feel it, at 1/20 of its rounding: fp16's every 4096 columns
// (2e-5), bf16's every 16384 (1e-4). (Every 1024 would cost 4 % of 8192 x 4096 x 4096, under dropout 42.)
#include "multilora_tc.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cudaTypedefs.h>

#include <algorithm>
#include <atomic>
#include <mutex>
#include <type_traits>

#include "common.cuh"
#include "multilora.h"
#include "multilora_layout.h"
#include "scalar.cuh"
#include "tc_ptx.cuh"

namespace bsml {

namespace {

// The code of a bounded wait that ran out, for the host (multilora_error_flag). Waits look at a word
// of their own block's, so that one which ran out ends its block's others early, and no later call's.
__device__ int g_ml_err = 0;
__device__ __forceinline__ void report(int gave_up) {
    if (gave_up != tc::TC_OK) atomicCAS(&g_ml_err, tc::TC_OK, gave_up);
}

// tc::mbar_wait for a role that waits, through others, for one that waits for the kernel before (which may
// take as long as it likes): the limit counts from that kernel's end.
__device__ __noinline__ bool wait_longer(uint64_t* bar, uint32_t parity, int* err, int code) {
    const uint64_t t0 = tc::global_timer_ns();
    for (uint32_t i = 1;; ++i) {
        if (tc::mbar_try_wait(bar, parity)) return true;
        if ((i & 255) == 0) {
            if (*(volatile int*)err != tc::TC_OK) return false;
            if (tc::global_timer_ns() - t0 > tc::kWaitLimitNs) break;
        }
    }
    tc::grid_dependency_wait();
    return tc::mbar_wait(bar, parity, err, code);
}
template <bool LONG>
__device__ __forceinline__ bool wait_for(uint64_t* bar, uint32_t parity, int* err, int code) {
    if (!LONG) return tc::mbar_wait(bar, parity, err, code);   // one sum a tile: no role waits so
    return tc::mbar_try_wait(bar, parity) || wait_longer(bar, parity, err, code);
}

constexpr int kSmemMax = 232448;      // opt-in shared memory per block, static and dynamic
constexpr int kDynMax = kSmemMax - 1024;   // of it dynamic, at most: the kernels' limit, whatever a call takes
constexpr int kTileA = 16384;         // 128 features x 128 bytes of K
constexpr int kMaxStages = 12;
constexpr int kThreads = 320;         // split kernel: TMA warp, MMA warp, 8 epilogue warps
constexpr int kMaxTerms = 6;
// K steps of 64 in one accumulator, where sums are longer
template <class T>
constexpr int kPromote = sizeof(T) == 4 ? 8 : std::is_same<T, __half>::value ? 64 : 256;
constexpr int kMaxExt = 12;

// One TMA stage of the low-rank K steps: 64 ranks of Q plane `plane` from rank `rank0`, 64
// columns of the parts from `col0`, and the steps of 16 ranks that pair them (4 at most).
struct ExtStage {
    int8_t plane, n;
    int16_t rank0, col0;
    int8_t a[6], b[6];
};

struct PArgs {
    int rows, feats, rank, adapters;
    int kchunks;                 // 128-byte chunks of the contraction
    int n_terms;
    int8_t zp[kMaxTerms], wp[kMaxTerms];   // planes of each pass
    int np;                      // accumulator columns a tile
    int n_ft, n_mt;              // tiles over features and rows
    int stages;
    int splits, qpo;             // split kernel: CTAs over K of one tile, quads of columns each of them finishes
    int n_ext;
    ExtStage ext[kMaxExt];
    uint32_t idesc;              // without N
    const int* ids;
    const RowGroup* groups;
    const uint8_t* power;
    const float* t;
    const void* Q;               // as the caller has it
    int part_cols;               // of one slot
    const void* bias;
    DropProb drop;
    const uint64_t* rng;
    int zero_padding, q_vec, t_vec;
    void* out;
    int64_t ldo;
};

__device__ __forceinline__ uint8_t* align1024(uint8_t* p) {
    return reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(p) + 1023) & ~uintptr_t(1023));
}

// What a warp knows of a tile's rows: lane g has the group of 16 rows g. An MMA's columns come in
// steps of G = 16, or 32 over a CTA pair, where the lanes of two groups know the same but for
// the rows. gid: the adapter of every live row of the G, or kNone (no adapter), kMixed (several,
// or rows without one; a slot each) or kMany (on the CUDA cores).
constexpr int kNone = -1, kMixed = -2, kMany = -3;
struct TileRows {
    int gid;
    int slot[kPartSlots];   // the adapter in each slot, -1 for none
    uint32_t rows;          // RowGroup::rows
};
// This lane's group as the kernel before left it (after the dependency wait): loaded ahead of
// its use, so that nothing waits for it between two tiles.
struct RawRows {
    int4 slot;              // and `rows`
    uint2 rest;
};
__device__ __forceinline__ RawRows load_rows(const PArgs& a, int m0, int lane) {
    RawRows r = {make_int4(-1, -1, -1, 0), make_uint2(0, 0)};
    if (lane * 16 < a.np && m0 + lane * 16 < a.rows) {
        const int4* p = reinterpret_cast<const int4*>(a.groups + m0 / 16 + lane);
        r.slot = p[0];
        r.rest = *reinterpret_cast<const uint2*>(p + 1);
    }
    return r;
}
template <int G>
__device__ __forceinline__ TileRows tile_rows(const RawRows& raw) {
    static_assert(kPartSlots == 3, "RowGroup in two vectors");
    const uint32_t all = 0xffffffffu;
    TileRows t;
    t.slot[0] = raw.slot.x; t.slot[1] = raw.slot.y; t.slot[2] = raw.slot.z;
    t.rows = (uint32_t)raw.slot.w;
    uint32_t many = raw.rest.x, without = raw.rest.y;
    if (G == 32) {
        many |= __shfl_xor_sync(all, many, 1);
        without |= __shfl_xor_sync(all, without, 1);
#pragma unroll
        for (int k = 0; k < kPartSlots; ++k) t.slot[k] = max(t.slot[k], __shfl_xor_sync(all, t.slot[k], 1));
    }
    int n = 0;
    t.gid = kNone;
#pragma unroll
    for (int k = 0; k < kPartSlots; ++k) {
        if (many) t.slot[k] = -1;
        n += t.slot[k] >= 0;
        t.gid = max(t.gid, t.slot[k]);
    }
    if (many) t.gid = kMany;
    else if (n > 1 || (n == 1 && without)) t.gid = kMixed;
    return t;
}

// Whether the group's low-rank product is the MMAs' work.
__device__ __forceinline__ bool by_mma(int gid) { return gid >= 0 || gid == kMixed; }
// Whether that product has an accumulator of its own where there is no dropout. (fp16's always: it is in the
// powers of two of its rows.)
template <class T>
__device__ __forceinline__ bool apart(int gid) {
    return gid == kMixed || (std::is_same<T, __half>::value && gid >= 0);
}

// The powers of a lane's row (lane & 15) in N groups of 16, every STEP-th one from `g`, a byte each.
template <int N, int STEP>
__device__ __forceinline__ uint64_t load_powers(const PArgs& a, int m0, int g, int lane) {
    uint64_t p = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int c = (g + STEP * i) * 16 + (lane & 15);
        if (c < a.np && m0 + c < a.rows) p |= (uint64_t)a.power[m0 + c] << (8 * i);
    }
    return p;
}
// Number j of 16 columns (rows) times the power of its row: `power` is that of this lane's row.
__device__ __forceinline__ uint32_t times_power(uint32_t v, uint32_t power, int j) {
    return __float_as_uint(__uint_as_float(v) * __uint_as_float((__shfl_sync(0xffffffffu, power, j) & 0xFFu) << 23));
}

// A run of groups of one adapter in one slot: what the issuing threads go through. first: no
// lower slot has an adapter in these groups; own: they are apart().
constexpr int kMaxGroups = 8;
struct Run {
    int ad;
    int16_t c0, cols;
    int16_t slot;
    int8_t first, own;
};
typedef Run Runs[kPartSlots * kMaxGroups];
// The tile's runs, by slot, then column; returns how many. By a whole warp: lane (slot k, group
// g), because one thread's way through 24 places takes longer than the K steps that wait for it.
template <class T, int G>
__device__ __forceinline__ int find_runs(Runs& out, const TileRows& rows, int groups, int lane) {
    const uint32_t all = 0xffffffffu;
    const int k = lane / kMaxGroups, g = lane % kMaxGroups;
    int ad = -1;
#pragma unroll
    for (int i = 0; i < kPartSlots; ++i) {
        const int v = __shfl_sync(all, rows.slot[i], g * (G / 16));
        if (k == i && g < groups) ad = v;
    }
    const uint32_t has = __ballot_sync(all, ad >= 0);
    int low = 0;
    for (int i = 0; i < kPartSlots - 1; ++i) low |= i < k ? has >> (i * kMaxGroups + g) & 1 : 0;
    const int own = apart<T>(__shfl_sync(all, rows.gid, g * (G / 16)));
    const int kind = low | own << 1, ad_before = __shfl_up_sync(all, ad, 1), kind_before = __shfl_up_sync(all, kind, 1);
    const bool start = ad >= 0 && (g == 0 || ad != ad_before || kind != kind_before);
    const uint32_t starts = __ballot_sync(all, start);
    if (start) {
        const uint32_t more = (has & ~starts) >> lane >> 1;   // lanes after this one that go on with it
        out[__popc(starts & ((1u << lane) - 1))] =
            Run{ad, (int16_t)(g * G), (int16_t)(__ffs(~more) * G), (int16_t)k, (int8_t)!low, (int8_t)own};
    }
    __syncwarp();
    return __popc(starts);
}

__device__ __forceinline__ uint32_t idesc_n(uint32_t idesc, int n) { return idesc | ((uint32_t)(n >> 3) << 17); }

// s[i] = sum_r t[m[i]][r] Q_ad[i](f, r) on the CUDA cores, in rank order; 0 where ad[i] < 0. The
// loads of kBatch rows go out together: one row's chain of loads and sums costs about a
// microsecond, whatever its length.
constexpr int kBatch = 4;
template <class T, bool TR>
__device__ __forceinline__ void low_dots(const PArgs& a, const int (&m)[kBatch], const int (&ad)[kBatch], int f,
                                         float (&s)[kBatch]) {
    const float* t[kBatch];
    const T* q[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
        s[i] = 0.f;
        t[i] = a.t + (int64_t)m[i] * a.rank;
        q[i] = (const T*)a.Q + (TR ? (int64_t)max(ad[i], 0) * a.rank * a.feats + f
                                   : ((int64_t)max(ad[i], 0) * a.feats + f) * a.rank);
    }
    // ranks at a time, every load before the first sum
    constexpr int V = 16 / sizeof(T), RB = TR || sizeof(T) == 4 ? 8 : 16;
#pragma unroll 1
    for (int r0 = 0; r0 < a.rank; r0 += RB) {
        float4 x[kBatch][RB / 4];
#pragma unroll
        for (int i = 0; i < kBatch; ++i)
#pragma unroll
            for (int r = 0; r < RB; r += 4) {   // (past the last rank: the last ones again, not summed)
                if (a.t_vec) {
                    x[i][r / 4] = *reinterpret_cast<const float4*>(t[i] + min(r0 + r, a.rank - 4));
                } else {
                    const int l = a.rank - 1;
                    x[i][r / 4] = make_float4(t[i][min(r0 + r, l)], t[i][min(r0 + r + 1, l)], t[i][min(r0 + r + 2, l)],
                                              t[i][min(r0 + r + 3, l)]);
                }
            }
        auto add = [&](int i, int r, float w) {
            const float4 v = x[i][r / 4];
            if (r0 + r < a.rank) s[i] = fmaf(r % 4 == 0 ? v.x : r % 4 == 1 ? v.y : r % 4 == 2 ? v.z : v.w, w, s[i]);
        };
        if (!TR && a.q_vec) {
            uint4 w[kBatch][RB / V];
#pragma unroll
            for (int i = 0; i < kBatch; ++i)
#pragma unroll
                for (int r = 0; r < RB; r += V)
                    w[i][r / V] = __ldg(reinterpret_cast<const uint4*>(q[i] + min(r0 + r, a.rank - V)));
#pragma unroll
            for (int i = 0; i < kBatch; ++i)
#pragma unroll
                for (int r = 0; r < RB; ++r) add(i, r, to_f(reinterpret_cast<const T*>(&w[i][r / V])[r % V]));
        } else {
            float w[kBatch][RB];
#pragma unroll
            for (int i = 0; i < kBatch; ++i)
#pragma unroll
                for (int r = 0; r < RB; ++r)
                    w[i][r] = to_f(__ldg(q[i] + min(r0 + r, a.rank - 1) * (TR ? (int64_t)a.feats : 1)));
#pragma unroll
            for (int i = 0; i < kBatch; ++i)
#pragma unroll
                for (int r = 0; r < RB; ++r) add(i, r, w[i][r]);
        }
    }
#pragma unroll
    for (int i = 0; i < kBatch; ++i)
        if (ad[i] < 0) s[i] = 0.f;
}

// The adapter of row m, -1 for none
__device__ __forceinline__ int row_adapter(const PArgs& a, int m) {
    const int ad = __ldg(a.ids + m);
    return ad < a.adapters ? max(ad, -1) : -1;
}

// Adds to v[j] (j = 0..n-1, n a multiple of kBatch) the low-rank products of rows m0 + j, each of its own
// adapter, where row j is live and its element kept.
template <class T, bool TR>
__device__ __forceinline__ void add_many(const PArgs& a, int m0, int n, uint32_t live, uint32_t keep, int f, float* v) {
    if (f >= a.feats) return;
#pragma unroll 1
    for (int j0 = 0; j0 < n; j0 += kBatch) {
        int m[kBatch], ad[kBatch];
        float s[kBatch];
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
            m[j] = min(m0 + j0 + j, a.rows - 1);
            ad[j] = live >> (j0 + j) & 1 ? row_adapter(a, m[j]) : -1;
        }
        low_dots<T, TR>(a, m, ad, f, s);
#pragma unroll
        for (int j = 0; j < kBatch; ++j)
            if (keep >> (j0 + j) & 1) v[j0 + j] += s[j];
    }
}

// The products of 4 rows of a group of many adapters, kept ones, for feature f. Whole warp. Not inlined: the
// registers that it takes would spill around the K loop's end, and the L1 is shared memory.
template <class T, bool TR, bool DROP>
__device__ __noinline__ void quad_products(const PArgs& a, int m0, int4 ads, int f, float4* out) {
    static_assert(kBatch == 4, "a quad of columns");
    const RngKey key = DROP ? load_rng(a.rng) : RngKey{};
    if (f >= a.feats) return;
    const int ad[kBatch] = {ads.x, ads.y, ads.z, ads.w};
    int m[kBatch];
    float s[kBatch];
#pragma unroll
    for (int j = 0; j < kBatch; ++j) m[j] = min(m0 + j, a.rows - 1);
    low_dots<T, TR>(a, m, ad, f, s);
    if (DROP)
#pragma unroll
        for (int j = 0; j < kBatch; ++j)
            if (!(keep_bits(f >> 3, (uint32_t)m[j], key, a.drop.thr) >> (f & 7) & 1)) s[j] = 0.f;
    *out = make_float4(s[0], s[1], s[2], s[3]);
}

// What the CUDA cores do to 16 rows: the products of a group of many adapters. Not inlined: long, and
// rarely reached.
template <class T, bool TR>
__device__ __noinline__ void many_rows(const PArgs& a, int m0, uint32_t live, uint32_t keep, int f, float* v) {
    add_many<T, TR>(a, m0, 16, live, keep, f, v);
}
// The low-rank products of 16 rows of a mixed group, each by itself, over those at taddr, some of which are not
// finite (which may be a neighbour's doing). Whole warp. (The work of a group of many adapters, whatever
// stands in the operands: others wait for it, and their waits are bounded.)
template <class T, bool TR>
__device__ __noinline__ void repair(const PArgs& a, uint32_t live, uint32_t taddr, int m0, int f) {
    float w[16] = {};
    add_many<T, TR>(a, m0, 16, live, 0xFFFFu, f, w);
    __syncwarp();
    tc::tmem_st16(taddr, w);
}

// Bits j of the result (j = 0..15): column c0 + j of feature f is kept. Lanes 8i..8i+7 of a
// warp share a generator group (f is lane-contiguous from a multiple of 32): each makes the
// bits of two columns and takes its own from the others.
__device__ __forceinline__ uint32_t keep_columns(const PArgs& a, int m0, int f, int lane, RngKey key) {
    uint32_t mine[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) mine[i] = keep_bits(f >> 3, (uint32_t)(m0 + 8 * i + (lane & 7)), key, a.drop.thr);
    uint32_t keep = 0;
#pragma unroll
    for (int j = 0; j < 16; ++j)
        keep |= (__shfl_sync(0xffffffffu, mine[j >> 3], (lane & 24) | (j & 7)) >> (lane & 7) & 1u) << j;
    return keep;
}

// Sums of 16 rows from m0 for feature f to the output. Rows that are all live are stored without tests,
// which cost as much as all the rest.
template <class T>
__device__ __forceinline__ void store_rows(const PArgs& a, uint32_t live, uint32_t pad, int m0, int f, float bias,
                                           const float (&v)[16]) {
    if (f >= a.feats) return;
    T* o = (T*)a.out + (int64_t)m0 * a.ldo + f;
    if (live == 0xFFFFu) {
#pragma unroll
        for (int j = 0; j < 16; ++j, o += a.ldo) *o = from_f<T>(v[j] + bias);
        return;
    }
#pragma unroll
    for (int j = 0; j < 16; ++j, o += a.ldo) {
        if (live >> j & 1) *o = from_f<T>(v[j] + bias);
        else if (a.zero_padding && (pad >> j & 1)) *o = from_f<T>(0.f);
    }
}

// v: the sums of 16 rows from m0 for feature f, to the output (and before it what the CUDA cores
// add). rows: this warp's rows of the tile, g: the group of 16 in it. (What spills here goes to L2, the L1
// being shared memory: 16 epilogue warps of fewer registers, two groups a turn and calls that
// are not inlined were all slower.)
template <class T, bool TR>
__device__ __forceinline__ void finish_rows(const PArgs& a, const TileRows& rows, int g, int gid, int m0, int f,
                                            uint32_t keep, float bias, float (&v)[16]) {
    const uint32_t bits = __shfl_sync(0xffffffffu, rows.rows, g), live = bits & 0xFFFFu, pad = bits >> 16;
    if (gid == kMany) {
        float w[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) w[j] = v[j];
        many_rows<T, TR>(a, m0, live, keep, f, w);
#pragma unroll
        for (int j = 0; j < 16; ++j) v[j] = w[j];
    }
    store_rows<T>(a, live, pad, m0, f, bias, v);
}
// Rows of a mixed group whose low-rank product came out not finite: the shared sums from TMEM, and every
// row's own product on the CUDA cores. Whole warp.
template <class T, bool TR, bool DROP>
__device__ __noinline__ void again(const PArgs& a, uint32_t bits, uint32_t taddr, int m0, int f, int lane, float bias) {
    float v[16];
    tc::tmem_ld16(taddr, v);
    uint32_t keep = 0xFFFFu;
    if (DROP) keep = keep_columns(a, m0, f, lane, load_rng(a.rng));
    add_many<T, TR>(a, m0, 16, bits & 0xFFFFu, keep, f, v);
    store_rows<T>(a, bits & 0xFFFFu, bits >> 16, m0, f, bias, v);
}

// Producer side of one stage: A block (128 features of this CTA) and nb rows of the B operand.
template <bool TR, bool PAIR>
__device__ __forceinline__ void load_stage(uint8_t* st, const CUtensorMap* mA, const CUtensorMap* mB, uint64_t* bar,
                                           uint32_t bar_lead, int f0, int ka, int pa, int kb, int row, int pb) {
    auto load = [&](uint8_t* dst, const CUtensorMap* map, int c0, int c1, int c2) {
        if constexpr (PAIR) tc::tma_load_3d_pair(dst, map, bar_lead, c0, c1, c2);
        else tc::tma_load_3d(dst, map, bar, c0, c1, c2);
    };
    if constexpr (TR) {
        load(st, mA, f0, ka, pa);
        load(st + kTileA / 2, mA, f0 + 64, ka, pa);
    } else {
        load(st, mA, ka, f0, pa);
    }
    load(st + kTileA, mB, kb, row, pb);
}

template <bool TR>
__device__ __forceinline__ uint64_t desc_a(uint32_t base, int step) {
    if constexpr (TR) return tc::desc_mnmajor(base + step * 2048, kTileA / 2, false);
    else return tc::desc_kmajor_sw128(base + step * 32);
}

template <bool PAIR>
__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    if constexpr (PAIR) tc::umma_f16_pair(d, a, b, idesc, acc);
    else tc::umma<false>(d, a, b, idesc, acc);
}
template <bool PAIR>
__device__ __forceinline__ void commit(uint64_t* bar) {
    if constexpr (PAIR) tc::umma_commit_pair(bar);
    else tc::umma_commit(bar);
}

struct Ring {
    int slot = 0;
    uint32_t phase = 0;
    __device__ __forceinline__ void next(int stages) {
        if (++slot == stages) {
            slot = 0;
            phase ^= 1;
        }
    }
};

// Accumulators of a pair, and columns of its tile. TMEM's 512 columns hold two sums, or with dropout
// (whose low-rank product has an accumulator of its own) one sum and that. fp32's sums are many a
// tile, so it has two beside that of the low-rank product. (16-bit with two of 160 columns: 244 us
// where one of 256, its epilogue not hidden, takes 200: 8192 x 4096 x 4096, 16 ranks. L2 bounds
// narrow tiles.)
template <class T, bool DROP>
constexpr int kSums = DROP && sizeof(T) == 2 ? 1 : 2;
template <class T, bool DROP>
constexpr int kMaxColumns = DROP && sizeof(T) == 4 ? 160 : 256;
// Epilogue warps of a pair's CTA. Many sums run in 16 columns x groups registers a
// thread: 16 warps of 64 sums (and at most 96 registers) hold 256 columns.
template <bool LONG>
constexpr int kPairEpi = LONG ? 16 : 8;

// A tile's sums go to the accumulators in turn, whose uses every role counts alike: `at` is the next one, bit i
// of `uses` whether i was used an odd number of times. A tile with groups apart() also uses, for these, the one after its last
// sum's, and the next tile's first sum then uses that.
struct Turns {
    int at = 0;
    uint32_t uses = 0;
    __device__ __forceinline__ uint32_t phase(int i) const { return uses >> i & 1; }
    __device__ __forceinline__ void used(int i) { uses ^= 1u << i; }
    template <int B>
    __device__ __forceinline__ int next() {
        const int i = at;
        at = B == 1 ? 0 : at ^ 1;
        return i;
    }
};

struct TilePos {
    int f, m;
};
__device__ __forceinline__ TilePos tile_pos(const PArgs& a, int tile) {
    return TilePos{tile % a.n_ft, tile / a.n_ft};
}

// ── large problems: persistent CTA pairs
// A pair computes 256 features x np rows a tile: cta_group::2 MMAs read 128 features from
// each CTA's shared memory and half the rows of z from each, so an SM takes 64 bytes of
// operand a cycle from L2 at the full rate, where 128 features x 256 rows by one CTA would
// take 96. Accumulators are double buffered in TMEM, so a tile's stores run under the next
// tile's MMAs. With dropout (backward) the low-rank product has an accumulator of its own,
// because its mask does not apply to the shared one (kSums); the masks are made while the sums are.
// Without, groups where adapters meet inside an MMA's columns have it in the accumulator of the next tile's
// shared sum, and the epilogue adds it to the tile's own, in TMEM, before anything else (Turns).
// Bound by the tensor pipe at 256 columns (about 560 cycles for 64 columns of K, of which 512 are
// MMAs), by L2's operand rate below. A call of 8192 x 4096 x 4096 bf16 with 16 ranks, its thin product (26 us)
// and all, on the GPU: one adapter 208 us, prompts of 1000 rows 214, of 40 (every group apart) 270, fp16 (always
// apart) 229, the backward's dx 208, under dropout 231; fp32 2048 x 2048 x 2048 118.
template <class T, bool TR, bool DROP, bool LONG>
__global__ void __launch_bounds__(64 + 32 * kPairEpi<LONG>, 1)
    project_pair_kernel(const __grid_constant__ CUtensorMap mW, const __grid_constant__ CUtensorMap mZ,
                        const __grid_constant__ CUtensorMap mQ, const __grid_constant__ CUtensorMap mT,
                        const __grid_constant__ PArgs a) {
    constexpr bool F16 = std::is_same<T, __half>::value;
    constexpr int B = kSums<T, DROP>;             // sums in TMEM
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = align1024(smem_raw);
    __shared__ uint64_t full[kMaxStages], empty[kMaxStages], accf[2], acce[2], mdone;
    __shared__ uint32_t tslot;
    __shared__ int gave_up;
    __shared__ Runs runs[2];
    int* err = &gave_up;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const bool leader = tc::elect_one();
    const uint32_t rank = tc::cluster_ctarank();
    const int nb = a.np / 2;                         // rows of z in this CTA's half
    const int stage_bytes = kTileA + nb * 128;
    const int groups = a.np / 32;

    if (threadIdx.x == 0) {
        for (int s = 0; s < a.stages; ++s) {
            tc::mbar_init(&full[s], 1);
            tc::mbar_init(&empty[s], 1);
        }
        for (int s = 0; s < 2; ++s) {
            tc::mbar_init(&accf[s], 1);
            tc::mbar_init(&acce[s], 2 * kPairEpi<LONG>);
        }
        tc::mbar_init(&mdone, 1);
        gave_up = tc::TC_OK;
        tc::fence_barrier_init();
        tc::prefetch_tmap(&mW);
        tc::prefetch_tmap(&mZ);
        tc::prefetch_tmap(&mQ);
        tc::prefetch_tmap(&mT);
    }
    if (warp == 1) tc::tmem_alloc_pair(&tslot, 512);
    tc::tc_fence_before();
    __syncthreads();
    tc::cluster_sync();
    tc::tc_fence_after();
    const uint32_t tbase = tslot;
    const int n_tiles = a.n_ft * a.n_mt;
    const int pair = blockIdx.x / 2, pairs = gridDim.x / 2;
    const int steps = a.n_terms * a.kchunks;
    // sums a tile
    const int sums = LONG ? (steps + kPromote<T> - 1) / kPromote<T> : 1;

    if (warp == 0) {
        // ── TMA producer (both CTAs, into their own shared memory; the even CTA's barrier
        // counts both CTAs' bytes)
        Ring r;
        int issued = 0;
        bool ok = true, dep = false;
        auto stage = [&](const CUtensorMap* mA, const CUtensorMap* mB, int f0, int ka, int pa, int kb, int row,
                         int pb) {
            if (!wait_for<LONG>(&empty[r.slot], r.phase ^ 1, err, tc::TC_ERR_WAIT_EMPTY)) return false;
            if (rank == 0) tc::mbar_arrive_expect_tx(&full[r.slot], 2 * stage_bytes);
            load_stage<TR, true>(smem + r.slot * stage_bytes, mA, mB, nullptr,
                                 tc::map_shared(tc::smem_u32(&full[r.slot]), 0), f0, ka, pa, kb, row, pb);
            r.next(a.stages);
            ++issued;
            return true;
        };
        for (int tile = pair; ok && tile < n_tiles; tile += pairs) {
            const TilePos at = tile_pos(a, tile);
            const int m0 = at.m * a.np, f0 = at.f * 256 + (int)rank * 128;
            RawRows raw;
            if (dep) raw = load_rows(a, m0, lane);
            if (leader)
                for (int t = 0; ok && t < a.n_terms; ++t)
                    for (int c = 0; ok && c < a.kchunks; ++c)
                        ok = stage(&mW, &mZ, f0, c * 64, a.wp[t], c * 64, m0 + (int)rank * nb, a.zp[t]);
            __syncwarp();
            if (!dep) {
                tc::grid_dependency_wait();
                raw = load_rows(a, m0, lane);
                dep = true;
            }
            const TileRows rows = tile_rows<32>(raw);
            const int n_runs = find_runs<T, 32>(runs[0], rows, groups, lane);
            if (leader)
                for (int i = 0; ok && i < n_runs; ++i) {
                    const Run u = runs[0][i];
                    for (int e = 0; ok && e < a.n_ext; ++e) {
                        const ExtStage& x = a.ext[e];
                        ok = stage(&mQ, &mT, f0, x.rank0, x.plane * a.adapters + u.ad, u.slot * a.part_cols + x.col0,
                                   m0 + u.c0 + (int)rank * (u.cols / 2), 0);
                    }
                }
            ok = __all_sync(0xffffffffu, ok);
        }
        if (!dep) tc::grid_dependency_wait();
        // after an error, copies issued into the ring may still be in flight
        if (!ok && leader && rank == 0) {
            const int first = issued > a.stages ? issued - a.stages : 0;
            for (int i = first; i < issued; ++i)
                tc::mbar_wait(&full[i % a.stages], (i / a.stages) & 1, nullptr, tc::TC_ERR_DRAIN);
        }
    } else if (warp == 1) {
        if (rank == 0) {
            // ── MMA issuer (the even CTA)
            Ring r;
            bool ok = true, dep = false;
            Turns u;
            auto vacant = [&](int i) {   // accumulator i is read out
                return wait_for<LONG>(&acce[i], u.phase(i) ^ 1, err, tc::TC_ERR_WAIT_ACC);   // (at first: at once)
            };
            for (int tile = pair; ok && tile < n_tiles; tile += pairs) {
                const int m0 = tile_pos(a, tile).m * a.np;
                RawRows raw;
                if (dep) raw = load_rows(a, m0, lane);
                int buf = 0;
                for (int g = 0; g < sums; ++g) {   // (every lane counts, one issues)
                    buf = u.next<B>();
                    if (leader && ok) {
                        const uint32_t idesc = idesc_n(a.idesc, a.np);
                        const int n = LONG ? min(steps - g * kPromote<T>, kPromote<T>) : steps;
                        ok = vacant(buf);
                        for (int c = 0; ok && c < n; ++c) {
                            ok = tc::mbar_wait(&full[r.slot], r.phase, err, tc::TC_ERR_WAIT_FULL);
                            if (!ok) break;
                            tc::tc_fence_after();
                            const uint32_t base = tc::smem_u32(smem + r.slot * stage_bytes);
#pragma unroll
                            for (int k = 0; k < 4; ++k)
                                mma<true>(tbase + (uint32_t)(buf * a.np), desc_a<TR>(base, k),
                                          tc::desc_kmajor_sw128(base + kTileA + k * 32), idesc, (c | k) != 0);
                            commit<true>(&empty[r.slot]);
                            r.next(a.stages);
                        }
                        if (ok && g + 1 < sums) commit<true>(&accf[buf]);
                    }
                    if (g + 1 < sums) u.used(buf);
                }
                // the low-rank accumulator of the tile before is read out (with one sum, or with several a
                // tile, the last of which waited for that)
                if (DROP && B == 2 && leader && ok && sums == 1) ok = vacant(buf ^ 1);
                __syncwarp();
                if (!dep) {
                    tc::grid_dependency_wait();
                    raw = load_rows(a, m0, lane);
                    dep = true;
                }
                const TileRows rows = tile_rows<32>(raw);
                const int n_runs = find_runs<T, 32>(runs[1], rows, groups, lane);
                const bool own = !DROP && __any_sync(0xffffffffu, apart<T>(rows.gid));
                if (leader && ok) {
                    if (own) ok = vacant(buf ^ 1);
                    for (int i = 0; ok && i < n_runs; ++i) {
                        const Run v = runs[1][i];
                        const uint32_t idesc = idesc_n(a.idesc, v.cols);
                        const bool alone = DROP || v.own;   // in an accumulator of its own
                        const uint32_t d = tbase + (uint32_t)((DROP ? B : v.own ? buf ^ 1 : buf) * a.np + v.c0);
                        for (int e = 0; e < a.n_ext; ++e) {
                            const ExtStage& x = a.ext[e];
                            ok = tc::mbar_wait(&full[r.slot], r.phase, err, tc::TC_ERR_WAIT_FULL);
                            if (!ok) break;
                            tc::tc_fence_after();
                            const uint32_t base = tc::smem_u32(smem + r.slot * stage_bytes);
                            for (int k = 0; k < x.n; ++k)
                                mma<true>(d, desc_a<TR>(base, x.a[k]),
                                          tc::desc_kmajor_sw128(base + kTileA + x.b[k] * 32), idesc,
                                          !alone || !v.first || (e | k) != 0);
                            commit<true>(&empty[r.slot]);
                            r.next(a.stages);
                        }
                    }
                    if (ok) commit<true>(&accf[buf]);
                    if (ok && own) commit<true>(&accf[buf ^ 1]);
                }
                u.used(buf);
                if (own) u.used(buf ^ 1);
                ok = __all_sync(0xffffffffu, ok);
            }
            if (!dep) tc::grid_dependency_wait();
            // every issued MMA has completed before TMEM and shared memory are released
            if (leader) {
                tc::umma_commit_pair(&mdone);
                tc::mbar_wait(&mdone, 0, nullptr, tc::TC_ERR_DRAIN);
            }
        } else {
            tc::grid_dependency_wait();
        }
    } else {
        // ── epilogue: warp (q, h) has TMEM lanes 32q.. and every HG-th group of 16 rows
        constexpr int HG = kPairEpi<LONG> / 4;
        tc::grid_dependency_wait();
        const int q = warp & 3, h = (warp - 2) >> 2;
        const RngKey key = DROP ? load_rng(a.rng) : RngKey{};
        const uint32_t lead[2] = {tc::map_shared(tc::smem_u32(&acce[0]), 0), tc::map_shared(tc::smem_u32(&acce[1]), 0)};
        bool ok = true;
        Turns u;
        for (int tile = pair; tile < n_tiles; tile += pairs) {
            const TilePos at = tile_pos(a, tile);
            const int m0 = at.m * a.np, f = at.f * 256 + (int)rank * 128 + q * 32 + lane;
            const TileRows rows = tile_rows<32>(load_rows(a, m0, lane));
            const float bias = a.bias && f < a.feats ? to_f(((const T*)a.bias)[f]) : 0.f;
            const uint32_t trow = tbase + ((uint32_t)(q * 32) << 16);
            const bool own = !DROP && __any_sync(0xffffffffu, apart<T>(rows.gid));
            // groups whose low-rank product is not finite, and their rows once more, with the shared
            // sums at `column`
            uint32_t bad = 0;
            auto finish_again = [&](int column) {
#pragma unroll 1
                for (int g = h; g * 16 < a.np; g += HG) {
                    const uint32_t bits = __shfl_sync(0xffffffffu, rows.rows, g);
                    if (bad >> g & 1)
                        again<T, TR, DROP>(a, bits, trow + (uint32_t)(column + g * 16), m0 + g * 16, f, lane, bias);
                }
            };
            auto finish = [&](int g, int gid, uint32_t keep, float (&v)[16]) {
                finish_rows<T, TR>(a, rows, g, gid, m0 + g * 16, f, keep, bias, v);
            };
            auto keep_of = [&](int g, int gid) {
                return DROP && gid != kNone ? keep_columns(a, m0 + g * 16, f, lane, key) : 0xFFFFu;
            };
            auto wait_sum = [&](int i) {   // of accumulator i
                bool w = true;
                if (lane == 0) w = tc::mbar_wait(&accf[i], u.phase(i), err, tc::TC_ERR_WAIT_ACC);
                const bool got = __shfl_sync(0xffffffffu, w ? 1 : 0, 0) != 0;
                tc::tc_fence_after();
                return got;
            };
            auto release = [&](int i) {
                tc::tc_fence_before();
                __syncwarp();
                if (lane == 0) tc::mbar_arrive_cluster(lead[i]);
                u.used(i);
            };
            if constexpr (LONG) {
                constexpr int NG = (kMaxColumns<T, DROP> / 16 + HG - 1) / HG;   // this warp's column groups
                uint32_t powers = 0;
                if (F16 && (DROP || own)) powers = (uint32_t)load_powers<NG, HG>(a, m0, h, lane);
                float v[NG][16] = {};
                uint32_t keep[NG];
                int buf = 0;
                for (int s = 0; s < sums; ++s) {
                    buf = u.next<B>();
                    ok = wait_sum(buf);
                    if (!ok) break;
#pragma unroll
                    for (int i = 0; i < NG; ++i) {
                        const int g = h + HG * i;
                        if (g * 16 >= a.np) break;
                        // (8 at a time: registers)
                        uint32_t x[8];
#pragma unroll
                        for (int o = 0; o < 16; o += 8) {
                            tc::tmem_ld8_nowait(trow + (uint32_t)(buf * a.np + g * 16 + o), x);
                            tc::tmem_wait_ld();
#pragma unroll
                            for (int j = 0; j < 8; ++j) v[i][o + j] += __uint_as_float(x[j]);
                        }
                    }
                    if (s + 1 < sums || own) release(buf);
                }
                if (ok && own) ok = wait_sum(buf ^ 1);
                if (!ok) break;
                const int low = own ? buf ^ 1 : buf, lowc = (DROP ? B : low) * a.np;
#pragma unroll
                for (int i = 0; i < NG; ++i) {
                    const int g = h + HG * i;
                    if (g * 16 >= a.np) break;
                    const int gid = __shfl_sync(0xffffffffu, rows.gid, g);
                    keep[i] = keep_of(g, gid);
                    if (!(DROP ? by_mma(gid) : apart<T>(gid))) continue;
                    uint32_t x[8];
                    if (gid == kMixed) {
                        bool b = false;
#pragma unroll
                        for (int o = 0; o < 16; o += 8) {
                            tc::tmem_ld8_nowait(trow + (uint32_t)(lowc + g * 16 + o), x);
                            tc::tmem_wait_ld();
#pragma unroll
                            for (int j = 0; j < 8; ++j) b |= !isfinite(__uint_as_float(x[j]));
                        }
                        if (__any_sync(0xffffffffu, b)) {   // the shared sums take its place, for again()
                            bad |= 1u << g;
                            tc::tmem_st16(trow + (uint32_t)(lowc + g * 16), v[i]);
                            continue;
                        }
                    }
#pragma unroll
                    for (int o = 0; o < 16; o += 8) {
                        tc::tmem_ld8_nowait(trow + (uint32_t)(lowc + g * 16 + o), x);
                        tc::tmem_wait_ld();
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            if (F16) x[j] = times_power(x[j], powers >> 8 * i, o + j);
                            if (keep[i] >> (o + j) & 1) v[i][o + j] += __uint_as_float(x[j]);
                        }
                    }
                }
                if (!bad) release(low);
#pragma unroll
                for (int i = 0; i < NG; ++i) {
                    const int g = h + HG * i;
                    if (g * 16 >= a.np) break;
                    finish(g, __shfl_sync(0xffffffffu, rows.gid, g), keep[i], v[i]);
                }
                if (bad) {
                    finish_again(lowc);
                    release(low);
                }
            } else {
                // the masks before the sums are there: 16 bits a group, the first lowest
                uint32_t kept[kMaxGroups / 2] = {};
                auto turn = [&](uint32_t in) {
#pragma unroll
                    for (int i = 0; i < kMaxGroups / 2; ++i)
                        kept[i] = __funnelshift_r(kept[i], i + 1 < kMaxGroups / 2 ? kept[i + 1] : in, 16);
                };
                if (DROP)
#pragma unroll 1
                    for (int i = 0; i < kMaxGroups; ++i) {
                        const int g = h + HG * i;
                        turn(g * 16 < a.np ? keep_of(g, __shfl_sync(0xffffffffu, rows.gid, g & 31)) : 0u);
                    }
                static_assert(HG == 2, "load_powers");
                uint64_t powers = 0;
                if (F16 && (DROP || own)) powers = load_powers<8, 2>(a, m0, h, lane);
                const int buf = u.next<B>();
                ok = wait_sum(buf) && (!own || wait_sum(buf ^ 1));
                if (!ok) break;
                const uint32_t xcol = trow + (uint32_t)(buf * a.np), ycol = trow + (uint32_t)((DROP ? B : buf ^ 1) * a.np);
                uint32_t x[16], y[16];
                float v[16];
                auto sums_of = [&](int g, bool low) {
                    tc::tmem_ld16_nowait(xcol + (uint32_t)(g * 16), x);
                    if (low) tc::tmem_ld16_nowait(ycol + (uint32_t)(g * 16), y);
                    tc::tmem_wait_ld();
                };
                auto broken = [&]() {
                    bool b = false;
#pragma unroll
                    for (int j = 0; j < 16; ++j) b |= !isfinite(__uint_as_float(y[j]));
                    return __any_sync(0xffffffffu, b) != 0;
                };
                if (own) {
                    // the low-rank products that stand apart to the sums, so that the MMAs go on
#pragma unroll 1
                    for (int g = h; g * 16 < a.np; g += HG) {
                        const int gid = __shfl_sync(0xffffffffu, rows.gid, g);
                        if (apart<T>(gid)) {
                            sums_of(g, true);
                            if (F16)
#pragma unroll
                                for (int j = 0; j < 16; ++j) y[j] = times_power(y[j], (uint32_t)powers, j);
                            if (gid == kMixed && broken()) {
                                bad |= 1u << g;
                            } else {
#pragma unroll
                                for (int j = 0; j < 16; ++j) v[j] = __uint_as_float(x[j]) + __uint_as_float(y[j]);
                                tc::tmem_st16(xcol + (uint32_t)(g * 16), v);
                            }
                        }
                        if (F16) powers >>= 8;
                    }
                    release(buf ^ 1);
                }
#pragma unroll 1
                for (int g = h; g * 16 < a.np; g += HG) {   // 16 columns at a time
                    const int gid = __shfl_sync(0xffffffffu, rows.gid, g);
                    const bool low = DROP && by_mma(gid);
                    sums_of(g, low);
                    const uint32_t keep = DROP ? kept[0] & 0xFFFFu : 0xFFFFu;
                    if (DROP) turn(0);
                    if (DROP && F16) {
#pragma unroll
                        for (int j = 0; j < 16; ++j) y[j] = times_power(y[j], (uint32_t)powers, j);
                        powers >>= 8;
                    }
                    if (low && gid == kMixed && broken()) bad |= 1u << g;
                    if (bad >> g & 1) continue;
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        v[j] = __uint_as_float(x[j]);
                        if (low && (keep >> j & 1)) v[j] += __uint_as_float(y[j]);
                    }
                    finish(g, gid, keep, v);
                }
                if (bad) finish_again(buf * a.np);
                release(buf);
            }
        }
    }
    tc::tc_fence_before();
    __syncthreads();
    tc::cluster_sync();   // no CTA leaves while its peer's MMAs, copies or arrivals may reach it
    tc::tc_fence_after();
    if (threadIdx.x == 0) report(gave_up);
    if (warp == 1) tc::tmem_dealloc_pair(tbase, 512);
}

// ── few tiles: one tile of 128 features x np rows a cluster, its K loop split over the
// cluster's CTAs. Each CTA sends its fp32 partial columns to the CTA that finishes them (qpo
// quads of columns each) through distributed shared memory; they are summed in CTA order. Bound by
// reading W once: every SM has a TMA ring of its own share of K in flight. One token of 4096 x 4096
// bf16 (34 MB) 14 us beside a thin product of 5.6 that it overlaps (15.2 in all); 64 tokens of 32 requests x
// 4096 x 8192 (81 MB) 24 (28.4).
template <class T, bool TR, bool DROP, bool LONG>
__global__ void __launch_bounds__(kThreads, 1)
    project_split_kernel(const __grid_constant__ CUtensorMap mW, const __grid_constant__ CUtensorMap mZ,
                         const __grid_constant__ CUtensorMap mQ, const __grid_constant__ CUtensorMap mT,
                         const __grid_constant__ PArgs a) {
    constexpr bool F16 = std::is_same<T, __half>::value;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = align1024(smem_raw);
    __shared__ uint64_t full[kMaxStages], empty[kMaxStages], accf[2], acce[2], mdone;
    __shared__ uint32_t tslot;
    __shared__ int gave_up;
    __shared__ Runs runs[2];
    int* err = &gave_up;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const bool leader = tc::elect_one();
    const int split = blockIdx.x % a.splits, tile = blockIdx.x / a.splits;
    const int ft = tile % a.n_ft, m0 = (tile / a.n_ft) * a.np, f0 = ft * 128;
    const int stage_bytes = kTileA + a.np * 128;
    const int groups = a.np / 16;
    float4* recv = reinterpret_cast<float4*>(smem + a.stages * stage_bytes);   // [splits][qpo][128]
    // this CTA's chunks of K, in each pass
    const int k_lo = split * a.kchunks / a.splits, k_n = (split + 1) * a.kchunks / a.splits - k_lo;
    const int steps = a.n_terms * k_n;

    // one sum in TMEM, or two in turn, and the low-rank product
    constexpr int kLow = LONG ? 256 : 128, kColumns = 2 * kLow;
    const int sums = LONG ? (steps + kPromote<T> - 1) / kPromote<T> : 1;
    // The ring's barriers are this CTA's own: its first loads go out before the cluster meets. (A
    // few: the TMA unit takes more only at the pace of memory, and the others wait here.)
    const int head = min(min(steps, a.stages), 2);
    if (warp == 0 && leader) {
        for (int s = 0; s < a.stages; ++s) {
            tc::mbar_init(&full[s], 1);
            tc::mbar_init(&empty[s], 1);
        }
        for (int s = 0; s < 2; ++s) {
            tc::mbar_init(&accf[s], 1);
            tc::mbar_init(&acce[s], kThreads / 32 - 2);
        }
        tc::mbar_init(&mdone, 1);
        gave_up = tc::TC_OK;
        tc::fence_barrier_init();
        tc::fence_async_shared();
        for (int c = 0; c < head; ++c) {
            const int t = c / k_n, k = (k_lo + c - t * k_n) * 64;
            tc::mbar_arrive_expect_tx(&full[c], stage_bytes);
            load_stage<TR, false>(smem + c * stage_bytes, &mW, &mZ, &full[c], 0, f0, k, a.wp[t], k, m0, a.zp[t]);
        }
    }
    if (warp == 1) {
        tc::tmem_alloc(&tslot, kColumns);
        tc::tmem_relinquish();
    }
    tc::tc_fence_before();
    __syncthreads();
    tc::cluster_sync();   // every CTA of the cluster runs before any writes to its shared memory
    tc::tc_fence_after();
    const uint32_t tbase = tslot, de = tbase + kLow;

    // epilogue state that outlives the cluster barrier
    const int q = warp & 3, h = (warp - 2) >> 2;
    const int f = f0 + q * 32 + lane;
    // Of the quads of columns that this CTA finishes, this warp has every second one.
    const int quad0 = split * a.qpo, quads = min(a.qpo, a.np / 4 - quad0);
    float4* low = recv + a.splits * a.qpo * 128 + q * 32 + lane;   // [quad][128]: this thread's own
    float bias = 0.f;
    TileRows rows = {};

    if (warp == 0) {
        Ring r;
        for (int c = 0; c < head; ++c) r.next(a.stages);
        int issued = head;
        bool ok = true;
        auto stage = [&](const CUtensorMap* mA, const CUtensorMap* mB, int ka, int pa, int kb, int row, int pb) {
            if (!wait_for<LONG>(&empty[r.slot], r.phase ^ 1, err, tc::TC_ERR_WAIT_EMPTY)) return false;
            tc::mbar_arrive_expect_tx(&full[r.slot], stage_bytes);
            load_stage<TR, false>(smem + r.slot * stage_bytes, mA, mB, &full[r.slot], 0, f0, ka, pa, kb, row, pb);
            r.next(a.stages);
            ++issued;
            return true;
        };
        if (leader)
            for (int c = head; ok && c < steps; ++c) {
                const int t = c / k_n, k = (k_lo + c - t * k_n) * 64;
                ok = stage(&mW, &mZ, k, a.wp[t], k, m0, a.zp[t]);
            }
        __syncwarp();
        tc::grid_dependency_wait();
        if (split == 0) {
            const TileRows rows = tile_rows<16>(load_rows(a, m0, lane));
            const int n_runs = find_runs<T, 16>(runs[0], rows, groups, lane);
            if (leader)
                for (int i = 0; ok && i < n_runs; ++i) {
                    const Run u = runs[0][i];
                    for (int e = 0; ok && e < a.n_ext; ++e) {
                        const ExtStage& x = a.ext[e];
                        ok = stage(&mQ, &mT, x.rank0, x.plane * a.adapters + u.ad, u.slot * a.part_cols + x.col0,
                                   m0 + u.c0, 0);
                    }
                }
        }
        if (!ok && leader) {
            const int first = issued > a.stages ? issued - a.stages : 0;
            for (int i = first; i < issued; ++i)
                tc::mbar_wait(&full[i % a.stages], (i / a.stages) & 1, nullptr, tc::TC_ERR_DRAIN);
        }
    } else if (warp == 1) {
        Ring r;
        bool ok = true;
        if (leader) {
            const uint32_t idesc = idesc_n(a.idesc, a.np);
            for (int s = 0; ok && s < sums; ++s) {
                const int n = LONG ? min(steps - s * kPromote<T>, kPromote<T>) : steps;
                const uint32_t d = tbase + (uint32_t)((s & 1) * 128);
                if (LONG && s >= 2) ok = wait_for<LONG>(&acce[s & 1], (s / 2 - 1) & 1, err, tc::TC_ERR_WAIT_ACC);
                for (int c = 0; ok && c < n; ++c) {
                    ok = tc::mbar_wait(&full[r.slot], r.phase, err, tc::TC_ERR_WAIT_FULL);
                    if (!ok) break;
                    tc::tc_fence_after();
                    const uint32_t base = tc::smem_u32(smem + r.slot * stage_bytes);
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        mma<false>(d, desc_a<TR>(base, k), tc::desc_kmajor_sw128(base + kTileA + k * 32), idesc,
                                   (c | k) != 0);
                    commit<false>(&empty[r.slot]);
                    r.next(a.stages);
                }
                if (ok && s + 1 < sums) commit<false>(&accf[s & 1]);
            }
        }
        __syncwarp();
        tc::grid_dependency_wait();
        if (split == 0) {
            const TileRows rows = tile_rows<16>(load_rows(a, m0, lane));
            const int n_runs = find_runs<T, 16>(runs[1], rows, groups, lane);
            if (leader)
                for (int i = 0; ok && i < n_runs; ++i) {
                    const Run u = runs[1][i];
                    const uint32_t idesc = idesc_n(a.idesc, u.cols);
                    const bool alone = DROP || u.own;   // in an accumulator of its own
                    const uint32_t d = (alone ? de : tbase + (LONG ? (uint32_t)((sums - 1) & 1) * 128 : 0u)) + (uint32_t)u.c0;
                    for (int e = 0; e < a.n_ext; ++e) {
                        const ExtStage& x = a.ext[e];
                        ok = tc::mbar_wait(&full[r.slot], r.phase, err, tc::TC_ERR_WAIT_FULL);
                        if (!ok) break;
                        tc::tc_fence_after();
                        const uint32_t base = tc::smem_u32(smem + r.slot * stage_bytes);
                        for (int k = 0; k < x.n; ++k)
                            mma<false>(d, desc_a<TR>(base, x.a[k]),
                                       tc::desc_kmajor_sw128(base + kTileA + x.b[k] * 32), idesc,
                                       !alone || !u.first || (e | k) != 0);
                        commit<false>(&empty[r.slot]);
                        r.next(a.stages);
                    }
                }
        }
        if (leader) {   // also after an error: whatever was issued completes
            if (ok) commit<false>(&accf[(sums - 1) & 1]);
            commit<false>(&mdone);
            tc::mbar_wait(&mdone, 0, nullptr, tc::TC_ERR_DRAIN);
        }
    } else {
        // The adapters of this CTA's rows, lane l those of columns l, l + 32, .., and the rows of Q
        // that the CUDA cores may need, towards L2 before W's stream fills the queues there (behind
        // it a load takes some 3 us).
        int col_ad[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int m = m0 + quad0 * 4 + lane + 32 * i;
            col_ad[i] = lane + 32 * i < quads * 4 && m < a.rows ? row_adapter(a, m) : -1;
        }
        auto ad_of = [&](int c) {   // of this CTA's column c
            const int x = c < 32 ? col_ad[0] : c < 64 ? col_ad[1] : c < 96 ? col_ad[2] : col_ad[3];
            return __shfl_sync(0xffffffffu, x, c & 31);
        };
        if (!TR && a.splits > 1)
            for (int c = h * 4; c < quads * 4; c += 8)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int ad = ad_of(c + j);
                    if (ad >= 0 && f < a.feats) tc::prefetch_l2((const T*)a.Q + ((int64_t)ad * a.feats + f) * a.rank);
                }
        // Many sums as they come: the first half of them before anything that waits for the kernel before, the
        // others but the last one after it.
        constexpr int NG = 4;   // this warp's groups, at most
        const uint32_t trow = tbase + ((uint32_t)(q * 32) << 16);
        float acc[LONG ? NG : 1][16] = {};
        auto wait_sum = [&](int s) {
            bool w = true;
            if (lane == 0) w = tc::mbar_wait(&accf[s & 1], (s >> 1) & 1, err, tc::TC_ERR_WAIT_ACC);
            const bool got = __shfl_sync(0xffffffffu, w ? 1 : 0, 0) != 0;
            tc::tc_fence_after();
            return got;
        };
        bool ok = true;
        auto take_sums = [&](int first, int end) {
            if constexpr (LONG) {
#pragma unroll 1
                for (int s = first; ok && s < end; ++s) {
                    ok = wait_sum(s);
                    if (!ok) break;
#pragma unroll
                    for (int i = 0; i < NG; ++i) {
                        const int g = h + 2 * i;
                        if (g >= groups) break;
                        uint32_t x[16];
                        tc::tmem_ld16_nowait(trow + (uint32_t)((s & 1) * 128 + g * 16), x);
                        tc::tmem_wait_ld();
#pragma unroll
                        for (int j = 0; j < 16; ++j) acc[i][j] += __uint_as_float(x[j]);
                    }
                    tc::tc_fence_before();
                    __syncwarp();
                    if (lane == 0) tc::mbar_arrive(&acce[s & 1]);
                }
            }
        };
        take_sums(0, sums / 2);
        tc::grid_dependency_wait();
        const RngKey key = DROP ? load_rng(a.rng) : RngKey{};
        rows = tile_rows<16>(load_rows(a, m0, lane));
        bias = a.bias && f < a.feats ? to_f(((const T*)a.bias)[f]) : 0.f;
        if (a.splits > 1)   // the rows' t into L1, a load for every 32 bytes, all in flight
            for (int r = 0; r < a.rank; r += 8)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int64_t m = m0 + quad0 * 4 + lane + 32 * i;
                    const float touch = col_ad[i] >= 0 ? a.t[m * a.rank + r] : 0.f;
                    asm volatile("" ::"f"(touch));
                }
        // products for the CUDA cores, made while the K loop runs
        if (a.splits > 1)
#pragma unroll 1
            for (int i = h; i < quads; i += 2) {
                const int quad = quad0 + i;
                if (__shfl_sync(0xffffffffu, rows.gid, quad >> 2) != kMany) continue;
                int ad[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) ad[j] = ad_of(i * 4 + j);
                quad_products<T, TR, DROP>(a, m0 + quad * 4, make_int4(ad[0], ad[1], ad[2], ad[3]), f, low + i * 128);
            }
        uint32_t powers = 0;
        if (F16 && split == 0) powers = (uint32_t)load_powers<NG, 2>(a, m0, h, lane);
        take_sums(sums / 2, sums - 1);
        if (ok && wait_sum(sums - 1)) {
            const int last = LONG ? ((sums - 1) & 1) * 128 : 0;
            const uint32_t mine = tc::smem_u32(recv) + (uint32_t)((split * a.qpo * 128 + q * 32 + lane) * 16);
#pragma unroll(LONG ? NG : 1)
            for (int i = 0; i < NG; ++i) {
                const int g = h + 2 * i;
                if (g >= groups) break;
                uint32_t v[16], y[16];
                const int gid = __shfl_sync(0xffffffffu, rows.gid, g);
                const uint32_t live = __shfl_sync(0xffffffffu, rows.rows, g) & 0xFFFFu;
                const bool ext = split == 0 && (DROP ? by_mma(gid) : apart<T>(gid));
                const uint32_t low_at = trow + (uint32_t)(kLow + g * 16);
                tc::tmem_ld16_nowait(trow + (uint32_t)(last + g * 16), v);
                if (ext) tc::tmem_ld16_nowait(low_at, y);
                tc::tmem_wait_ld();
                uint32_t keep = 0xFFFFu;
                if (DROP && (ext || (a.splits == 1 && gid == kMany))) keep = keep_columns(a, m0 + g * 16, f, lane, key);
                float s[16];
#pragma unroll
                for (int j = 0; j < 16; ++j) s[j] = (LONG ? acc[LONG ? i : 0][j] : 0.f) + __uint_as_float(v[j]);
                if (ext) {
                    bool b = false;
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        if (F16) y[j] = times_power(y[j], powers, j);
                        b |= !isfinite(__uint_as_float(y[j]));
                    }
                    if (gid == kMixed && __any_sync(0xffffffffu, b)) {
                        repair<T, TR>(a, live, low_at, m0 + g * 16, f);
                        tc::tmem_ld16_nowait(low_at, y);
                        tc::tmem_wait_ld();
                    }
#pragma unroll
                    for (int j = 0; j < 16; ++j)
                        if (keep >> j & 1) s[j] += __uint_as_float(y[j]);
                }
                if (F16) powers >>= 8;
                if (a.splits == 1) {   // nothing to join
                    finish_rows<T, TR>(a, rows, g, gid, m0 + g * 16, f, keep, bias, s);
                    continue;
                }
                int to = g * 4 / a.qpo, at = g * 4 - to * a.qpo;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    tc::st_cluster_v4(tc::map_shared(mine + (uint32_t)(at * 2048), to),
                                      make_float4(s[4 * j], s[4 * j + 1], s[4 * j + 2], s[4 * j + 3]));
                    if (++at == a.qpo) {
                        at = 0;
                        ++to;
                    }
                }
            }
        }
    }
    tc::tc_fence_before();
    __syncthreads();
    tc::cluster_sync();
    tc::tc_fence_after();
    if (threadIdx.x == 0) report(gave_up);
    if (warp == 1) tc::tmem_dealloc(tbase, kColumns);
    if (warp >= 2 && a.splits > 1) {
        const bool live_f = f < a.feats;
#pragma unroll 1
        for (int i = h; i < quads; i += 2) {
            const int quad = quad0 + i, gid = __shfl_sync(0xffffffffu, rows.gid, quad >> 2);
            const uint32_t bits = __shfl_sync(0xffffffffu, rows.rows, quad >> 2) >> (quad & 3) * 4;
            if (!live_f) continue;
            float4 v = recv[i * 128 + q * 32 + lane];
            for (int k = 1; k < a.splits; ++k) {
                const float4 w = recv[(k * a.qpo + i) * 128 + q * 32 + lane];
                v.x += w.x;
                v.y += w.y;
                v.z += w.z;
                v.w += w.w;
            }
            if (gid == kMany) {
                const float4 w = low[i * 128];
                v.x += w.x;
                v.y += w.y;
                v.z += w.z;
                v.w += w.w;
            }
            const float s[4] = {v.x, v.y, v.z, v.w};
            T* o = (T*)a.out + (int64_t)(m0 + quad * 4) * a.ldo + f;
            if ((bits & 0xFu) == 0xFu) {
#pragma unroll
                for (int j = 0; j < 4; ++j, o += a.ldo) *o = from_f<T>(s[j] + bias);
                continue;
            }
#pragma unroll
            for (int j = 0; j < 4; ++j, o += a.ldo) {
                if (bits >> j & 1) *o = from_f<T>(s[j] + bias);
                else if (a.zero_padding && (bits >> (16 + j) & 1)) *o = from_f<T>(0.f);
            }
        }
    }
}

// ── operands laid out for TMA: rows on 16-byte boundaries, fp32 as three bf16 planes
struct Layout {
    const void* src;
    int64_t lds;
    void* dst;
    int64_t rows;
    int cols, ldd;
    int64_t first;     // first unit (8 columns of a row) of this operand in the launch
};
struct Layouts {
    Layout j[4];
    int n;
    int64_t units;
};

template <class T>
__global__ void layout_kernel(const __grid_constant__ Layouts L) {
    const int64_t u = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (u >= L.units) return;
    int at = 0;
    for (int i = 1; i < L.n; ++i)
        if (u >= L.j[i].first) at = i;
    const Layout& j = L.j[at];
    const int per = j.ldd / 8;
    const int64_t row = (u - j.first) / per;
    const int c = (int)((u - j.first) - row * per) * 8;
    const T* s = (const T*)j.src + row * j.lds + c;
    if constexpr (sizeof(T) == 4) {
        __nv_bfloat16 p[3][8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            float v = c + i < j.cols ? s[i] : 0.f;
#pragma unroll
            for (int k = 0; k < 3; ++k) {
                // rounded to nearest, but not over the range's end; a number that is not
                // finite has no remainder
                __nv_bfloat16 b = __float2bfloat16_rn(v);
                if (isinf(__bfloat162float(b)) && isfinite(v)) b = __float2bfloat16_rz(v);
                p[k][i] = b;
                v = isfinite(v) ? v - __bfloat162float(b) : 0.f;
            }
        }
        __nv_bfloat16* d = (__nv_bfloat16*)j.dst + row * j.ldd + c;
#pragma unroll
        for (int k = 0; k < 3; ++k)
            *reinterpret_cast<uint4*>(d + k * j.rows * j.ldd) = *reinterpret_cast<uint4*>(p[k]);
    } else {
        T p[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) p[i] = c + i < j.cols ? s[i] : from_f<T>(0.f);
        *reinterpret_cast<uint4*>((T*)j.dst + row * j.ldd + c) = *reinterpret_cast<uint4*>(p);
    }
}

// ── host side
PFN_cuTensorMapEncodeTiled_v12000 encode() {
    static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
    });
    if (!fn) fail("multilora", "cuTensorMapEncodeTiled is unavailable");
    return fn;
}

struct Operands {
    Operand z, W, Q, P;
    int64_t bytes() const { return z.bytes + W.bytes + Q.bytes + P.bytes; }
};
Operands operands(const ProjectTc& p) {
    Operands o;
    const bool tr = p.transposed, f32 = p.dtype == DT_F32;
    // (fp32's planes of z are for the wide product and the thin one of tiles; rows read z as it is)
    if (!f32 || p.out || p.P) o.z = operand(p.z, p.ldz, p.rows, p.width, f32, false);
    if (p.out) {
        const int64_t q_rows = (int64_t)p.adapters * (tr ? p.rank : p.feats);
        o.W = operand(p.W, tr ? p.feats : p.width, tr ? p.width : p.feats, tr ? p.feats : p.width, f32, false);
        o.Q = operand(p.Q, tr ? p.feats : p.rank, q_rows, tr ? p.feats : p.rank, f32, false);
    }
    if (p.P) {
        const int64_t p_rows = (int64_t)p.adapters * (tr ? p.width : p.rank);
        // (transposed, the thin kernels take its rows of ranks in pieces of 8 or 2)
        o.P = operand(p.P, tr ? p.rank : p.width, p_rows, tr ? p.rank : p.width, f32, tr);
    }
    return o;
}
void place(Operands& o, void* scratch) {
    char* at = (char*)scratch;
    for (Operand* x : {&o.z, &o.W, &o.Q, &o.P})
        if (x->moved) {
            x->p = at;
            at += x->bytes;
        }
}

// dims (innermost first) of 16-bit numbers, box {64, box1, 1}, 128-byte swizzle
CUtensorMap tensor_map(const void* base, int dtype, uint64_t d0, uint64_t d1, uint64_t d2, int64_t ld1, int64_t ld2,
                       int box1) {
    CUtensorMap m;
    cuuint64_t dims[3] = {d0, d1, d2};
    cuuint64_t strides[2] = {(cuuint64_t)ld1 * 2, (cuuint64_t)ld2 * 2};
    cuuint32_t box[3] = {64, (cuuint32_t)box1, 1};
    cuuint32_t estr[3] = {1, 1, 1};
    const auto type = dtype == DT_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    const CUresult rc = encode()(&m, type, 3, const_cast<void*>(base), dims, strides, box, estr,
                                 CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                                 CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (rc != CUDA_SUCCESS) fail("multilora", "cuTensorMapEncodeTiled failed (" + std::to_string((int)rc) + ")");
    return m;
}

int sm_count() {
    static std::atomic<int> n[64] = {};
    int dev = 0;
    BSML_CUDA(cudaGetDevice(&dev));
    int v = dev < 64 ? n[dev].load() : 0;
    if (v == 0) {
        BSML_CUDA(cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, dev));
        if (dev < 64) n[dev].store(v);
    }
    return v;
}

template <class K>
void launch(K kernel, int grid, int threads, int cluster, int smem, cudaStream_t st, const CUtensorMap (&m)[4],
            const PArgs& a) {
    // the limit belongs to the kernel, not to the call: every call sets the same one, so that calls
    // from several host threads do not lower each other's
    BSML_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kDynMax));
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    ::bsml::count_launch();
    BSML_CUDA(cudaLaunchKernelEx(&cfg, kernel, m[0], m[1], m[2], m[3], a));
}

// The plane products of the low-rank stages, smallest first: a stage is 64 ranks of a plane of Q and 64 columns of
// the parts, which hold several parts where the ranks are few.
void make_ext(PArgs& a, const LowParts& lp, int planes) {
    const int blocks = (int)ceil_div(a.rank, 64);
    a.n_ext = 0;
    for (int q = planes - 1; q >= 0; --q)
        for (int b = 0; b < blocks; ++b)
            for (int i = (planes == 1 ? lp.n : lp.n - q) - 1; i >= 0; --i) {   // fp32: plane q meets parts 0 .. 2 - q
                const int col = i * lp.pitch + b * 64, col0 = col / 64 * 64;
                ExtStage* x = a.n_ext ? &a.ext[a.n_ext - 1] : nullptr;
                if (!x || x->plane != q || x->rank0 != b * 64 || x->col0 != col0) {
                    x = &a.ext[a.n_ext++];
                    *x = ExtStage{};
                    x->plane = (int8_t)q;
                    x->rank0 = (int16_t)(b * 64);
                    x->col0 = (int16_t)col0;
                }
                const int steps = (int)ceil_div(std::min(a.rank - b * 64, 64), 16);
                for (int s = 0; s < steps; ++s) {
                    x->a[x->n] = (int8_t)s;
                    x->b[x->n] = (int8_t)(s + (col - col0) / 16);
                    ++x->n;
                }
            }
}

// The launch of a plan made as far as split or pairs (run).
template <class T, bool TR, bool DROP, bool LONG>
void run_sums(const ProjectTc& p, const Operands& o, PArgs& a, bool split, int sms, cudaStream_t st) {
    if (!split) {
        a.n_ft = (int)ceil_div(p.feats, 256);
        // Columns a tile (steps of 32, an MMA's over a pair): the fewest cycles of a pair's turns,
        // about 1.1 a step of K for each of the 256 features and np rows that it loads (L2 bounds the
        // main loop), and for a tile's end 2500, and 30 a row where no second sum hides the epilogue.
        const int pairs = sms / 2;
        const int64_t steps = (int64_t)a.kchunks * a.n_terms;
        int64_t best = -1;
        for (int np = kMaxColumns<T, DROP>; np >= 96; np -= 32) {
            const int64_t turns = ceil_div(ceil_div(p.rows, np) * a.n_ft, pairs);
            const int64_t cost = turns * ((np + 256) * steps * 11 / 10 + 2500 + (kSums<T, DROP> == 1 ? 30 * np : 0));
            if (best < 0 || cost < best) {
                best = cost;
                a.np = np;
            }
        }
        a.n_mt = (int)ceil_div(p.rows, a.np);
        a.np = (int)round_up(ceil_div(p.rows, a.n_mt), 32);
        a.splits = 1;
    }
    const int nb = split ? a.np : a.np / 2;   // rows of z a CTA loads
    const int stage = kTileA + nb * 128;
    // the join's partial sums, and the CUDA cores' products beside them
    const int recv = split && a.splits > 1 ? (a.splits + 1) * a.qpo * 2048 : 0;
    a.stages = std::min(kMaxStages, (kDynMax - 1024 - recv) / stage);
    const int smem = a.stages * stage + recv + 1024;
    a.idesc = tc::make_idesc(p.dtype == DT_F16 ? 0u : 1u, TR ? 1u : 0u, 0u, split ? 128 : 256, 0);

    const int wd = p.dtype;
    CUtensorMap m[4];
    if (TR) {
        m[0] = tensor_map(o.W.p, wd, p.feats, p.width, o.W.planes, o.W.ld, o.W.rows * o.W.ld, 64);
        m[2] = tensor_map(o.Q.p, wd, p.feats, p.rank, o.Q.planes * p.adapters, o.Q.ld, p.rank * o.Q.ld, 64);
    } else {
        m[0] = tensor_map(o.W.p, wd, p.width, p.feats, o.W.planes, o.W.ld, o.W.rows * o.W.ld, 128);
        m[2] = tensor_map(o.Q.p, wd, p.rank, p.feats, o.Q.planes * p.adapters, o.Q.ld, p.feats * o.Q.ld, 128);
    }
    m[1] = tensor_map(o.z.p, wd, p.width, p.rows, o.z.planes, o.z.ld, o.z.rows * o.z.ld, nb);
    const int64_t pc = (int64_t)kPartSlots * a.part_cols;
    m[3] = tensor_map(p.low.parts, wd, pc, p.rows, 1, pc, p.rows * pc, nb);
    if (split) {
        launch(project_split_kernel<T, TR, DROP, LONG>, a.n_ft * a.n_mt * a.splits, kThreads, a.splits, smem, st, m, a);
    } else {
        const int pairs = (int)std::min<int64_t>(sms / 2, (int64_t)a.n_ft * a.n_mt);
        launch(project_pair_kernel<T, TR, DROP, LONG>, 2 * pairs, 64 + 32 * kPairEpi<LONG>, 2, smem, st, m, a);
    }
}
template <class T, bool TR, bool DROP>
void run(const ProjectTc& p, const Operands& o, cudaStream_t st) {
    PArgs a = {};
    a.rows = p.rows; a.feats = p.feats; a.rank = p.rank; a.adapters = p.adapters;
    a.kchunks = (int)ceil_div(p.width, 64);
    if (p.dtype == DT_F32) {
        const int8_t zs[6] = {1, 0, 2, 0, 1, 0}, ws[6] = {1, 2, 0, 1, 0, 0};
        a.n_terms = 6;
        std::copy(zs, zs + 6, a.zp);
        std::copy(ws, ws + 6, a.wp);
    } else {
        a.n_terms = 1;
    }
    const LowParts lp = low_parts(p.rank, p.dtype);
    make_ext(a, lp, p.dtype == DT_F32 ? 3 : 1);
    a.ids = p.ids; a.groups = p.low.groups; a.power = p.low.power; a.t = p.low.t;
    a.Q = p.Q; a.bias = p.bias;
    a.part_cols = lp.cols;
    a.drop = p.drop; a.rng = p.rng; a.zero_padding = p.zero_padding;
    a.q_vec = !TR && (reinterpret_cast<uintptr_t>(p.Q) & 15) == 0 && (p.rank * sizeof(T)) % 16 == 0;
    a.t_vec = (reinterpret_cast<uintptr_t>(p.low.t) & 15) == 0 && p.rank % 4 == 0;
    a.out = p.out; a.ldo = p.ldo;

    const int sms = sm_count();
    // Split kernel while its tiles (128 features x at most 128 rows) leave SMs idle; else pairs.
    // (tiles start at multiples of 32 rows, so one of 16 columns is the only one)
    int np_s = p.rows <= 16 ? 16 : (int)round_up(ceil_div(p.rows, ceil_div(p.rows, 128)), 32);
    const int64_t fts = ceil_div(p.feats, 128);
    const bool split = fts * ceil_div(p.rows, np_s) <= sms;
    // more than half the SMs busy with whole K loops: narrower tiles rather than idle SMs
    if (2 * fts * ceil_div(p.rows, np_s) > sms)
        while (np_s > 32 && fts * ceil_div(p.rows, np_s - 32) <= sms) np_s -= 32;
    const int64_t tiles_s = fts * ceil_div(p.rows, np_s);
    if (split) {
        a.np = np_s;
        a.n_ft = (int)ceil_div(p.feats, 128);
        a.n_mt = (int)ceil_div(p.rows, np_s);
        // (two chunks of K a CTA at least, over the passes)
        const int most = a.n_terms > 1 ? a.kchunks : a.kchunks / 2;
        a.splits = (int)std::max<int64_t>(1, std::min<int64_t>({8, sms / tiles_s, most}));
        a.qpo = (int)ceil_div(a.np / 4, a.splits);
    }
    // Sums longer than an accumulator's? (Of fp32's passes only the last adds numbers of the sum's own size.)
    if (ceil_div(a.kchunks, split ? a.splits : 1) > kPromote<T>) run_sums<T, TR, DROP, true>(p, o, a, split, sms, st);
    else run_sums<T, TR, DROP, false>(p, o, a, split, sms, st);
}

template <class T>
void run_type(const ProjectTc& p, const Operands& o, cudaStream_t st) {
    if (!p.transposed) run<T, false, false>(p, o, st);
    else if (p.drop.thr == 0) run<T, true, false>(p, o, st);
    else run<T, true, true>(p, o, st);
}

}  // namespace

LowParts low_parts(int rank, int dtype) {
    LowParts l;
    l.n = dtype == DT_F16 ? 2 : 3;
    l.pitch = rank <= 16 ? 16 : rank <= 32 ? 32 : (int)round_up(rank, 64);   // no part over a stage's end
    l.cols = (int)round_up(l.n * l.pitch, 64);
    return l;
}

int64_t project_tc_scratch(const ProjectTc& p) { return operands(p).bytes(); }

LaidOut project_tc_prepare(const ProjectTc& p, void* scratch, cudaStream_t st) {
    Operands o = operands(p);
    place(o, scratch);
    Layouts L = {};
    auto add = [&](const Operand& x, const void* src, int64_t lds) {
        if (!x.moved) return;
        Layout& j = L.j[L.n++];
        j.src = src; j.lds = lds; j.dst = const_cast<void*>(x.p);
        j.rows = x.rows; j.cols = x.cols; j.ldd = (int)x.ld;
        j.first = L.units;
        L.units += x.rows * (x.ld / 8);
    };
    add(o.z, p.z, p.ldz);
    add(o.W, p.W, p.transposed ? p.feats : p.width);
    add(o.Q, p.Q, p.transposed ? p.feats : p.rank);
    add(o.P, p.P, p.transposed ? p.rank : p.width);
    LaidOut l;
    l.z = o.z.p; l.ldz = o.z.ld; l.z_plane = o.z.rows * o.z.ld;
    l.P = o.P.p; l.ldp = o.P.ld; l.p_plane = o.P.rows * o.P.ld;
    if (L.n == 0) return l;
    const int64_t blocks = ceil_div(L.units, 256);
    if (blocks > 0x7fffffff) fail("multilora", "operands of more than 2^42 elements");
    ::bsml::count_launch();
    if (p.dtype == DT_F32) layout_kernel<float><<<(unsigned)blocks, 256, 0, st>>>(L);
    else layout_kernel<__half><<<(unsigned)blocks, 256, 0, st>>>(L);   // a copy of 16-bit numbers
    BSML_LAUNCH("multilora layout");
    return l;
}

void project_tc(const ProjectTc& p, void* scratch, cudaStream_t st) {
    Operands o = operands(p);
    place(o, scratch);
    if (p.dtype == DT_F32) run_type<float>(p, o, st);
    else if (p.dtype == DT_BF16) run_type<__nv_bfloat16>(p, o, st);
    else run_type<__half>(p, o, st);
}

__global__ void multilora_wait_selftest_kernel() {
    __shared__ uint64_t bar;
    __shared__ int gave_up;
    if (threadIdx.x == 0) {
        tc::mbar_init(&bar, 1);
        tc::fence_barrier_init();
        gave_up = tc::TC_OK;
        tc::mbar_wait(&bar, 0, &gave_up, tc::TC_ERR_WAIT_FULL);
        report(gave_up);
    }
}

void multilora_wait_selftest(cudaStream_t st) {
    ::bsml::count_launch();
    multilora_wait_selftest_kernel<<<1, 32, 0, st>>>();
    BSML_LAUNCH("multilora_wait_selftest_kernel");
}

int multilora_error_flag() {
    int v = 0, zero = 0;
    BSML_CUDA(cudaMemcpyFromSymbol(&v, g_ml_err, sizeof(int)));
    BSML_CUDA(cudaMemcpyToSymbol(g_ml_err, &zero, sizeof(int)));
    return v;
}

}  // namespace bsml
