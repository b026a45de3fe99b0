// Tiles of the attention kernels (attention.hip, attention_bwd.hip, attention_plan.hip).
//
// A side of the graph (destinations with their sources, or sources with their destinations) is
// cut into tiles of 16 rows, neighbours in space.  A tile's rows share many columns: the plan
// lists the union of the columns, 32 to a chunk, with a 32-bit mask per row and chunk of the
// edges that exist.  The kernels then take a chunk's 16 x 32 pairs as matrix products on the
// matrix cores, so a column's data is read once per tile and head instead of once per edge (a
// 5000-atom box with 28 neighbours: 448 edges of a tile lead to about 150 columns), and 5 of 6
// products of a pair without an edge are thrown away, which costs less than reading the rows
// again.  Edges of a row are numbered along the row: the k-th set bit of a row over the chunks
// is its k-th edge, so the masks also give each pair's place in the arrays per edge.
//
// Every wave works on one (item, head), an item being a tile, or a part of one that has a long
// row or many edges, and is a workgroup of its own: nothing is shared, and there are no
// barriers.
#pragma once
#include "common.h"
#include "batmobile_hip.h"

namespace bmhip {

constexpr int kAttnRows = 16;     // rows of a tile
constexpr int kAttnCols = 32;     // columns of a chunk

// ---------------------------------------------------------------------------
// the plan of one side, in one int32 array
// ---------------------------------------------------------------------------
constexpr int kPlanHead = 16;     // items, parts, what is wrong, edges of all tiles (64 bits)
constexpr int kPlanItems = 0, kPlanParts = 1, kPlanBad = 2, kPlanEdges = 4;

// An item, read by a wave with one load: tile, first chunk, columns, part (-1: the tile's only
// item); the tile's rows (-1 past the end); each row's first edge in the item; their number.
constexpr int kItemInts = 64, kItemRows = 16, kItemBase = 32, kItemCount = 48;

struct PlanLayout {
    int64_t tiles, max_items, max_chunks;
    int64_t rows, tile_item, tile_chunk, tile_part, items, masks, ids, total;
};

// A tile of more than kTileEdges edges, or with a row of more than kTileRow, is cut into items of
// plan_cut edges or more, along its columns; their results are joined by a second kernel.  The cuts
// stand between columns, so that each is listed once, but for a column of more than kCutColumn edges
// (parallel edges), which is cut where the item is full.  Items then differ by fewer than kCutColumn
// edges from equal shares of at most 768, and none has more than kTileEdges, which is what the kernels
// keep of them in LDS (twice that costs the training steps 3 to 14 %) and what bounds the rounding of
// their sums: of 1500 equal edges in one item the fp32 sums were 1.7e-5 off.  Items of
// 64 edges serve a graph too small to fill the card (one row of 1000 edges, 64 bf16 components:
// 9.4 us against 14.5 with 256 edges and 22.0 uncut), but a large one pays for their number (100
// rows of 500, 8 heads of 256 in bf16: 111 us with 256 edges, 92 with 512).
constexpr int kTileEdges = 1024, kTileRow = 512, kCutColumn = 256;

__host__ __device__ inline int64_t plan_cut(int64_t n_edges) {
    const int64_t c = n_edges / 128;
    return c < 64 ? 64 : c > 512 ? 512 : c;
}

constexpr int64_t kPlanRows = ((int64_t)1 << 26) - 64;    // 64 threads a row, < 2^32 a launch

inline PlanLayout plan_layout(int64_t n_rows, int64_t n_edges) {
    PlanLayout p;
    p.tiles = ceil_div(n_rows, kAttnRows);
    p.max_items = p.tiles + n_edges / plan_cut(n_edges);
    p.max_chunks = n_edges / kAttnCols + p.max_items;
    int64_t at = kPlanHead;
    auto take = [&](int64_t n) {
        const int64_t r = at;
        at += (n + 15) / 16 * 16;   // 64-byte sections
        return r;
    };
    p.rows = take(p.tiles * kAttnRows);
    p.tile_item = take(p.tiles + 1);
    p.tile_chunk = take(p.tiles + 1);
    p.tile_part = take(p.tiles + 1);
    p.items = take(p.max_items * kItemInts);
    p.masks = take(p.max_chunks * kAttnRows);
    p.ids = take(p.max_chunks * kAttnCols);
    p.total = at;
    return p;
}

struct AttnSide {
    const int* rows;          // [16 tiles], -1 past the end
    const int* tile_part;     // [tiles + 1] first part
    const int* items;         // [items][64]
    const uint32_t* masks;    // [16 chunks]
    const int* ids;           // [32 chunks] columns
    int n_items, n_tiles, n_edges;
};

// The tile of part p, the tile's first part and their number.
__device__ __forceinline__ int tile_of_part(const AttnSide& s, int p, int& first, int& parts) {
    int lo = 0, hi = s.n_tiles - 1;
    while (lo < hi) {
        const int m = (lo + hi + 1) >> 1;
        if (s.tile_part[m] <= p) lo = m; else hi = m - 1;
    }
    first = s.tile_part[lo];
    parts = s.tile_part[lo + 1] - first;
    return lo;
}

// a / b of numbers that are the same in every lane, as a scalar.  The division runs on the VALU; where
// the compiler leaves its result there, a buffer based on it is loaded from lane by lane, in a loop for
// each load (training step of 5000 atoms 202 us against 191).
__device__ __forceinline__ int uniform_quotient(int a, int b) {
    return __builtin_amdgcn_readfirstlane((int)((uint32_t)a / (uint32_t)b));
}

// The work unit of workgroup b, which is one wave.  It runs on XCD b % 8, which takes a
// contiguous eighth of the items, so that tiles that share columns meet in one L2, and those
// head by head: the columns of the tiles in flight are then one head's only, which fit the L2
// (50,000 atoms, 8 heads of 256 in bf16: 1 KB a column against 8).
__device__ __forceinline__ bool attn_unit(unsigned block, int n_items, int heads, int& item,
                                          int& head) {
    const int x = block & 7;
    const int i0 = (int)((int64_t)n_items * x >> 3), i1 = (int)((int64_t)n_items * (x + 1) >> 3);
    const uint32_t w = block >> 3;
    if (w >= (uint64_t)(i1 - i0) * heads) return false;
    head = uniform_quotient((int)w, i1 - i0);
    item = i0 + (int)(w - (uint32_t)head * (uint32_t)(i1 - i0));
    return true;
}
inline unsigned attn_grid(int64_t n_items, int64_t heads) {
    return (unsigned)(ceil_div(n_items, 8) * heads * 8);
}

// ---------------------------------------------------------------------------
// Fragments.  l = lane, n = l % 16, g = l / 16.  A step takes kTiles tiles of 16 columns.
//
// Row form (the contraction runs along a row's components): lane l holds row n.  Read like that
// from memory, 16 lanes in a row would ask for 16 cache lines (37 line accesses a load were
// measured); the columns' rows go to LDS first, whole rows at a time (RowTile).
//   bf16: components 32 s + 8 g + (0..7) in step s of v_mfma_f32_16x16x32_bf16
//   fp32: components 16 s + 4 g + (0..3), one v_mfma_f32_16x16x4f32 for each of the four
// Column form (the contraction runs over the step's columns j): lane l holds kW components
// kW n + (0..) of a block of 16 kW, for kRowsPerLane columns; matrix product c of the block
// takes component c of each, so that its row m is component kW m + c.
//   bf16: columns 4 g + (0..3) and 16 + 4 g + (0..3), fp32: 4 g + (0..3)
// The products are taken transposed, (columns) x (tile rows): lane l then has the pairs of tile
// row n with columns 16 t + 4 g + r in tile t, element r, which is at once the layout that the
// second product takes its factor in.  A result of the column form lies with tile row n in lane
// l, components kW (4 g + r) + c of block b in acc[b kW + c][r].
// ---------------------------------------------------------------------------
template <typename T>
struct Attn;

template <>
struct Attn<float> {
    static constexpr int kTiles = 1, kRowsPerLane = 4, kSteps = 16, kAlign = 4;
    using Vec = float4;                          // a row-form load
    static __device__ __forceinline__ v4f rowprod(const float4& a, const float4& b, v4f acc) {
        return mfma4(a, b, acc);
    }
};
template <>
struct Attn<uint16_t> {
    static constexpr int kTiles = 2, kRowsPerLane = 8, kSteps = 32, kAlign = 8;
    using Vec = v4u;
    static __device__ __forceinline__ v4f rowprod(const v4u& a, const v4u& b, v4f acc) {
        return mfma_bf16(a, b, acc);
    }
};

// row of a matrix whose rows are `stride` bytes apart (one 32 x 32 -> 64-bit multiply-add)
template <typename T>
__device__ __forceinline__ const T* row_of(const void* p, int row, uint32_t stride) {
    return (const T*)((const char*)p + (uint64_t)(uint32_t)row * stride);
}

// Over the lanes of the same n: the row pairs, then the halves, swapped and combined.
typedef unsigned v2u __attribute__((ext_vector_type(2)));
template <typename F>
__device__ __forceinline__ float over_groups(float x, F&& f) {
    v2u r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = f(__uint_as_float(r[0]), __uint_as_float(r[1]));
    r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return f(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float max_over_groups(float x) {
    return over_groups(x, [](float a, float b) { return fmaxf(a, b); });
}
__device__ __forceinline__ float sum_over_groups(float x) {
    return over_groups(x, [](float a, float b) { return a + b; });
}

// exp(x) of x <= 0 in natural units (v_exp_f32: a result below 2^-126 is 0)
__device__ __forceinline__ float attn_exp(float x) {
    return __builtin_amdgcn_exp2f(x * 1.4426950408889634f);
}

// Row form of one row: D components of at most P, zero past D.
template <typename T, int P>
struct RowFrag {
    static constexpr int kN = P / Attn<T>::kSteps;
    typename Attn<T>::Vec v[kN];
    // No load is under a condition: a branch would make the waits for later loads wait for all.
    template <bool FULL>
    __device__ __forceinline__ void load(const T* row, int D, int g) {
#pragma unroll
        for (int s = 0; s < kN; ++s) {
            const int d = s * Attn<T>::kSteps + g * Attn<T>::kAlign;
            const bool in = FULL || d < D;
            v[s] = *reinterpret_cast<const typename Attn<T>::Vec*>(row + (in ? d : 0));
            if (!FULL && !in) v[s] = typename Attn<T>::Vec{};
        }
    }
};

// The rows of a step's columns in LDS, moved there by loads that pass no registers: lane l of
// load k brings the 16-byte piece l % kPieces of row k + kLoads (l / kPieces) to place 64 k + l.
// Which piece of its row it brings is that number with the row's low bits flipped, so that the
// 16 rows of a fragment read lie in different banks.
template <typename T, int P, int TILES>
struct RowTile {
    static constexpr int kRows = 16 * TILES, kPieces = P * (int)sizeof(T) / 16;
    static constexpr int kPer = 64 / kPieces, kLoads = kRows / kPer;
    static constexpr int kFlip = (kPieces < 16 ? kPieces : 16) - 1;
    static constexpr int kBytes = kLoads * 1024;
    // Buffer loads, whose completion the compiler counts one by one (it takes the global form for
    // an access to both memories and waits for everything); their offsets have 32 bits, so
    // matrices of 2^32 bytes or more take the global form all the same.  Nothing tells the
    // compiler that a fill writes what is read: arrived<LATER>() stands before the reads, LATER
    // the number of loads issued after the fill that may still be under way (loads complete in
    // order), and reads_done() after them.
    template <int LATER>
    static __device__ __forceinline__ void arrived() {
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"(LATER) : "memory");
    }
    static __device__ __forceinline__ void reads_done() {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
    template <bool FULL, bool WIDE>
    static __device__ __forceinline__ void fill(char* lds, int ids, const T* base,
                                                uint32_t stride, int D, int lane) {
        int id[kLoads];
#pragma unroll
        for (int k = 0; k < kLoads; ++k) id[k] = __shfl(ids, k + kLoads * (lane / kPieces));
        const __amdgpu_buffer_rsrc_t rsrc =
            buffer_rsrc(reinterpret_cast<const float*>(base), 0xffffffffu);
        int place = ((lane % kPieces) ^ (kLoads * (lane / kPieces) & kFlip)) * 16;
        asm volatile("" : "+v"(place));        // kLoads offsets kept over the steps would not fit
#pragma unroll
        for (int k = 0; k < kLoads; ++k) {
            int off = place ^ ((k & kFlip) * 16);
            if (!FULL) off = off < D * (int)sizeof(T) ? off : 0;
            __attribute__((address_space(3))) void* to =
                (__attribute__((address_space(3))) void*)(lds + k * 1024);
            if constexpr (WIDE)
                __builtin_amdgcn_global_load_lds(
                    (const __attribute__((address_space(1))) void*)((const char*)row_of<T>(
                                                                        base, id[k], stride) +
                                                                    off),
                    to, 16, 0, 0);
            else
                __builtin_amdgcn_raw_ptr_buffer_load_lds(
                    rsrc, to, 16, (int)((uint32_t)id[k] * stride + (uint32_t)off), 0, 0, 0);
        }
        asm volatile("" ::: "memory");         // later loads stay later
    }
    template <bool FULL>
    static __device__ __forceinline__ void read(RowFrag<T, P>& f, const char* lds, int t, int D,
                                                int n, int g) {
        const int row = 16 * t + n;
        const char* at = lds + row % kLoads * 1024 + row / kLoads * kPieces * 16;
#pragma unroll
        for (int s = 0; s < RowFrag<T, P>::kN; ++s) {
            // the piece's bits above kFlip apart: a constant offset
            f.v[s] = *reinterpret_cast<const typename Attn<T>::Vec*>(
                at + (((4 * s & kFlip) + g) ^ (row & kFlip)) * 16 + (4 * s & ~kFlip) * 16);
            if (!FULL && s * Attn<T>::kSteps + g * Attn<T>::kAlign >= D)
                f.v[s] = typename Attn<T>::Vec{};
        }
    }
};

template <typename T, int P>
__device__ __forceinline__ v4f row_product(const RowFrag<T, P>& a, const RowFrag<T, P>& b) {
    // two chains: a chain of one accumulator would wait for every product
    v4f x = {0, 0, 0, 0}, y = {0, 0, 0, 0};
#pragma unroll
    for (int s = 0; s < RowFrag<T, P>::kN; s += 2) {
        x = Attn<T>::rowprod(a.v[s], b.v[s], x);
        if (s + 1 < RowFrag<T, P>::kN) y = Attn<T>::rowprod(a.v[s + 1], b.v[s + 1], y);
    }
    return x + y;
}

// Column form of a step's columns: kW components a lane and block.  Past D a lane reads the
// row's start: its results are never stored.
template <typename T, int P>
struct ColFrag;

template <int P>
struct ColFrag<float, P> {
    static constexpr int kW = 4, kBlocks = P / 64, kAcc = kBlocks * kW, kLoads = 4 * kBlocks;
    float4 v[4][kBlocks];
    template <typename F>
    __device__ __forceinline__ void load(F&& row, int D, int n) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float* p = row(j);
#pragma unroll
            for (int b = 0; b < kBlocks; ++b) {
                const int d = b * 64 + 4 * n;
                v[j][b] = *reinterpret_cast<const float4*>(p + (d < D ? d : 0));
            }
        }
    }
    // acc += (columns' components) x w, w[j] the factor of column j and tile row n
    __device__ __forceinline__ void mac(const float* w, v4f* acc) const {
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int b = 0; b < kBlocks; ++b) {
                acc[b * 4 + 0] = mfma1(v[j][b].x, w[j], acc[b * 4 + 0]);
                acc[b * 4 + 1] = mfma1(v[j][b].y, w[j], acc[b * 4 + 1]);
                acc[b * 4 + 2] = mfma1(v[j][b].z, w[j], acc[b * 4 + 2]);
                acc[b * 4 + 3] = mfma1(v[j][b].w, w[j], acc[b * 4 + 3]);
            }
    }
};

template <int P>
struct ColFrag<uint16_t, P> {
    static constexpr int kW = P >= 128 ? 8 : 4, kBlocks = P / (16 * kW), kAcc = kBlocks * kW;
    static constexpr int kLoads = 8 * kBlocks;
    using Vec = unsigned __attribute__((ext_vector_type(kW / 2)));
    Vec v[8][kBlocks];
    template <typename F>
    __device__ __forceinline__ void load(F&& row, int D, int n) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const uint16_t* p = row(j);
#pragma unroll
            for (int b = 0; b < kBlocks; ++b) {
                const int d = b * 16 * kW + kW * n;
                v[j][b] = *reinterpret_cast<const Vec*>(p + (d < D ? d : 0));
            }
        }
    }
    // The factors as the sum of two bf16 values (16 bits): rounded to one they would add an
    // error of the size of the result's own rounding.  The second product costs nothing next to
    // reading the rows.
    __device__ __forceinline__ void mac(const float* w, v4f* acc) const {
        v4u hi, lo;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            hi[i] = bf16_pack(w[2 * i], w[2 * i + 1]);
            lo[i] = bf16_pack(w[2 * i] - bf16_lo(hi[i]), w[2 * i + 1] - bf16_hi(hi[i]));
        }
#pragma unroll
        for (int b = 0; b < kBlocks; ++b)
#pragma unroll
            for (int c = 0; c < kW; ++c) {
                const unsigned sel = c & 1 ? 0x07060302u : 0x05040100u;
                v4u a;
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    a[i] = __builtin_amdgcn_perm(v[2 * i + 1][b][c / 2], v[2 * i][b][c / 2], sel);
                acc[b * kW + c] = mfma_bf16(a, lo, acc[b * kW + c]);
                acc[b * kW + c] = mfma_bf16(a, hi, acc[b * kW + c]);
            }
    }
};

// For items with infinities or NaN in a row that not every tile row has an edge to (the matrix
// product's 0 times them is NaN): f(edge, column) over the edges of one tile row, the whole wave
// together.  Rare, so what uses it is only short.
template <typename F>
__device__ __forceinline__ void each_edge(const AttnSide& s, int item, int r, F&& f) {
    const int* it = s.items + (int64_t)item * kItemInts;
    int e = it[kItemBase + r];
    for (int c = it[1]; c < it[1] + (it[2] + kAttnCols - 1) / kAttnCols; ++c)
        for (uint32_t m = s.masks[(int64_t)c * kAttnRows + r]; m; m &= m - 1)
            f(e++, s.ids[(int64_t)c * kAttnCols + __builtin_ctz(m)]);
}

__device__ __forceinline__ float attn_f32(float x) { return x; }
__device__ __forceinline__ float attn_f32(uint16_t x) { return __uint_as_float((uint32_t)x << 16); }
__device__ __forceinline__ void attn_st(float* p, float v) { *p = v; }
__device__ __forceinline__ void attn_st(uint16_t* p, float v) {
    *p = (uint16_t)(bf16_pack(v, 0.0f) & 0xffffu);
}
__device__ __forceinline__ float attn_wave_sum(float v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    return v;
}
// sum_e w x over a wave's lanes, components lane + 64 c
template <typename T>
__device__ __forceinline__ void add_row(float* acc, float w, const T* x, int D) {
#pragma unroll
    for (int c = 0; c < 4; ++c)
        if (c * 64 + (int)threadIdx.x < D)
            acc[c] = fmaf(w, attn_f32(x[c * 64 + threadIdx.x]), acc[c]);
}

template <int N>
__device__ __forceinline__ bool any_not_finite(const v4f* acc) {
    float t = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) t = fmaf(acc[i][r], 0.0f, t);
    return __any(t != 0.0f);
}

template <int W>
__device__ __forceinline__ void attn_store_w(uint16_t* p, const float* v) {
    if constexpr (W == 8)
        *reinterpret_cast<v4u*>(p) = v4u{bf16_pack(v[0], v[1]), bf16_pack(v[2], v[3]),
                                         bf16_pack(v[4], v[5]), bf16_pack(v[6], v[7])};
    else
        *reinterpret_cast<uint2*>(p) = make_uint2(bf16_pack(v[0], v[1]), bf16_pack(v[2], v[3]));
}
template <int W>
__device__ __forceinline__ void attn_store_w(float* p, const float* v) {
#pragma unroll
    for (int i = 0; i < W; i += 4)
        *reinterpret_cast<float4*>(p + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
}

// f times a tile row's sums to its row of an fp32 part (a cut tile).
template <typename T, int P>
__device__ __forceinline__ void store_part(float* row, const v4f* acc, float f, int D, int g) {
    constexpr int kW = ColFrag<T, P>::kW, kBlocks = ColFrag<T, P>::kBlocks;
#pragma unroll
    for (int b = 0; b < kBlocks; ++b)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int d = b * 16 * kW + kW * (4 * g + r);
            float v[kW];
#pragma unroll
            for (int c = 0; c < kW; ++c) v[c] = acc[b * kW + c][r] * f;
            if (d < D) attn_store_w<kW>(row + d, v);
        }
}

// f times the tile's sums to its rows of results, row i's at out + i * stride elements.  A lane
// holds 16-byte pieces of one row; written as they are, a store would send 64 pieces to 64 cache
// lines.  They go through LDS (the pieces' places with the row's low bits flipped, as in RowTile)
// and leave as whole rows.
template <typename T, int P>
struct OutTile {
    static constexpr int kPieces = P * (int)sizeof(T) / 16, kBytes = 16 * kPieces * 16;
    static constexpr int kFlip = (kPieces < 16 ? kPieces : 16) - 1;
    static __device__ __forceinline__ void store(char* lds, T* out, int64_t stride, int row,
                                                 const v4f* acc, float f, int D, int lane) {
        constexpr int kW = ColFrag<T, P>::kW, kBlocks = ColFrag<T, P>::kBlocks;
        constexpr int kBytesW = kW * (int)sizeof(T);       // 16, or 8: half a piece
        const int n = lane & 15, g = lane >> 4;
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int b = 0; b < kBlocks; ++b)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                float v[kW];
#pragma unroll
                for (int c = 0; c < kW; ++c) v[c] = acc[b * kW + c][r] * f;
                const int at = (b * 16 + 4 * g + r) * kBytesW;
                attn_store_w<kW>(reinterpret_cast<T*>(lds + n * kPieces * 16 +
                                                      ((at / 16) ^ (n & kFlip)) * 16 + at % 16),
                                 v);
            }
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int k = 0; k < kPieces / 4; ++k) {
            const int i = k * 64 + lane, to = i / kPieces, piece = i % kPieces;
            const v4u v = *reinterpret_cast<const v4u*>(
                lds + to * kPieces * 16 + (piece ^ (to & kFlip)) * 16);
            const int at = __shfl(row, to);
            if (at >= 0 && piece * 16 < D * (int)sizeof(T))
                *reinterpret_cast<v4u*>((char*)(out + at * stride) + piece * 16) = v;
        }
    }
};

// ---------------------------------------------------------------------------
// A wave's item, and its values per edge in LDS in the order of the rows: read from memory once,
// contiguous along each row, instead of one gather per pair and step.
// ---------------------------------------------------------------------------
struct Item {
    int tile, chunk, columns, part;        // uniform
    int row, base, count, off, total;      // of tile row n (lane % 16): its LDS place off; all
    int longest;                           // uniform
    __device__ __forceinline__ Item(const AttnSide& s, int item, int lane) {
        const int v = s.items[(int64_t)item * kItemInts + lane];
        tile = __builtin_amdgcn_readlane(v, 0);
        chunk = __builtin_amdgcn_readlane(v, 1);
        columns = __builtin_amdgcn_readlane(v, 2);
        part = __builtin_amdgcn_readlane(v, 3);
        const int n = lane & 15;
        row = __shfl(v, kItemRows + n);
        base = __shfl(v, kItemBase + n);
        count = __shfl(v, kItemCount + n);
        // sum and maximum over lanes 0 .. n of a row of 16
        int x = count, m = count;
        x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);
        x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
        x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
        x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
        m = max(m, __builtin_amdgcn_update_dpp(0, m, 0x111, 0xf, 0xf, false));
        m = max(m, __builtin_amdgcn_update_dpp(0, m, 0x112, 0xf, 0xf, false));
        m = max(m, __builtin_amdgcn_update_dpp(0, m, 0x114, 0xf, 0xf, false));
        m = max(m, __builtin_amdgcn_update_dpp(0, m, 0x118, 0xf, 0xf, false));
        off = x - count;
        total = __builtin_amdgcn_readlane(x, 15);
        longest = __builtin_amdgcn_readlane(m, 15);
    }
    __device__ __forceinline__ int steps(int tiles) const {
        return (columns + 16 * tiles - 1) / (16 * tiles);
    }
    // The item's edges, 16 lanes a row and kStage x 64 at a time: get(edge) for all of them (an
    // edge that exists, also in lanes without one), then put(LDS place, edge, value, k) of tile row
    // 4 k + g.
    static constexpr int kStage = 12;      // rows of up to 48 edges in one go
    template <typename V, typename G, typename P>
    __device__ __forceinline__ void each(const AttnSide& s, int lane, G&& get, P&& put) const {
        const int n = lane & 15, g = lane >> 4;
        int b[4], c[4], o[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            b[k] = __shfl(base, 4 * k + g);
            c[k] = __shfl(count, 4 * k + g);
            o[k] = __shfl(off, 4 * k + g);
        }
        for (int j = n; j - n < longest; j += 4 * kStage) {
            V v[kStage];
#pragma unroll
            for (int u = 0; u < kStage; ++u)
                v[u] = get(min(b[u & 3] + j + (u >> 2) * 16, s.n_edges - 1));
#pragma unroll
            for (int u = 0; u < kStage; ++u) {
                const int i = j + (u >> 2) * 16;
                if (i < c[u & 3]) put(o[u & 3] + i, b[u & 3] + i, v[u], u & 3);
            }
        }
    }
};

// Loads, and work on what earlier loads bring, stay on their side of it: loads complete in
// order, so what is needed first must be issued first, and before waiting for others.
__device__ __forceinline__ void load_fence() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}

// The steps of an item, as buffer loads (scalar base and step, the lane's own offset).
template <int TILES>
struct Steps {
    __amdgpu_buffer_rsrc_t ids_r, masks_r;
    int chunk, last, lane4, n4;
    __device__ __forceinline__ Steps(const AttnSide& s, const Item& item, int lane)
        : ids_r(buffer_rsrc(reinterpret_cast<const float*>(s.ids), 0xffffffffu)),
          masks_r(buffer_rsrc(reinterpret_cast<const float*>(s.masks), 0xffffffffu)),
          chunk(item.chunk), last(item.steps(TILES) - 1),
          lane4(lane % (16 * TILES) * 4), n4((lane & 15) * 4) {}
    // columns of step i, lane l the l-th (modulo their number); a lane that needs others takes
    // them from there
    __device__ __forceinline__ int ids(int i) const {
        const uint32_t at = (uint32_t)chunk * (kAttnCols * 4) +
                            (uint32_t)min(i, last) * (16 * TILES * 4);
        return __builtin_amdgcn_raw_buffer_load_b32(ids_r, lane4, (int)at, 0);
    }
    // tile row n's edges of step i, bit 16 t + 4 g + r
    __device__ __forceinline__ uint32_t mask(int i) const {
        i = min(i, last);
        const uint32_t at = (uint32_t)(chunk + i * TILES / 2) * (kAttnRows * 4);
        const uint32_t m = __builtin_amdgcn_raw_buffer_load_b32(masks_r, n4, (int)at, 0);
        return TILES == 2 ? m : (m >> ((i & 1) * 16)) & 0xffffu;
    }
};
// The columns whose column form this lane holds.
template <typename T>
struct StepCols {
    int col[Attn<T>::kRowsPerLane];
    __device__ __forceinline__ StepCols(int ids, int g) {
#pragma unroll
        for (int j = 0; j < Attn<T>::kRowsPerLane; ++j)
            col[j] = __shfl(ids, (j >> 2) * 16 + 4 * g + (j & 3));
    }
};
// Place of pair (n, 16 t + 4 g + r) along row n's edges, r = 0..3, `done` of which lie before the
// step; on[r]: whether it is an edge.
__device__ __forceinline__ void edge_places(uint32_t mask, int t, int g, int done, int* at,
                                            bool* on) {
    const int bit = 16 * t + 4 * g;
    int a = done + __popc(mask & ((1u << bit) - 1u));
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const uint32_t m = (mask >> (bit + r)) & 1u;
        on[r] = m != 0;
        at[r] = a;
        a += (int)m;
    }
}

// The bias of an edge and head: value[edge_id e][h] as the caller has it, or value[h][e] in the
// side's order (edges_by_head).
struct EdgeBias {
    const float* value;
    const int* eid;
    int64_t edge_step, head_step;
    __device__ __forceinline__ float at(int e, int h) const {
        return value[(int64_t)(eid ? eid[e] : e) * edge_step + h * head_step];
    }
};
inline EdgeBias edge_bias(const float* value, const int32_t* eid, int64_t n_edges, int H,
                          bool by_head) {
    if (by_head) return {value, nullptr, 1, n_edges};
    return {value, eid, H, 1};
}

inline AttnSide side_args(const batmobile_attention_side& s) {
    const PlanLayout p = plan_layout(s.n_rows, s.n_edges);
    AttnSide a;
    a.rows = s.plan + p.rows;
    a.tile_part = s.plan + p.tile_part;
    a.items = s.plan + p.items;
    a.masks = reinterpret_cast<const uint32_t*>(s.plan + p.masks);
    a.ids = s.plan + p.ids;
    a.n_items = s.n_items;
    a.n_tiles = (int)p.tiles;
    a.n_edges = (int)s.n_edges;
    return a;
}

inline bool attn_shape_ok(const batmobile_attention_side& s, int H, int Hkv, int Dk, int Dv,
                          int dtype) {
    return s.n_rows >= 0 && s.n_cols >= 0 && s.n_edges >= 0 && (s.n_rows == 0 || s.plan) &&
           s.n_items >= 0 && s.n_parts >= 0 && H > 0 && H <= 65535 && Hkv > 0 && H % Hkv == 0 &&
           Dk > 0 && Dv > 0 && Dk <= 256 && Dv <= 256 && (dtype == 0 || dtype == 1) &&
           (s.n_edges == 0 || s.n_cols > 0) && s.n_rows < kPlanRows &&
           s.n_edges < INT32_MAX / 4 &&
           // the three sums are one launch, of fewer than 2^32 threads
           3 * ((int64_t)s.n_items + 8) * H < (int64_t)1 << 26;
}

inline bool attn_strides_ok(std::initializer_list<int64_t> strides) {
    for (int64_t s : strides)
        if (s < 0 || s >= (int64_t)1 << 30) return false;
    return true;
}

// Whether rows at these strides (bytes) pass 32-bit offsets.  Within them k and v are loaded through
// a buffer's 32-bit offsets; past them through 64-bit addresses, before which the compiler waits
// for every load under way: 51 and 60 us for 5000 atoms, 8 heads of 128 in f32, 364 and 378 us for
// 50,000 atoms, 8 heads of 256 in bf16.
inline bool attn_wide(int64_t rows, int64_t stride_bytes) {
    return rows * stride_bytes >= (int64_t)1 << 32;
}

}  // namespace bmhip
