// Builds a side's plan (attention.h): tiles of 16 rows in the given order, the union of their
// columns in chunks of 32, the masks.  Three kernels and one scan, no host synchronisation:
//
//   plan_tiles   a thread per tile: its rows, its number of items and the bound of its chunks
//   plan_scan    one workgroup: first item, chunk and part of every tile
//   plan_items   a workgroup per item: the item's edges of the 16 rows sorted by column in LDS,
//                equal columns of different rows merged into one entry (a column that a row
//                holds k times, parallel edges, gets k entries), masks from the entries
//
// A tile with many edges or a long row is cut into items of equal edge counts, each found by
// searching for its first column, and within a column that has very many.
//
// Once per graph and side: 5000 atoms with 28 neighbours take 53 us (35 of them plan_items, whose sort
// is steps of LDS latency and barriers), 50,000 atoms 109 us.
#include "attention.h"

namespace bmhip {

constexpr int kPlanThreads = 256;

struct PlanArgs {
    const int64_t *row_ptr, *col, *order;
    int* plan;
    PlanLayout at;
    int64_t n_rows, n_cols, n_edges;
};

__global__ __launch_bounds__(kPlanThreads) void plan_tiles_kernel(PlanArgs a) {
    const int64_t t = (int64_t)blockIdx.x * kPlanThreads + threadIdx.x;
    int64_t edges = 0, longest = 0;
    for (int s = 0; t < a.at.tiles && s < kAttnRows; ++s) {
        const int64_t i = t * kAttnRows + s;
        int64_t row = i < a.n_rows ? (a.order ? a.order[i] : i) : -1;
        if (row >= a.n_rows || row < 0) row = -1;
        a.plan[a.at.rows + i] = (int)row;
        if (row < 0) continue;
        const int64_t e0 = a.row_ptr[row], e1 = a.row_ptr[row + 1];
        // (edges out of range are left out and reported by the check)
        const int64_t len = e0 >= 0 && e1 >= e0 && e1 <= a.n_edges ? e1 - e0 : 0;
        edges += len;
        longest = max(longest, len);
    }
    long long all = edges;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) all += __shfl_xor(all, o);
    if ((threadIdx.x & 63) == 0)
        atomicAdd(reinterpret_cast<unsigned long long*>(a.plan + kPlanEdges),
                  (unsigned long long)all);
    if (t >= a.at.tiles) return;
    const int64_t cuts = longest > kTileRow || edges > kTileEdges
                             ? max(edges / plan_cut(a.n_edges), (int64_t)1)
                             : 1;
    a.plan[a.at.tile_item + t] = (int)cuts;
    a.plan[a.at.tile_chunk + t] = (int)(edges / kAttnCols + cuts);
    a.plan[a.at.tile_part + t] = cuts > 1 ? (int)cuts : 0;
}

// Exclusive sums of the three arrays, in place; 1024 threads.  The plan has room for the items and
// chunks of n_edges edges: where the tiles hold more (a row_ptr that falls and rises again, an order
// that names a row twice), there are no items, and nothing is written past it.
__global__ __launch_bounds__(1024) void plan_scan_kernel(PlanArgs a) {
    __shared__ int sums[16];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int64_t n = a.at.tiles;
    for (int k = 0; k < 3; ++k) {
        int* v = a.plan + (k == 0 ? a.at.tile_item : k == 1 ? a.at.tile_chunk : a.at.tile_part);
        int carry = 0;
        for (int64_t i0 = 0; i0 < n; i0 += 1024) {
            const int64_t i = i0 + threadIdx.x;
            const int x = i < n ? v[i] : 0, incl = wave_incl_scan(x);
            __syncthreads();
            if (lane == 63) sums[w] = incl;
            __syncthreads();
            int before = carry, total = 0;
            for (int j = 0; j < 16; ++j) {
                before += j < w ? sums[j] : 0;
                total += sums[j];
            }
            if (i < n) v[i] = before + incl - x;
            carry += total;
        }
        if (threadIdx.x == 0) {
            v[n] = carry;
            if (k == 0) a.plan[kPlanItems] = carry;
            if (k == 2) a.plan[kPlanParts] = carry;
        }
    }
    if (threadIdx.x == 0 &&
        *reinterpret_cast<const unsigned long long*>(a.plan + kPlanEdges) >
            (unsigned long long)a.n_edges) {
        a.plan[kPlanItems] = a.plan[kPlanParts] = 0;
        a.plan[kPlanBad] |= 8;
    }
}

// Edges of row [e0, e1) whose column is below c.
__device__ __forceinline__ int64_t edges_below(const int64_t* col, int64_t e0, int64_t e1,
                                               int64_t c) {
    int64_t lo = e0, hi = e1;
    while (lo < hi) {
        const int64_t m = (lo + hi) >> 1;
        if (col[m] < c) lo = m + 1; else hi = m;
    }
    return lo - e0;
}

__global__ __launch_bounds__(kPlanThreads) void plan_items_kernel(PlanArgs a) {
    __shared__ uint64_t key[kTileEdges];
    __shared__ uint16_t before[kTileEdges + 1];       // entries before each sorted edge
    __shared__ uint32_t mask[kTileEdges / kAttnCols * kAttnRows];
    __shared__ int64_t start[kAttnRows], stop[kAttnRows], full[2][kAttnRows];
    __shared__ int pre[kAttnRows + 1], sums[kPlanThreads / 64];
    __shared__ int64_t cut[2], below[2][2][kAttnRows];
    __shared__ int count[16];
    const int item = blockIdx.x, tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    if (item >= a.plan[kPlanItems]) return;
    const int* tile_item = a.plan + a.at.tile_item;
    int lo = 0, hi = (int)a.at.tiles - 1;
    while (lo < hi) {
        const int m = (lo + hi + 1) >> 1;
        if (tile_item[m] <= item) lo = m; else hi = m - 1;
    }
    const int tile = lo, part = item - tile_item[tile], parts = tile_item[tile + 1] - tile_item[tile];
    if (tid < kAttnRows) {
        const int row = a.plan[a.at.rows + tile * kAttnRows + tid];
        int64_t e0 = 0, e1 = 0;
        if (row >= 0) {
            e0 = a.row_ptr[row];
            e1 = a.row_ptr[row + 1];
            if (!(e0 >= 0 && e1 >= e0 && e1 <= a.n_edges)) e0 = e1 = 0;
        }
        full[0][tid] = start[tid] = e0;
        full[1][tid] = stop[tid] = e1;
    }
    __syncthreads();
    int64_t chunk0 = a.plan[a.at.tile_chunk + tile];
    if (parts > 1) {
        int64_t edges = 0;
        for (int r = 0; r < kAttnRows; ++r) edges += full[1][r] - full[0][r];
        // the first column with at least `want` edges below it, 16 candidates at a time
        for (int side = 0; side < 2; ++side) {
            const int64_t want = edges * (part + side) / parts;
            int64_t c0 = 0, c1 = a.n_cols;
            if (part + side == 0) c1 = 0;
            if (part + side == parts) c0 = c1;
            while (c0 < c1) {
                const int k = tid >> 4, r = tid & 15;
                const int64_t c = c0 + (c1 - c0) * (k + 1) / 17;
                if (tid < 16) count[tid] = 0;
                __syncthreads();
                atomicAdd(&count[k], (int)edges_below(a.col, full[0][r], full[1][r], c));
                __syncthreads();
                int64_t n0 = c0, n1 = c1;
                for (int j = 0; j < 16; ++j) {
                    const int64_t cj = c0 + (c1 - c0) * (j + 1) / 17;
                    if (count[j] < want) n0 = max(n0, cj + 1);
                    else n1 = min(n1, cj);
                }
                __syncthreads();
                c0 = min(n0, n1);
                c1 = n1;
            }
            if (tid == 0) cut[side] = c0;
        }
        __syncthreads();
        // a row's edges before the cut's column (0: the column before, which crosses the share)
        if (tid < 4 * kAttnRows) {
            const int r = tid & 15, side = (tid >> 4) & 1, k = tid >> 5;
            below[k][side][r] = edges_below(a.col, full[0][r], full[1][r], cut[side] - 1 + k);
        }
        __syncthreads();
        if (tid < 2 * kAttnRows) {
            const int r = tid & 15, side = tid >> 4;
            int64_t column = 0, left = edges * (part + side) / parts;
            for (int i = 0; i < kAttnRows; ++i) {
                const int64_t n = below[1][side][i] - below[0][side][i];
                column += n;
                left -= below[0][side][i] + (i < r ? n : 0);
            }
            int64_t e = below[1][side][r];
            if (column > kCutColumn)                 // its edges row by row up to the share
                e = below[0][side][r] + min(max(left, (int64_t)0), e - below[0][side][r]);
            (side ? stop : start)[r] = part + side == parts ? full[1][r] : full[0][r] + e;
        }
        __syncthreads();
        if (tid < kAttnRows) stop[tid] = max(stop[tid], start[tid]);
        __syncthreads();
        int64_t skipped = 0;
        for (int r = 0; r < kAttnRows; ++r) skipped += start[r] - full[0][r];
        chunk0 += skipped / kAttnCols + part;
    }
    if (tid == 0) {
        int n = 0;
        for (int r = 0; r < kAttnRows; ++r) {
            pre[r] = n;
            n += (int)(stop[r] - start[r]);
        }
        pre[kAttnRows] = n;
    }
    int* out = a.plan + a.at.items + (int64_t)item * kItemInts;
    if (tid < kAttnRows) {
        out[kItemRows + tid] = a.plan[a.at.rows + (int64_t)tile * kAttnRows + tid];
        out[kItemBase + tid] = (int)start[tid];
        out[kItemCount + tid] = (int)(stop[tid] - start[tid]);
    }
    __syncthreads();
    const int n = pre[kAttnRows];
    uint32_t* masks = reinterpret_cast<uint32_t*>(a.plan) + a.at.masks + chunk0 * kAttnRows;
    int* ids = a.plan + a.at.ids + chunk0 * kAttnCols;
    const int part_at = parts > 1 ? a.plan[a.at.tile_part + tile] + part : -1;
    auto finish = [&](int columns) {
        if (tid == 0) *reinterpret_cast<int4*>(out) = make_int4(tile, (int)chunk0, columns, part_at);
    };
    auto column = [&](int i, int& r) {               // of the i-th edge, row by row
        r = 0;
#pragma unroll
        for (int s = 8; s > 0; s >>= 1)
            if (pre[r + s] <= i) r += s;
        const int64_t c = a.col[start[r] + (i - pre[r])];
        return (int)(c >= 0 && c < a.n_cols ? c : 0);
    };
    if (n > kTileEdges) {                            // only of columns that do not ascend
        if (tid < kAttnRows) out[kItemCount + tid] = 0;
        if (tid == 0) atomicOr(&a.plan[kPlanBad], 4);
        finish(0);
        return;
    }
    int size = 64;
    while (size < n) size <<= 1;
    for (int i = tid; i < size; i += kPlanThreads) {
        uint64_t k = ~0ull;
        if (i < n) {
            int r;
            const int c = column(i, r);
            k = ((uint64_t)c << 20) | ((uint64_t)r << 16) | (uint64_t)(i - pre[r]);
        }
        key[i] = k;
    }
    for (int i = tid; i < kTileEdges / kAttnCols * kAttnRows; i += kPlanThreads) mask[i] = 0;
    for (int k = 2; k <= size; k <<= 1)
        for (int j = k >> 1; j > 0; j >>= 1) {
            __syncthreads();
            for (int p = tid; p < size / 2; p += kPlanThreads) {
                const int i = 2 * p - (p & (j - 1)), q = i + j;
                const uint64_t x = key[i], y = key[q];
                if ((x > y) == ((i & k) == 0)) {
                    key[i] = y;
                    key[q] = x;
                }
            }
        }
    __syncthreads();
    // k-th edge of its row to this column, and whether it is the first such of its column: then
    // it opens an entry.  Sorted by (column, row, place): a column's rows are runs.
    auto kth = [&](int i) {
        int k = 0;
        while (i - k > 0 && (key[i - k - 1] >> 16) == (key[i] >> 16)) ++k;
        return k;
    };
    auto opens = [&](int i, int k) {
        int at = i - k;                               // start of the row's run
        while (at > 0 && (key[at - 1] >> 20) == (key[i] >> 20)) {
            int len = 1;
            while (at - len > 0 && (key[at - len - 1] >> 16) == (key[at - 1] >> 16)) ++len;
            if (len > k) return false;
            at -= len;
        }
        return true;
    };
    const int per = (size + kPlanThreads - 1) / kPlanThreads, i0 = tid * per;
    int mine = 0;
    for (int i = i0; i < min(i0 + per, n); ++i) mine += opens(i, kth(i));
    const int incl = wave_incl_scan(mine);
    if (lane == 63) sums[w] = incl;
    __syncthreads();
    int run = incl - mine, total = 0;
    for (int j = 0; j < kPlanThreads / 64; ++j) {
        run += j < w ? sums[j] : 0;
        total += sums[j];
    }
    for (int i = i0; i < min(i0 + per, n); ++i) {
        before[i] = (uint16_t)run;
        run += opens(i, kth(i));
    }
    __syncthreads();
    const int chunks = (total + kAttnCols - 1) / kAttnCols;
    for (int i = i0; i < min(i0 + per, n); ++i) {
        const int k = kth(i);
        int g = i;                                    // the column's first edge
        while (g > 0 && (key[g - 1] >> 20) == (key[i] >> 20)) --g;
        const int e = before[g] + k, r = (int)(key[i] >> 16) & 15;
        atomicOr(&mask[(e >> 5) * kAttnRows + r], 1u << (e & 31));
        if (opens(i, k)) ids[e] = (int)(key[i] >> 20);
    }
    __syncthreads();
    for (int i = tid; i < chunks * kAttnRows; i += kPlanThreads) masks[i] = mask[i];
    for (int i = total + tid; i < chunks * kAttnCols; i += kPlanThreads)
        ids[i] = (int)(key[n - 1] >> 20);             // read with factor 0
    finish(total);
}

// A wave per row: offsets in order, columns in range and ascending.
__global__ __launch_bounds__(256) void plan_check_kernel(PlanArgs a) {
    const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (row >= a.n_rows) return;
    const int64_t e0 = a.row_ptr[row], e1 = a.row_ptr[row + 1];
    int bad = 0;
    if (e0 < 0 || e1 < e0 || e1 > a.n_edges || (row == 0 && e0 != 0) ||
        (row == a.n_rows - 1 && e1 != a.n_edges)) {
        bad = 1;
    } else {
        for (int64_t e = e0 + (threadIdx.x & 63); e < e1; e += 64) {
            const int64_t c = a.col[e];
            if (c < 0 || c >= a.n_cols) bad |= 2;
            if (e > e0 && a.col[e - 1] > c) bad |= 4;
        }
    }
    if (bad) atomicOr(&a.plan[kPlanBad], bad);
}

__global__ void plan_head_kernel(int* plan) {
    if (threadIdx.x < kPlanHead) plan[threadIdx.x] = 0;
}

}  // namespace bmhip

using namespace bmhip;

static bool plan_shape_ok(int64_t n_rows, int64_t n_cols, int64_t n_edges) {
    return n_rows >= 0 && n_cols >= 0 && n_edges >= 0 && n_rows < kPlanRows &&
           n_cols < INT32_MAX && n_edges < INT32_MAX / 4 && (n_edges == 0 || n_cols > 0);
}

extern "C" size_t batteries_attention_plan_bytes(int64_t n_rows, int64_t n_edges) {
    if (!plan_shape_ok(n_rows, 1, n_edges)) return 0;
    return (size_t)plan_layout(n_rows, n_edges).total * sizeof(int);
}

extern "C" int batteries_attention_plan(const int64_t* row_ptr, const int64_t* col,
                                        const int64_t* order, int64_t n_rows, int64_t n_cols,
                                        int64_t n_edges, int check, void* plan, size_t plan_bytes,
                                        hipStream_t stream) {
    if (!plan_shape_ok(n_rows, n_cols, n_edges) || (n_rows > 0 && !row_ptr) ||
        (n_edges > 0 && !col))
        return BM_ERR_ARG;
    if (!plan || (reinterpret_cast<uintptr_t>(plan) & 63) ||
        plan_bytes < batteries_attention_plan_bytes(n_rows, n_edges))
        return BM_ERR_WORKSPACE;
    PlanArgs a{row_ptr, col, order, (int*)plan, plan_layout(n_rows, n_edges), n_rows, n_cols,
               n_edges};
    plan_head_kernel<<<1, 64, 0, stream>>>(a.plan);
    if (n_rows == 0) return (int)hipGetLastError();
    if (check)
        plan_check_kernel<<<(unsigned)ceil_div(n_rows, 4), 256, 0, stream>>>(a);
    plan_tiles_kernel<<<(unsigned)ceil_div(a.at.tiles, kPlanThreads), kPlanThreads, 0, stream>>>(a);
    plan_scan_kernel<<<1, 1024, 0, stream>>>(a);
    plan_items_kernel<<<(unsigned)a.at.max_items, kPlanThreads, 0, stream>>>(a);
    return (int)hipGetLastError();
}
