// What the kernels of attn_kv4.cu share: parameters, which keys a row sees,
// addressing of Q, the output and the split workspace.
#pragma once

#include "kv4.h"
#include "kv4_pieces.h"

namespace kvp {

constexpr int kKv4Head = 128;

struct Kv4Params {
    Kv4Span span;
    Kv4Attn attn;
    int* status;
    float* ws_o;             // partial O of split c: [sequence][K/V head][row][split][128]
    float* ws_ml;            // its max (log2 units) and sum: [...][split][2]
    int* ws_unit;            // chunked: [0] a CTA's share, [1 + unit] where the unit's first page is in the list
    long long window_rows;   // window * tokens (0: all keys)
    int sink_rows;           // sinks * tokens, at most the capacity
    int group, max_rows;     // query heads per K/V head; rows * group
    int tokens, row_tiles, splits;
    int cluster;             // the splits of a row tile are one cluster and join by themselves
    int ctas;                // (chunked) CTAs of the launch
    int join_ctas;           // (chunked) CTAs of the join for a unit
    int chunked;             // (many rows) the CTAs share the list of all units' pages evenly: see Kv4Unit
    float scale_log2;        // log2(e) / sqrt(128)
    float rise;              // kRise in score units
    float inv_group;         // 1 / group
};

namespace kv4_dev {

// The keys [0, sink_rows) and [lo, hi) below hi are visible at position pos.
struct Sees {
    int lo, hi;
};
__device__ __forceinline__ Sees sees(const Kv4Params& P, int pos, int end) {
    const int f0 = pos / P.tokens * P.tokens;                  // the frame's first row
    Sees r;
    r.hi = (int)min((long long)f0 + P.tokens, (long long)end);
    r.lo = P.window_rows ? (int)max((long long)f0 + P.tokens - P.window_rows, 0LL) : 0;
    return r;
}

__device__ __forceinline__ const __nv_bfloat16* q_row(const Kv4Params& P, int b, int h, int r) {
    return static_cast<const __nv_bfloat16*>(P.attn.q) + b * P.attn.q_batch_stride +
           (long long)(r / P.group) * P.attn.q_row_stride + (long long)(h * P.group + r % P.group) * kKv4Head;
}

__device__ __forceinline__ __nv_bfloat16* out_row(const Kv4Params& P, int b, int h, int r) {
    return static_cast<__nv_bfloat16*>(P.attn.out) + b * P.attn.out_batch_stride +
           (long long)(r / P.group) * P.attn.out_row_stride + (long long)(h * P.group + r % P.group) * kKv4Head;
}

constexpr int kKv4UnitCost = 3;

// The units of the kernel for many rows: 256 query rows of one sequence and
// K/V head, against the pages that any of them sees (those of the sinks
// below the window, then the window's).  Unit u = pair * kv_heads + head,
// pairs of (row tile, sequence) with the last rows, the longest spans, first.
// Chunked, CTA i takes [i C, (i + 1) C) of the list of all units' costs, a unit's
// being kKv4UnitCost (what its beginning and end take, in pages' time) and then
// its pages; a piece that is not its whole unit is a partial, in slot 2 i + 1 if
// it begins the unit (it is the CTA's last then), 2 i if not (its first).
struct Kv4Unit {
    int b, start, end, rows, r0;       // rows = count * group; this unit's [r0, r0 + 256)
    int na, b0, pages;                 // pages [0, na) and [b0, b0 + pages - na); 0: nothing to do
    Sees first, last;                  // what its first and last row see
    bool refused;                      // the sequence's start or count does not fit
};
__device__ __forceinline__ Kv4Unit unit_of(const Kv4Params& P, int pair) {
    Kv4Unit u;
    u.b = pair % P.span.batch;
    u.r0 = (P.row_tiles - 1 - pair / P.span.batch) * 256;
    u.pages = 0;
    int count;
    u.refused = !sequence(P.span, u.b, u.start, count);
    u.rows = u.refused ? 0 : count * P.group;
    if (u.r0 >= u.rows) return u;
    u.end = u.start + count;
    u.first = sees(P, u.start + u.r0 / P.group, u.end);
    u.last = sees(P, u.start + (min(u.r0 + 256, u.rows) - 1) / P.group, u.end);
    u.b0 = u.first.lo / kKv4PageRows;
    u.na = min((min(P.sink_rows, u.last.hi) + kKv4PageRows - 1) / kKv4PageRows, u.b0);
    u.pages = u.na + (u.last.hi + kKv4PageRows - 1) / kKv4PageRows - u.b0;
    return u;
}
__device__ __forceinline__ long long unit_slot(int cta, bool begins) { return 2LL * cta + (begins ? 1 : 0); }

// A row's partial O and (max, sum) of one split.
__device__ __forceinline__ long long ws_slot(const Kv4Params& P, int b, int h, int r, int split) {
    return (((long long)b * P.span.kv_heads + h) * P.max_rows + r) * P.splits + split;
}
__device__ __forceinline__ float* ws_o(const Kv4Params& P, int b, int h, int r, int split) {
    return P.ws_o + ws_slot(P, b, h, r, split) * kKv4Head;
}
__device__ __forceinline__ float2* ws_ml(const Kv4Params& P, int b, int h, int r, int split) {
    return reinterpret_cast<float2*>(P.ws_ml) + ws_slot(P, b, h, r, split);
}

// Dims [d, d + 4) of a finished row; a row without keys (sum 0) is 0.
__device__ __forceinline__ void store_out(const Kv4Params& P, int b, int h, int r, int d, const float4& o, float sum) {
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    const __nv_bfloat162 lo = __floats2bfloat162_rn(o.x * inv, o.y * inv);
    const __nv_bfloat162 hi = __floats2bfloat162_rn(o.z * inv, o.w * inv);
    *reinterpret_cast<uint2*>(out_row(P, b, h, r) + d) =
        make_uint2(reinterpret_cast<const uint32_t&>(lo), reinterpret_cast<const uint32_t&>(hi));
}

// Dims [d, d + 4) of a row of one split: finished, or a partial for the join
// (of a row without keys in this split only the sum 0 is read).
__device__ __forceinline__ void put(const Kv4Params& P, int b, int h, int r, int split, int d, const float4& o,
                                    float m, float sum) {
    if (P.splits == 1) {
        store_out(P, b, h, r, d, o, sum);
        return;
    }
    if (sum != 0.f) *reinterpret_cast<float4*>(ws_o(P, b, h, r, split) + d) = o;
    if (d == 0) *ws_ml(P, b, h, r, split) = make_float2(m, sum);
}

}  // namespace kv4_dev

constexpr int kKv4ChunkPairs = 1152;     // (row tile, sequence) pairs that the CTAs of a chunked launch add up

// The kernel for many query rows (attn_kv4_sm100.cu): P.row_tiles of 256 rows.
int launch_kv4_tiles(const Kv4Params& P, unsigned grid, cudaStream_t stream);

}  // namespace kvp
