// What the kernels of attn_kv4.cu share: parameters, which keys a row sees,
// addressing of Q, the output and the split workspace.
#pragma once

#include "kv4.h"

namespace kvp {

constexpr int kKv4Head = 128;

struct Kv4Params {
    Kv4Span span;
    Kv4Attn attn;
    int* status;
    float* ws_o;             // partial O of split c: [sequence][K/V head][row][split][128]
    float* ws_ml;            // its max (log2 units) and sum: [...][split][2]
    long long window_rows;   // window * tokens (0: all keys)
    int sink_rows;           // sinks * tokens, at most the capacity
    int group, max_rows;     // query heads per K/V head; rows * group
    int tokens, row_tiles, splits;
    int cluster;             // the splits of a row tile are one cluster and join by themselves
    float scale_log2;        // log2(e) / sqrt(128)
    float rise;              // kRise in score units
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

// The kernel for many query rows (attn_kv4_sm100.cu): P.row_tiles of 256 rows.
int launch_kv4_tiles(const Kv4Params& P, unsigned grid, cudaStream_t stream);

}  // namespace kvp
