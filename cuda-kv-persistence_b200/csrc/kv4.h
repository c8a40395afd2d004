// The 4-bit K/V cache (kv4_cache.cu) and the attention over it
// (attn_kv4.cu): the format, descriptors and launchers.
//
// Format.  Every 16 dims of a K or V row share one scale s and hold 4-bit
// codes c, value (c - 8) * s.  A scale byte eeeee mmm is s = (1 + m/8) *
// 2^(e - 15): no zero, no infinity, no NaN, so any bytes decode to finite
// numbers and a masked key can never spread a NaN.  (c - 8) has at most 3
// significant bits and s has 4, so every value is exact in bf16, and in fp16
// once divided by 64: the tensor cores see just what the cache stands for.
//
// Writing: s = max|x| / 7 rounded to 4 significant bits (halves up), within
// [2^-15, 3840] (bytes 0 to 215); c - 8 = x / s rounded to the nearest integer
// (halves away from zero).  Rounding s moves max|x| / s to 7.4375 at most, so
// no value is clipped.  fp32 rows are rounded to bf16 first.  NaN is stored
// as 0 and |x| > 26880 = 7 * 3840 as that bound; both set KVP_STATUS_RANGE.
// Bytes above 215 can stand in unwritten rows only: K's at their value, V's
// as 215 (vscale2), in reads and in attention.
//
// Layout.  Pages of 128 rows, uint8 [n_pages][kv_heads][18432]; a head's
// share of a page is 16 blocks of 8 rows, each 1152 bytes: K codes [8 rows]
// [64 B], K scales [8 rows][8], V codes [8 groups][8 rows][8 B], V scales
// [8 groups][8 rows].  Eight dims make a 32-bit word: dim 2i in bits
// [4i, 4i + 4), dim 2i + 1 sixteen bits higher, so one shift and one mask
// give two neighbouring dims in the halves of a register.  A warp reads a
// block's K or V as 32 consecutive 16-byte words whichever way its matrix
// fragments run: K by (row, quarter of the dims), V by (16-dim group, row
// pair).
#pragma once

#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include "kvp_common.h"

namespace kvp {

constexpr int kKv4PageRows = 128;
constexpr int kKv4BlockRows = 8;
constexpr int kKv4BlockBytes = 1152;                      // 8 rows of one head
constexpr int kKv4PageHeadBytes = 16 * kKv4BlockBytes;    // 18432
constexpr int kKv4KScale = 512;                           // offsets inside a block
constexpr int kKv4VCode = 576;
constexpr int kKv4VScale = 1088;
constexpr float kKv4Top = 26880.f;                        // 7 * 1.875 * 2^11
constexpr int kKv4TopScale = 215;                         // the scale byte of 1.875 * 2^11
constexpr int kKv4MaxRows = 1 << 30;                      // positions of a sequence stay below

// Which rows of a cache a call touches: row i < count of sequence b is
// position start + i, in page page_map[b][position / 128].
struct Kv4Span {
    void* pages;             // uint8 [n_pages][kv_heads][18432]
    const int* page_map;     // device [batch][map_stride]; null: page b * map_stride + p
    const int* starts;       // device [batch]; null: `start` for all
    const int* counts;       // device [batch], <= rows; null: `rows` for all
    long long n_pages;
    int kv_heads, batch, map_stride, start, rows;
};

// K and V rows (or outputs): head h of row i of sequence b at element
// b * batch_stride + i * row_stride + 128 * h.  Either may be null when read.
struct Kv4Rows {
    void* k;
    void* v;
    long long row_stride, batch_stride;
    int elem_bytes;          // 2 bf16, 4 fp32
    long long v_row_stride, v_batch_stride;   // V's; outputs have K's
};

struct Kv4Attn {
    const void* q;           // bf16, head h of row i of sequence b as in Kv4Rows
    void* out;
    long long q_row_stride, q_batch_stride, out_row_stride, out_batch_stride;
    int heads;               // a multiple of kv_heads; query head h reads K/V head h / (heads / kv_heads)
    int tokens;              // rows per frame
    int window;              // frames visible (own frame included); 0 = all
    int sinks;               // first frames that stay visible
};

// Argument checks, touching no device state (KVP_OK or KVP_ERR_ARG with a message).
int check_kv4_rows(const Kv4Span& s, const Kv4Rows& r, bool write);
int check_kv4_attn(const Kv4Span& s, const Kv4Attn& a);

int launch_kv4_write(const Kv4Span& s, const Kv4Rows& r, int* d_status, cudaStream_t stream);
int launch_kv4_read(const Kv4Span& s, const Kv4Rows& r, int* d_status, cudaStream_t stream);
int launch_attn_kv4(const Kv4Span& s, const Kv4Attn& a, int* d_status, cudaStream_t stream);

#ifdef __CUDACC__
// A launch that is prepared while what is before it in the stream still runs: the
// kernels wait for that (cudaGridDependencySynchronize) before they touch memory,
// and use no read-only loads: what they read may change while they wait.
// Back to back, a decoding step over 4099 keys x 12 heads then takes 8.2 us
// instead of 10.3, 131071 keys 53.4 instead of 56.5.
inline cudaLaunchConfig_t kv4_config(unsigned grid, unsigned threads, size_t smem, cudaLaunchAttribute* attr,
                                     cudaStream_t stream) {
    attr->id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr->val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cfg;
}

namespace kv4_dev {

// A sequence's first position and row count; false (with the status bit set
// by one thread of the caller's choosing) when the device values do not fit.
__device__ __forceinline__ bool sequence(const Kv4Span& s, int b, int& start, int& count) {
    start = s.starts ? s.starts[b] : s.start;
    count = s.counts ? s.counts[b] : s.rows;
    return start >= 0 && count >= 0 && count <= s.rows &&
           (long long)start + count <= (long long)s.map_stride * kKv4PageRows;
}

// Physical page of position page p of sequence b; -1 when it is not in the pool.
__device__ __forceinline__ int page_of(const Kv4Span& s, int b, int p) {
    const long long i = (long long)b * s.map_stride + p;
    const long long page = s.page_map ? (long long)s.page_map[i] : i;
    return page >= 0 && page < s.n_pages ? (int)page : -1;
}

__device__ __forceinline__ uint32_t bf2_fma(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t d;
    asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
    return d;
}
__device__ __forceinline__ uint32_t bf2_mul(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}

// Two scale bytes (one in the low byte of each half of b2) as the factors of
// field(): hi = 128 * s per half, by putting eeeee mmm into a bf16's bits,
// lo = -(17/16) * hi = -136 * s.  Both exact (4 and 8 significant bits).
struct Scale2 {
    uint32_t hi, lo;
};
__device__ __forceinline__ Scale2 scale2(uint32_t b2) {
    Scale2 r;
    r.hi = b2 * 16u + 0x3B803B80u;
    r.lo = bf2_mul(r.hi, 0xBF88BF88u);
    return r;
}
// Nibble i of both halves of w as bf16 values: 0x3F80 | c is 1 + c/128, and
// (1 + c/128) * 128 s - 136 s = (c - 8) s, exact.
template <int i>
__device__ __forceinline__ uint32_t field(uint32_t w, const Scale2& s) {
    uint32_t x;   // one lop3: (w & mask) | one
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(x) : "r"(w >> (4 * i)), "r"(0x000F000Fu), "r"(0x3F803F80u));
    return bf2_fma(x, s.hi, s.lo);
}

// V in fp16, as V / 64 (kVUnit): its ten mantissa bits take two codes without
// a shift (0x3C00 | c is 1 + c/1024, 0x3C00 | c << 4 is 1 + c/64), so a word
// needs one shift instead of three, and P in fp16 keeps eleven bits.  With s' =
// s / 64, hi = 1024 s' and lo = -1032 s' = -(129/128) hi, hi4 = 64 s' and lo4 =
// -72 s': at most 11 significant bits, between 2^-24 and 61920 for bytes up
// to 215, all exact, and so is (c - 8) s'.  Higher bytes, which only unwritten
// rows can hold, count as 215 so that they stay finite.
//
// P is 2^(x - m + kPShift), and a score passes the running max m by 8 at most:
// up to 2^15, and fp16's floor of 2^-25 lies 2^-32 below the largest weight.
// The sum l holds the same factor, which cancels in O / l.
constexpr float kVUnit = 64.f;
constexpr float kPShift = 7.f;

__device__ __forceinline__ uint32_t h2_fma(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t d;
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
    return d;
}
__device__ __forceinline__ uint32_t h2_mul(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}
struct VScale2 {
    uint32_t hi, lo, hi4, lo4;
};
__device__ __forceinline__ VScale2 vscale2(uint32_t b2) {
    VScale2 r;
    r.hi = __vminu2(b2, 0x00D700D7u) * 128u + 0x10001000u;
    r.lo = h2_mul(r.hi, 0xBC08BC08u);    // -129/128
    r.hi4 = h2_mul(r.hi, 0x2C002C00u);   // 1/16
    r.lo4 = h2_mul(r.hi, 0xAC80AC80u);   // -72/1024
    return r;
}
template <int i>
__device__ __forceinline__ uint32_t vfield(uint32_t w, const VScale2& s) {
    uint32_t x;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;"
        : "=r"(x) : "r"(i < 2 ? w : w >> 8), "r"(i % 2 ? 0x00F000F0u : 0x000F000Fu), "r"(0x3C003C00u));
    return i % 2 ? h2_fma(x, s.hi4, s.lo4) : h2_fma(x, s.hi, s.lo);
}

}  // namespace kv4_dev
#endif

}  // namespace kvp
