// Writing the 4-bit K/V cache and reading it back (format: kv4.h).
//
// Both are byte movement: 512 B of a bf16 row and head against 144 B in the
// cache, every byte touched once.  A warp owns one 8-row block of one head,
// which is what a scale's 16 dims and a page's blocks both divide into, so no
// two warps share a byte; consecutive warps take consecutive heads of the same
// rows, so a CTA's global rows are contiguous.  At 32760 bf16 rows x 12 heads
// (258 MB) a write takes 45.7 us and a read 44.1, 5.6 and 5.8 TB/s; one
// frame's write (1560 rows) 4.0 us and a token's 2.4, which is a launch.  fp32:
// 9000 rows x 8 heads (84 MB) in 21.7 us, 3.9 TB/s (a warp's loads, staging and
// conversion follow one another, two CTAs of 117 registers an SM), out in 14.6, 5.8.
#include "kernels.h"
#include "kv4.h"

namespace kvp {

namespace {

using namespace kv4_dev;

constexpr int kThreads = 256;

// One warp's block: sequence b, head h, positions [pos0, pos0 + 8) of which
// [start, start + count) are the call's.
struct Item {
    int b, h, start, count, pos0;
    uint8_t* blk;            // null: the page is not in the pool
};

// Warp item w of batch * kv_heads * blocks; false: nothing to do.
__device__ __forceinline__ bool item_of(const Kv4Span& s, long long w, int blocks, int lane, int* status,
                                        Item& it) {
    it.h = (int)(w % s.kv_heads);
    const long long x = w / s.kv_heads;
    const int j = (int)(x % blocks);
    it.b = (int)(x / blocks);
    if (!sequence(s, it.b, it.start, it.count)) {
        if (lane == 0 && it.h == 0 && j == 0) atomicOr(status, KVP_STATUS_MAP);
        return false;
    }
    it.pos0 = (it.start & ~(kKv4BlockRows - 1)) + j * kKv4BlockRows;
    if (it.count == 0 || it.pos0 >= it.start + it.count) return false;
    const int page = page_of(s, it.b, it.pos0 / kKv4PageRows);
    if (page < 0) {
        if (lane == 0) atomicOr(status, KVP_STATUS_MAP);
        it.blk = nullptr;
        return true;
    }
    it.blk = static_cast<uint8_t*>(s.pages) + ((long long)page * s.kv_heads + it.h) * kKv4PageHeadBytes +
             (it.pos0 % kKv4PageRows) / kKv4BlockRows * kKv4BlockBytes;
    return true;
}

// 16 bf16 values, two to a register.
__device__ __forceinline__ void load16(const __nv_bfloat16* p, uint32_t (&x)[8]) {
    const uint4 a = *reinterpret_cast<const uint4*>(p), b = *reinterpret_cast<const uint4*>(p + 8);
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
    x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
}

// fp32 rows are twice as long: a lane's 64 or 128 bytes of a row no longer
// stay in L1 between its loads (3.4 TB/s), so they come in whole rows, 16
// bytes a lane, and go as bf16 through shared memory, [8 rows][16 chunks of
// 16 bytes], the chunks swapped so that neither way of reading conflicts.
__device__ __forceinline__ int stage_at(int row, int chunk) {
    return row * 256 + ((chunk ^ (chunk >> 3 & 1) ^ (row & 1) << 1 ^ (row >> 1 & 1) << 2 ^ (row >> 2 & 1)) << 4);
}
__device__ __forceinline__ void load16(const uint8_t* stage, int row, int chunk, uint32_t (&x)[8]) {
    const uint4 a = *reinterpret_cast<const uint4*>(stage + stage_at(row, chunk));
    const uint4 b = *reinterpret_cast<const uint4*>(stage + stage_at(row, chunk + 1));
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
    x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
}
__device__ __forceinline__ void fetch_rows(float4 (&y)[kKv4BlockRows], const float* p, long long row_stride, int first,
                                           int count, int lane) {
#pragma unroll
    for (int r = 0; r < kKv4BlockRows; ++r)
        y[r] = first + r >= 0 && first + r < count
                   ? __ldcs(reinterpret_cast<const float4*>(p + (first + r) * row_stride + 4 * lane))
                   : make_float4(0.f, 0.f, 0.f, 0.f);
}
__device__ __forceinline__ void stage_rows(uint8_t* stage, const float4 (&y)[kKv4BlockRows], int lane) {
#pragma unroll
    for (int r = 0; r < kKv4BlockRows; ++r) {
        const __nv_bfloat162 lo = __floats2bfloat162_rn(y[r].x, y[r].y), hi = __floats2bfloat162_rn(y[r].z, y[r].w);
        *reinterpret_cast<uint2*>(stage + stage_at(r, lane >> 1) + (lane & 1) * 8) =
            make_uint2(reinterpret_cast<const uint32_t&>(lo), reinterpret_cast<const uint32_t&>(hi));
    }
}

__device__ __forceinline__ float lo_f(uint32_t x) { return __uint_as_float(x << 16); }
__device__ __forceinline__ float hi_f(uint32_t x) { return __uint_as_float(x & 0xFFFF0000u); }

// 16 bf16 values -> two code words and the scale byte.  n = x / s is rounded
// by one fma: x * r + (1.5 * 2^23 + 8) keeps c = n + 8 in its low bits.  r =
// (1 + 2^-14) / s pushes an exact half away from zero; nothing else crosses
// a half, because x and (n + 1/2) s both have at most 8 significant bits and
// so differ by 2^-8 of their size or not at all.  The quotient max / 7 falls
// on a half of the 4-bit scale only exactly, by the same count.
__device__ __forceinline__ uint32_t quantise16(uint32_t (&x)[8], uint32_t (&word)[2], int* status) {
    uint32_t m2 = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint32_t a = x[i] & 0x7FFF7FFFu;       // |x|: as bf16 bits, ordered like integers
        m2 = __vmaxu2(m2, a);
    }
    float top = fmaxf(lo_f(m2), hi_f(m2));
    if ((m2 & 0xFFFFu) > 0x7F80u || (m2 >> 16) > 0x7F80u || top > kKv4Top) {
        // NaN -> 0, beyond the format -> its bound
        atomicOr(status, KVP_STATUS_RANGE);
        top = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            float a = lo_f(x[i]), b = hi_f(x[i]);
            a = a != a ? 0.f : fminf(fmaxf(a, -kKv4Top), kKv4Top);
            b = b != b ? 0.f : fminf(fmaxf(b, -kKv4Top), kKv4Top);
            top = fmaxf(top, fmaxf(fabsf(a), fabsf(b)));
            x[i] = (__float_as_uint(a) >> 16) | (__float_as_uint(b) & 0xFFFF0000u);
        }
    }
    const uint32_t q = __float_as_uint(__fdiv_rn(top, 7.f)) + 0x80000u;   // halves up, at 4 bits
    const int code = min(max((int)(q >> 20) - 896, 0), kKv4TopScale);              // 896 = (127 - 15) << 3
    const float s = __uint_as_float((uint32_t)(code + 896) << 20);
    const float r = __frcp_rn(s) * (1.f + 0x1p-14f);
#pragma unroll
    for (int w = 0; w < 2; ++w) {
        uint32_t p[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t a = __float_as_uint(fmaf(lo_f(x[4 * w + i]), r, 12582920.f));
            const uint32_t b = __float_as_uint(fmaf(hi_f(x[4 * w + i]), r, 12582920.f));
            p[i] = __byte_perm(a, b, 0x5410);        // the sums' low halves are c, 1 <= c <= 15
        }
        word[w] = p[0] | (p[1] << 4) | (p[2] << 8) | (p[3] << 12);
    }
    return (uint32_t)code;
}

template <class T>
__global__ void __launch_bounds__(kThreads, sizeof(T) == 4 ? 2 : 4)
    kv4_write_kernel(const Kv4Span s, const Kv4Rows r, int blocks, long long items, int* status) {
    __shared__ __align__(16) uint8_t stage[sizeof(T) == 4 ? kThreads / 32 : 1][4096];
    const int lane = threadIdx.x & 31;
    const long long step = (long long)gridDim.x * (kThreads / 32);
    cudaGridDependencySynchronize();                  // (kv4_config)
    for (long long w = (long long)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5); w < items; w += step) {
        Item it;
        if (!item_of(s, w, blocks, lane, status, it) || !it.blk) continue;
        const T* k = static_cast<const T*>(r.k) + it.b * r.batch_stride + it.h * 128;
        const T* v = static_cast<const T*>(r.v) + it.b * r.v_batch_stride + it.h * 128;
        const int first = it.pos0 - it.start;          // row index of the block's row 0 (may be < 0)
        const int g = lane >> 2, t = lane & 3;
        // K: this lane's row g, dims [32t, 32t + 32)
        const bool on = first + g >= 0 && first + g < it.count;
        // V: this lane's rows 2t and 2t + 1, dims [16g, 16g + 16)
        const bool on0 = first + 2 * t >= 0 && first + 2 * t < it.count;
        const bool on1 = first + 2 * t + 1 >= 0 && first + 2 * t + 1 < it.count;
        uint32_t ka[8], kb[8], va[8], vb[8];
        if constexpr (sizeof(T) == 4) {
            uint8_t* st = stage[threadIdx.x >> 5];
            __syncwarp();                              // (the block before has been read)
            float4 yk[kKv4BlockRows], yv[kKv4BlockRows];
            fetch_rows(yk, k, r.row_stride, first, it.count, lane);
            fetch_rows(yv, v, r.v_row_stride, first, it.count, lane);
            stage_rows(st, yk, lane);
            stage_rows(st + 2048, yv, lane);
            __syncwarp();
            load16(st, g, 4 * t, ka);
            load16(st, g, 4 * t + 2, kb);
            load16(st + 2048, 2 * t, 2 * g, va);
            load16(st + 2048, 2 * t + 1, 2 * g, vb);
        } else {
            const T* kp = k + (first + g) * r.row_stride + 32 * t;
            const T* vp = v + (first + 2 * t) * r.v_row_stride + 16 * g;
            if (on) {
                load16(kp, ka);
                load16(kp + 16, kb);
            }
            if (on0) load16(vp, va);
            if (on1) load16(vp + r.v_row_stride, vb);
        }
        if (on) {
            uint32_t c0[2], c1[2];
            const uint32_t s0 = quantise16(ka, c0, status), s1 = quantise16(kb, c1, status);
            *reinterpret_cast<uint4*>(it.blk + lane * 16) = make_uint4(c0[0], c0[1], c1[0], c1[1]);
            *reinterpret_cast<uint16_t*>(it.blk + kKv4KScale + lane * 2) = (uint16_t)(s0 | (s1 << 8));
        }
        uint32_t c0[2], c1[2], s0 = 0, s1 = 0;
        if (on0) s0 = quantise16(va, c0, status);
        if (on1) s1 = quantise16(vb, c1, status);
        uint8_t* vc = it.blk + kKv4VCode + lane * 16;
        uint8_t* vs = it.blk + kKv4VScale + lane * 2;
        if (on0 && on1) {
            *reinterpret_cast<uint4*>(vc) = make_uint4(c0[0], c0[1], c1[0], c1[1]);
            *reinterpret_cast<uint16_t*>(vs) = (uint16_t)(s0 | (s1 << 8));
        } else if (on0) {
            *reinterpret_cast<uint2*>(vc) = make_uint2(c0[0], c0[1]);
            vs[0] = (uint8_t)s0;
        } else if (on1) {
            *reinterpret_cast<uint2*>(vc + 8) = make_uint2(c1[0], c1[1]);
            vs[1] = (uint8_t)s1;
        }
    }
}

// The read kernel's lanes: kDims consecutive dims a lane, so that a warp's
// store is 512 consecutive bytes of one or two rows (bf16: a whole word of
// eight dims, fp32: half of one).
template <class T>
struct Out;
template <>
struct Out<__nv_bfloat16> {
    static constexpr int kDims = 8;
    static __device__ __forceinline__ void store(__nv_bfloat16* p, uint32_t w, int, const Scale2& s) {
        __stcs(reinterpret_cast<uint4*>(p), make_uint4(field<0>(w, s), field<1>(w, s), field<2>(w, s), field<3>(w, s)));
    }
};
template <>
struct Out<float> {
    static constexpr int kDims = 4;
    static __device__ __forceinline__ void store(float* p, uint32_t w, int part, const Scale2& s) {
        w >>= 8 * part;
        const uint32_t a = field<0>(w, s), b = field<1>(w, s);
        __stcs(reinterpret_cast<float4*>(p), make_float4(lo_f(a), hi_f(a), lo_f(b), hi_f(b)));
    }
};

template <class T>
__global__ void __launch_bounds__(kThreads)
    kv4_read_kernel(const Kv4Span s, const Kv4Rows rows, int blocks, long long items, int* status) {
    constexpr int kDims = Out<T>::kDims, kLanes = 128 / kDims, kRows = 32 / kLanes;   // lanes of a row, rows of a pass
    T* const k = static_cast<T*>(rows.k);
    T* const v = static_cast<T*>(rows.v);
    const int lane = threadIdx.x & 31;
    const int dim = lane % kLanes * kDims, word = dim / 8, part = dim % 8 / 4;
    const long long step = (long long)gridDim.x * (kThreads / 32);
    cudaGridDependencySynchronize();                  // (kv4_config)
    for (long long w = (long long)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5); w < items; w += step) {
        Item it;
        if (!item_of(s, w, blocks, lane, status, it)) continue;
        const int first = it.pos0 - it.start;
        const long long at0 = it.b * rows.batch_stride + it.h * 128 + dim;
        // every load first: a page that is not in the pool reads as codes of 0
        uint32_t c[2][8 / kRows], e[2][8 / kRows];
#pragma unroll
        for (int i = 0; i < 8 / kRows; ++i) {
            const int r = kRows * i + lane / kLanes;
            c[0][i] = c[1][i] = 0x88888888u;
            e[0][i] = e[1][i] = 0u;
            if (!it.blk || first + r < 0 || first + r >= it.count) continue;
            if (k) {
                c[0][i] = *reinterpret_cast<const uint32_t*>(it.blk + r * 64 + word * 4);
                e[0][i] = it.blk[kKv4KScale + r * 8 + (word >> 1)];
            }
            if (v) {
                c[1][i] = *reinterpret_cast<const uint32_t*>(it.blk + kKv4VCode + (word >> 1) * 64 + r * 8 +
                                                             (word & 1) * 4);
                e[1][i] = min((uint32_t)it.blk[kKv4VScale + (word >> 1) * 8 + r], (uint32_t)kKv4TopScale);
            }
        }
#pragma unroll
        for (int i = 0; i < 8 / kRows; ++i) {
            const int r = kRows * i + lane / kLanes;
            if (first + r < 0 || first + r >= it.count) continue;
            const long long at = at0 + (first + r) * rows.row_stride;
            if (k) Out<T>::store(k + at, c[0][i], part, scale2(e[0][i] * 0x00010001u));
            if (v) Out<T>::store(v + at, c[1][i], part, scale2(e[1][i] * 0x00010001u));
        }
    }
}

// The pool, the map and the rows: what check_kv4_rows and check_kv4_attn share.
int check_span(const char* who, const Kv4Span& s) {
    if (!s.pages || s.n_pages <= 0 || s.n_pages > 0x7fffffffLL || s.kv_heads <= 0 || s.kv_heads > 4096 ||
        s.batch < 0 || s.rows < 0 || s.map_stride <= 0) {
        set_error("%s: bad cache (pages, n_pages, kv_heads, batch, rows or map_stride)", who);
        return KVP_ERR_ARG;
    }
    if ((long long)s.map_stride * kKv4PageRows > kKv4MaxRows || s.rows > kKv4MaxRows) {
        set_error("%s: a sequence holds at most %d rows", who, kKv4MaxRows);
        return KVP_ERR_ARG;
    }
    if ((uintptr_t)s.pages & 15 || ((uintptr_t)s.page_map | (uintptr_t)s.starts | (uintptr_t)s.counts) & 3) {
        set_error("%s: pages must be 16-byte aligned, page_map, starts and counts 4-byte", who);
        return KVP_ERR_ARG;
    }
    if (!s.page_map && (long long)s.batch * s.map_stride > s.n_pages) {
        set_error("%s: without a page map %d sequences of %d pages need as many pages (have %lld)", who, s.batch,
                  s.map_stride, s.n_pages);
        return KVP_ERR_ARG;
    }
    if (!s.starts && (s.start < 0 || (!s.counts &&
                                      (long long)s.start + s.rows > (long long)s.map_stride * kKv4PageRows))) {
        set_error("%s: rows [%d, %lld) do not fit %d pages", who, s.start, (long long)s.start + s.rows,
                  s.map_stride);
        return KVP_ERR_ARG;
    }
    return KVP_OK;
}

// The rows of an output, `len` elements each, lie apart: sequence by sequence
// or, row by row, with the sequences inside (the strides of a single row or
// sequence mean nothing).
bool apart(const Kv4Span& s, long long row_stride, long long batch_stride, long long len) {
    if (s.rows > 1 && row_stride < len) return false;
    if (s.batch <= 1 || s.rows <= 0) return true;
    if (batch_stride < len) return false;
    return s.rows == 1 || batch_stride >= (s.rows - 1) * row_stride + len ||
           row_stride >= (s.batch - 1) * batch_stride + len;
}

int launch(const Kv4Span& s, const Kv4Rows& r, int* status, cudaStream_t stream,
           void (*kernel)(Kv4Span, Kv4Rows, int, long long, int*)) {
    // rows may begin anywhere in a block: the last row's block is
    // (start % 8 + rows - 1) / 8 blocks after the first
    const int lead = s.starts ? kKv4BlockRows - 1 : s.start % kKv4BlockRows;
    const int blocks = (int)(((long long)lead + s.rows + kKv4BlockRows - 1) / kKv4BlockRows);
    const long long items = (long long)s.batch * s.kv_heads * blocks;
    const long long ctas = (items + kThreads / 32 - 1) / (kThreads / 32);
    cudaLaunchAttribute early;
    const cudaLaunchConfig_t cfg =
        kv4_config((unsigned)(ctas < 0x7fffffffLL ? ctas : 0x7fffffffLL), kThreads, 0, &early, stream);
    KVP_CUDA(cudaLaunchKernelEx(&cfg, kernel, s, r, blocks, items, status));
    return KVP_OK;
}

}  // namespace

int check_kv4_rows(const Kv4Span& s, const Kv4Rows& r, bool write) {
    const char* who = write ? "kv4_write" : "kv4_read";
    const int rc = check_span(who, s);
    if (rc != KVP_OK) return rc;
    if (r.elem_bytes != 2 && r.elem_bytes != 4) {
        set_error("%s: elem_bytes must be 2 (bf16) or 4 (fp32)", who);
        return KVP_ERR_ARG;
    }
    if (s.rows > 0 && s.batch > 0 && (write ? (!r.k || !r.v) : (!r.k && !r.v))) {
        set_error("%s: no rows", who);
        return KVP_ERR_ARG;
    }
    const long long per16 = 16 / r.elem_bytes, len = s.kv_heads * 128LL;
    if (((uintptr_t)r.k | (uintptr_t)r.v) & 15 || r.row_stride % per16 || r.batch_stride % per16 ||
        r.v_row_stride % per16 || r.v_batch_stride % per16 ||
        (s.rows > 1 && (r.row_stride < len || r.v_row_stride < len)) ||
        (s.batch > 1 && (r.batch_stride < 0 || r.v_batch_stride < 0))) {
        set_error("%s: rows must be 16-byte aligned, strides too, and a row stride at least kv_heads * 128", who);
        return KVP_ERR_ARG;
    }
    if (!write && s.rows > 0 && s.batch > 0 &&
        (r.k == r.v || !apart(s, r.row_stride, r.batch_stride, len))) {
        set_error("kv4_read: the output rows overlap");
        return KVP_ERR_ARG;
    }
    return KVP_OK;
}

int check_kv4_attn(const Kv4Span& s, const Kv4Attn& a) {
    const int rc = check_span("attn_kv4", s);
    if (rc != KVP_OK) return rc;
    if (a.heads <= 0 || a.heads % s.kv_heads || a.tokens <= 0 || a.window < 0 || a.sinks < 0 ||
        (s.rows > 0 && s.batch > 0 && (!a.q || !a.out))) {
        set_error("attn_kv4: bad descriptor (heads must be a multiple of kv_heads, tokens > 0)");
        return KVP_ERR_ARG;
    }
    if ((long long)s.rows * (a.heads / s.kv_heads) > kKv4MaxRows) {
        set_error("attn_kv4: rows * heads / kv_heads exceeds %d", kKv4MaxRows);
        return KVP_ERR_ARG;
    }
    if (((uintptr_t)a.q | (uintptr_t)a.out) & 15 || (a.q_row_stride | a.q_batch_stride | a.out_row_stride |
                                                     a.out_batch_stride) % 8) {
        set_error("attn_kv4: q and out must be 16-byte aligned, strides multiples of 8 elements");
        return KVP_ERR_ARG;
    }
    if ((s.rows > 1 && a.q_row_stride < a.heads * 128LL) || (s.batch > 1 && a.q_batch_stride < 0) ||
        !apart(s, a.out_row_stride, a.out_batch_stride, a.heads * 128LL)) {
        set_error("attn_kv4: strides overlap (a row is heads * 128 elements)");
        return KVP_ERR_ARG;
    }
    return KVP_OK;
}

int launch_kv4_write(const Kv4Span& s, const Kv4Rows& r, int* d_status, cudaStream_t stream) {
    const int rc = check_kv4_rows(s, r, true);
    if (rc != KVP_OK || s.rows == 0 || s.batch == 0) return rc;
    return r.elem_bytes == 2 ? launch(s, r, d_status, stream, kv4_write_kernel<__nv_bfloat16>)
                             : launch(s, r, d_status, stream, kv4_write_kernel<float>);
}

int launch_kv4_read(const Kv4Span& s, const Kv4Rows& r, int* d_status, cudaStream_t stream) {
    const int rc = check_kv4_rows(s, r, false);
    if (rc != KVP_OK || s.rows == 0 || s.batch == 0) return rc;
    return r.elem_bytes == 2 ? launch(s, r, d_status, stream, kv4_read_kernel<__nv_bfloat16>)
                             : launch(s, r, d_status, stream, kv4_read_kernel<float>);
}

}  // namespace kvp
