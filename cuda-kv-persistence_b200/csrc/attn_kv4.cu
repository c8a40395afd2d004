// Attention over the 4-bit K/V cache (kv4.h): the kernel for few query rows
// and the launcher.
//
// For query row i of sequence b at position p = start + i in frame f = p / T,
//   out = sum_j 2^(x_j - m) v_j / sum_j 2^(x_j - m),
//   x_j = q . k_j * log2(e) / sqrt(128),
// over the keys j < min((f + 1) T, start + count) with j >= max(f - W + 1, 0) T
// (W = 0: every j) or j < S T.  No visible key: 0.  The query rows of a K/V
// head are its (row, query head of the group) pairs, r = i * group + g.
#include <algorithm>
#include <cstring>

#include "attn_kv4.cuh"
#include "kernels.h"
#include "kv4.h"
#include "sm100_ptx.h"

namespace kvp {

namespace {

using namespace kv4_dev;
using ptx::pack_f16;

// ------------------------------------------------- few query rows: mma.sync
// Bound by the cache's bytes: 144 a key and K/V head, against 2 * 128
// multiply-adds per query row.  Keys and dims go on the M side of
// m16n8k16 and the query rows on the N side, so up to 8 rows cost the same:
//   S^T[16 keys x 8] = K[16 x 128] Q^T,  O^T[16 dims x 8] += V^T[16 x 16] P^T.
// A lane's fragment of K is one 16-byte word of a row (a quarter of its dims;
// the order of the dims inside the sum is free, Q's fragment follows it), its
// fragment of V is two neighbouring rows of one 16-dim group, so both come
// straight from global memory, 512 consecutive bytes a warp, without shared
// memory on the way; movmatrix turns P^T into the second product's operand.
//
// One query row over 32768 keys x 12 heads (56.6 MB) takes 20.1 us with its
// join, 131072 keys x 12 heads 52.9 (4.3 TB/s).  The copies alone would take 41
// of those 53: turning codes into operands is about 530 instructions' issue
// cycles of the 1000 that a step of 32 keys takes, and the exponentials'
// latency, which the warps of a scheduler reach together, most of the rest.
// 16 ragged sequences of up to 8191 keys x 8 heads take 33.8 (3.4 TB/s): two
// splits each, the longest of 4096 keys where an even share of what runs at
// once is 2712.
// K and V through a ring in shared memory, four warps a CTA, the next step's
// first product between this one's exponentials and second: all measured
// 0 to 6 % slower.
constexpr int kWarps = 8;
constexpr int kDecThreads = kWarps * 32;
constexpr int kKeys = 32;                      // keys of one step of a warp
constexpr float kRise = 8.f;                   // how far a score may pass the running max, log2 units

// d += A B: bf16 (K Q^T) or fp16 (V^T P^T)
template <bool kHalf>
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
    if (kHalf)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 "
            "{%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 "
            "{%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
template <int NB>
struct RowsSmem {
    float o[kWarps][8 * NB][kKv4Head];
    float m[kWarps][8 * NB], l[kWarps][8 * NB];
    float jo[8 * NB][kKv4Head];                // the CTA's partial, read by its cluster
    float jm[8 * NB], jl[8 * NB];
};

// Shared memory of another CTA of the cluster.
__device__ __forceinline__ uint32_t peer(const void* p, int rank) {
    uint32_t a;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank));
    return a;
}
__device__ __forceinline__ float peer_f(const float* p, int rank) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(peer(p, rank)));
    return v;
}
__device__ __forceinline__ float4 peer_f4(const float* p, int rank) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(peer(p, rank)));
    return v;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// NB blocks of 8 query rows.
template <int NB>
__global__ void __launch_bounds__(kDecThreads, NB == 1 ? 2 : 1) attn_kv4_rows_kernel(const Kv4Params P) {
    extern __shared__ __align__(16) uint8_t smem_raw[];
    RowsSmem<NB>& sm = *reinterpret_cast<RowsSmem<NB>*>(smem_raw);
    const Kv4Span& s = P.span;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = lane >> 2, t = lane & 3;
    // CTA = (split, row tile, K/V head, sequence), split fastest
    uint32_t x = blockIdx.x;
    const int split = (int)(x % (uint32_t)P.splits);
    x /= (uint32_t)P.splits;
    const int tile = (int)(x % (uint32_t)P.row_tiles);
    x /= (uint32_t)P.row_tiles;
    const int h = (int)(x % (uint32_t)s.kv_heads), b = (int)(x / (uint32_t)s.kv_heads);
    int start, count;
    cudaGridDependencySynchronize();                  // what was queued before is complete and visible
    // What comes next, a join or the next call, may be launched (it waits for the
    // data).  Not where the splits are clusters: the next call's CTAs between
    // these made 38.7 us of 33.9 at 16 sequences of 8191 keys x 8 heads.  With one
    // split, and so no join, it is as long either way (20 sequences of 4096 keys
    // x 8 heads 36.7 us, 160 of 300 30.4; 31 keys x 8 heads 3.8, without 3.9).
    if (!P.cluster) cudaTriggerProgrammaticLaunchCompletion();
    if (!sequence(s, b, start, count)) {
        if (threadIdx.x == 0) atomicOr(P.status, KVP_STATUS_MAP);
        return;
    }
    const int rows = count * P.group, r0 = tile * 8 * NB;
    if (r0 >= rows) return;
    const int end = start + count;
    const Sees first = sees(P, start + r0 / P.group, end);
    const Sees last = sees(P, start + (min(r0 + 8 * NB, rows) - 1) / P.group, end);
    // key steps: those of the sinks below the window, then the window's
    const int b0 = first.lo / kKeys, nb = (last.hi + kKeys - 1) / kKeys - b0;
    const int na = min((min(P.sink_rows, last.hi) + kKeys - 1) / kKeys, b0);
    const int n = na + nb, per = (n + P.splits - 1) / P.splits;
    const int u0 = min(split * per, n), u1 = min(u0 + per, n);

    // Q^T fragments: step 2w + j of the 128 dims is dims 32t + 8w + 4j .. + 3
    uint32_t qf[NB][16];
#pragma unroll
    for (int i = 0; i < NB; ++i) {
        const int r = r0 + 8 * i + g;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            uint4 y = make_uint4(0, 0, 0, 0);
            if (r < rows)
                y = *reinterpret_cast<const uint4*>(q_row(P, b, h, r) + 32 * t + 8 * w);
            qf[i][4 * w] = y.x; qf[i][4 * w + 1] = y.y; qf[i][4 * w + 2] = y.z; qf[i][4 * w + 3] = y.w;
        }
    }
    float m[NB][2], l[NB][2], o[NB][8][4];       // m in score units (before the scale)
#pragma unroll
    for (int i = 0; i < NB; ++i) {
        m[i][0] = m[i][1] = -INFINITY;
        l[i][0] = l[i][1] = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) o[i][j][0] = o[i][j][1] = o[i][j][2] = o[i][j][3] = 0.f;
    }

    const uint32_t page_bytes = (uint32_t)s.kv_heads * kKv4PageHeadBytes;
    const uint8_t* head = static_cast<const uint8_t*>(s.pages) + h * kKv4PageHeadBytes;
    auto key_of = [&](int u) { return (u < na ? u : u - na + b0) * kKeys; };
    auto lookup = [&](int u) { return u < u1 ? page_of(s, b, key_of(u) / kKv4PageRows) : 0; };
    auto at = [&](int u, int page) {
        return head + (unsigned long long)(uint32_t)max(page, 0) * page_bytes +
               key_of(u) % kKv4PageRows / kKv4BlockRows * kKv4BlockBytes;
    };
    uint4 kc[4], vc[4];                            // codes of the step's four 8-row blocks
    uint32_t ks[4], vs[4];                         // their scale bytes
    auto load_k = [&](const uint8_t* p) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            kc[j] = *reinterpret_cast<const uint4*>(p + j * kKv4BlockBytes + lane * 16);
            ks[j] = *reinterpret_cast<const uint16_t*>(p + j * kKv4BlockBytes + kKv4KScale + lane * 2);
        }
    };
    auto load_v = [&](const uint8_t* p) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            vc[j] = *reinterpret_cast<const uint4*>(p + j * kKv4BlockBytes + kKv4VCode + lane * 16);
            vs[j] = *reinterpret_cast<const uint16_t*>(p + j * kKv4BlockBytes + kKv4VScale + lane * 2);
        }
    };

    // A warp takes every eighth step of the CTA's range.  The next step's K
    // is on its way from the moment the current K is used up, its V likewise,
    // and the page number after that one step longer: up to one step's 4.6 KB
    // a warp in flight, in that step's registers.
    bool any_bad = false;
    int u = u0 + warp, page = lookup(u), next = lookup(u + kWarps);
    if (u < u1) {
        load_k(at(u, page));
        load_v(at(u, page));
    }
    for (; u < u1; u += kWarps) {
        const bool more = u + kWarps < u1, bad = page < 0;
        const int key0 = key_of(u);
        page = next;
        const uint8_t* np = at(more ? u + kWarps : u, page);
        next = lookup(u + 2 * kWarps);
        any_bad |= bad;
        // S^T
        float c[NB][2][4];
#pragma unroll
        for (int i = 0; i < NB; ++i)
#pragma unroll
            for (int e = 0; e < 2; ++e) c[i][e][0] = c[i][e][1] = c[i][e][2] = c[i][e][3] = 0.f;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const uint32_t k0[4] = {kc[2 * e].x, kc[2 * e].y, kc[2 * e].z, kc[2 * e].w};
            const uint32_t k1[4] = {kc[2 * e + 1].x, kc[2 * e + 1].y, kc[2 * e + 1].z, kc[2 * e + 1].w};
#pragma unroll
            for (int d = 0; d < 2; ++d) {          // the quarter's two 16-dim groups
                const Scale2 s0 = scale2(__byte_perm(ks[2 * e], 0, d ? 0x4141 : 0x4040));
                const Scale2 s1 = scale2(__byte_perm(ks[2 * e + 1], 0, d ? 0x4141 : 0x4040));
#pragma unroll
                for (int w = 2 * d; w < 2 * d + 2; ++w) {
                    const uint32_t a0 = field<0>(k0[w], s0), a1 = field<0>(k1[w], s1);
                    const uint32_t a2 = field<1>(k0[w], s0), a3 = field<1>(k1[w], s1);
                    const uint32_t a4 = field<2>(k0[w], s0), a5 = field<2>(k1[w], s1);
                    const uint32_t a6 = field<3>(k0[w], s0), a7 = field<3>(k1[w], s1);
#pragma unroll
                    for (int i = 0; i < NB; ++i) {
                        mma16816<false>(c[i][e], a0, a1, a2, a3, qf[i][4 * w], qf[i][4 * w + 1]);
                        mma16816<false>(c[i][e], a4, a5, a6, a7, qf[i][4 * w + 2], qf[i][4 * w + 3]);
                    }
                }
            }
        }
        if (more) load_k(np);
        // masks
        if (bad || key0 + kKeys > first.hi || (key0 < last.lo && key0 + kKeys > P.sink_rows)) {
#pragma unroll
            for (int i = 0; i < NB; ++i)
#pragma unroll
                for (int a = 0; a < 2; ++a) {
                    const int r = min(r0 + 8 * i + 2 * t + a, rows - 1);
                    const Sees y = sees(P, start + r / P.group, end);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int key = key0 + g + 8 * e;
                        if (bad || key >= y.hi || (key < y.lo && key >= P.sink_rows))
                            c[i][e >> 1][a + 2 * (e & 1)] = -INFINITY;
                    }
                }
        }
        // The max moves only when some score passes it by more than 2^8 (or a
        // row sees its first key): P then stays below 2^15, inside fp16, and
        // most steps need no reduction over the keys.
        bool rise = false;
#pragma unroll
        for (int i = 0; i < NB; ++i)
#pragma unroll
            for (int a = 0; a < 2; ++a) {
                const float top = fmaxf(fmaxf(c[i][0][a], c[i][0][a + 2]), fmaxf(c[i][1][a], c[i][1][a + 2]));
                rise |= top > m[i][a] + P.rise;
            }
        if (__any_sync(0xffffffffu, rise)) {
#pragma unroll
            for (int i = 0; i < NB; ++i)
#pragma unroll
                for (int a = 0; a < 2; ++a) {
                    float top = fmaxf(fmaxf(c[i][0][a], c[i][0][a + 2]), fmaxf(c[i][1][a], c[i][1][a + 2]));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
                    const float up = fmaxf(m[i][a], top);
                    const float f = up == m[i][a] ? 1.f : ex2((m[i][a] - up) * P.scale_log2);
                    m[i][a] = up;
                    l[i][a] *= f;
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        o[i][j][a] *= f;
                        o[i][j][a + 2] *= f;
                    }
                }
        }
        uint32_t p[NB][4];
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            const float na0 = m[i][0] == -INFINITY ? 0.f : kPShift - m[i][0] * P.scale_log2;
            const float na1 = m[i][1] == -INFINITY ? 0.f : kPShift - m[i][1] * P.scale_log2;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float p0 = ex2(fmaf(c[i][e >> 1][2 * (e & 1)], P.scale_log2, na0));
                const float p1 = ex2(fmaf(c[i][e >> 1][2 * (e & 1) + 1], P.scale_log2, na1));
                l[i][0] += p0;
                l[i][1] += p1;
                // P to fp16 (a tensor-core operand): off by 2^-11 of itself at
                // most, or 2^-32 of the largest; the sum l keeps 32 bits
                p[i][e] = transpose8(pack_f16(p0, p1));
            }
        }
        // O^T: word d of a row holds dims 16g + 8d + 2i (low half's field i)
        // and + 1 (high half's); pairing two rows' halves puts two keys of one
        // dim into a register
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const uint4 v0 = vc[2 * e], v1 = vc[2 * e + 1];
            const VScale2 s0 = vscale2(__byte_perm(vs[2 * e], 0, 0x4140));
            const VScale2 s1 = vscale2(__byte_perm(vs[2 * e + 1], 0, 0x4140));
#pragma unroll
            for (int d = 0; d < 2; ++d) {
                const uint32_t e0 = __byte_perm(d ? v0.y : v0.x, d ? v0.w : v0.z, 0x5410);
                const uint32_t o0 = __byte_perm(d ? v0.y : v0.x, d ? v0.w : v0.z, 0x7632);
                const uint32_t e1 = __byte_perm(d ? v1.y : v1.x, d ? v1.w : v1.z, 0x5410);
                const uint32_t o1 = __byte_perm(d ? v1.y : v1.x, d ? v1.w : v1.z, 0x7632);
                auto step = [&](int j, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3) {
#pragma unroll
                    for (int i = 0; i < NB; ++i) mma16816<true>(o[i][j], a0, a1, a2, a3, p[i][2 * e], p[i][2 * e + 1]);
                };
                step(4 * d, vfield<0>(e0, s0), vfield<0>(o0, s0), vfield<0>(e1, s1), vfield<0>(o1, s1));
                step(4 * d + 1, vfield<1>(e0, s0), vfield<1>(o0, s0), vfield<1>(e1, s1), vfield<1>(o1, s1));
                step(4 * d + 2, vfield<2>(e0, s0), vfield<2>(o0, s0), vfield<2>(e1, s1), vfield<2>(o1, s1));
                step(4 * d + 3, vfield<3>(e0, s0), vfield<3>(o0, s0), vfield<3>(e1, s1), vfield<3>(o1, s1));
            }
        }
        if (more) load_v(np);
    }
    if (any_bad && lane == 0) atomicOr(P.status, KVP_STATUS_MAP);

    // Join the warps: l over the lanes of a column, then (O, m, l) over the warps.
#pragma unroll
    for (int i = 0; i < NB; ++i)
#pragma unroll
        for (int a = 0; a < 2; ++a) {
            l[i][a] += __shfl_xor_sync(0xffffffffu, l[i][a], 4);
            l[i][a] += __shfl_xor_sync(0xffffffffu, l[i][a], 8);
            l[i][a] += __shfl_xor_sync(0xffffffffu, l[i][a], 16);
            const int q = 8 * i + 2 * t + a;
            if (g == 0) {
                sm.m[warp][q] = m[i][a] * P.scale_log2;
                sm.l[warp][q] = l[i][a];
            }
#pragma unroll
            for (int j = 0; j < 8; j += 2)
                *reinterpret_cast<float4*>(&sm.o[warp][q][16 * g + 2 * j]) =
                    make_float4(o[i][j][a] * kVUnit, o[i][j][a + 2] * kVUnit, o[i][j + 1][a] * kVUnit,
                                o[i][j + 1][a + 2] * kVUnit);
        }
    __syncthreads();
    for (int e = threadIdx.x; e < 8 * NB * (kKv4Head / 4); e += kDecThreads) {
        const int q = e / (kKv4Head / 4), d = e % (kKv4Head / 4) * 4;
        const int r = r0 + q;
        if (r >= rows) continue;
        float top = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) top = fmaxf(top, sm.m[w][q]);
        float sum = 0.f;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            if (sm.l[w][q] == 0.f) continue;            // no key of this row
            const float f = ex2(sm.m[w][q] - top);
            sum += f * sm.l[w][q];
            const float4 y = *reinterpret_cast<const float4*>(&sm.o[w][q][d]);
            acc.x += f * y.x; acc.y += f * y.y; acc.z += f * y.z; acc.w += f * y.w;
        }
        if (P.cluster) {
            *reinterpret_cast<float4*>(&sm.jo[q][d]) = acc;
            if (d == 0) {
                sm.jm[q] = top;
                sm.jl[q] = sum;
            }
        } else {
            put(P, b, h, r, split, d, acc, top, sum);
        }
    }
    if (!P.cluster) return;
    // The splits are a cluster: each CTA joins its share of the rows' dims from
    // all of them, out of their shared memory.
    cluster_sync();
    const int items = 8 * NB * (kKv4Head / 4), share = (items + P.splits - 1) / P.splits;
    for (int e = split * share + threadIdx.x; e < min(items, (split + 1) * share); e += kDecThreads) {
        const int q = e / (kKv4Head / 4), d = e % (kKv4Head / 4) * 4;
        const int r = r0 + q;
        if (r >= rows) continue;
        float top = -INFINITY;
        for (int c = 0; c < P.splits; ++c) top = fmaxf(top, peer_f(&sm.jm[q], c));
        float sum = 0.f;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
        for (int c = 0; c < P.splits; ++c) {
            const float l1 = peer_f(&sm.jl[q], c), m1 = peer_f(&sm.jm[q], c);
            const float4 y = peer_f4(&sm.jo[q][d], c);
            const float f = l1 == 0.f ? 0.f : ex2(m1 - top);   // (no key of this row: O is 0)
            sum += f * l1;
            acc.x += f * y.x; acc.y += f * y.y; acc.z += f * y.z; acc.w += f * y.w;
        }
        store_out(P, b, h, r, d, acc, sum);
    }
    cluster_sync();                            // nobody leaves while its memory is read
}

// ------------------------------------------------------------- joining splits
// One row of kJoin warps' work, four dims a lane: the sum over its partials,
// rows at(0) .. at(splits - 1) of the workspace; a warp adds every kJoin-th.
// The lanes hold the partials' weights, so their loads wait for nothing but
// them.
template <class At>
__device__ __forceinline__ float add_partials(const Kv4Params& P, int splits, int first, int step, int lane, At&& at,
                                              float4& acc) {
    const float2* ml = reinterpret_cast<const float2*>(P.ws_ml);
    const float4* o = reinterpret_cast<const float4*>(P.ws_o) + lane;
    float top = -INFINITY, sum = 0.f;
    for (int c = lane; c < splits; c += 32) top = fmaxf(top, ml[at(c)].x);
#pragma unroll
    for (int x = 16; x; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
    for (int c0 = 0; c0 < splits; c0 += 32) {
        float f = 0.f;                                // stays 0 for a split without keys of this row
        if (c0 + lane < splits) {
            const float2 y = ml[at(c0 + lane)];
            if (y.y != 0.f) f = ex2(y.x - top);
            sum += f * y.y;
        }
        const int n = min(32, splits - c0);
#pragma unroll 4
        for (int c = first; c < n; c += step) {
            const float g = __shfl_sync(0xffffffffu, f, c);
            if (g != 0.f) {
                const float4 y = o[at(c0 + c) * (kKv4Head / 4)];
                acc.x += g * y.x; acc.y += g * y.y; acc.z += g * y.z; acc.w += g * y.w;
            }
        }
    }
#pragma unroll
    for (int x = 16; x; x >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
    return sum;
}

// Both joins are launched while the splits still run (programmatic stream
// serialization), so that their own launch costs no time after them.
template <int kJoin>
__global__ void __launch_bounds__(256) attn_kv4_join_kernel(const Kv4Params P) {
    __shared__ float4 part[8][32];
    const Kv4Span& s = P.span;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sub = warp % kJoin;
    const uint32_t w = blockIdx.x * (8 / kJoin) + warp / kJoin, max_rows = (uint32_t)P.max_rows;
    cudaGridDependencySynchronize();                  // the partials are complete and visible
    int start, count, r = 0, h = 0, b = 0;
    bool on = w < (uint32_t)(s.batch * s.kv_heads) * max_rows;   // (below 2^31: launch_attn_kv4)
    if (on) {
        r = (int)(w % max_rows);
        h = (int)(w / max_rows % (uint32_t)s.kv_heads);
        b = (int)(w / max_rows / (uint32_t)s.kv_heads);
        on = sequence(s, b, start, count) && r < count * P.group;
    }
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    float sum = 0.f;
    if (on)
        sum = add_partials(P, P.splits, sub, kJoin, lane, [&](int c) { return (long long)w * P.splits + c; }, acc);
    if (kJoin > 1) {
        part[warp][lane] = acc;
        __syncthreads();
        if (sub) return;
#pragma unroll
        for (int c = 1; c < kJoin; ++c) {
            const float4 y = part[warp + c][lane];
            acc.x += y.x; acc.y += y.y; acc.z += y.z; acc.w += y.w;
        }
    }
    if (on) store_out(P, b, h, r, 4 * lane, acc, sum);
}

// The units of the kernel for many rows that lie in several CTAs' chunks
// (Kv4Unit): P.join_ctas CTAs a unit, a warp a row at a time, or all eight
// warps where a unit is in many pieces.
__global__ void __launch_bounds__(256) attn_kv4_join_units_kernel(const Kv4Params P) {
    __shared__ float4 part[8][32];
    const int unit = (int)blockIdx.x / P.join_ctas, cta = (int)blockIdx.x % P.join_ctas;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    cudaGridDependencySynchronize();                  // the partials are complete, starts and counts visible
    const Kv4Unit u = unit_of(P, unit / P.span.kv_heads);
    if (u.pages == 0) return;
    const Kv4Pieces in = kv4_pieces(P.ws_unit[0], P.ws_unit[1 + unit], u.pages, P.ctas);
    const int c0 = in.first, splits = in.count;
    if (splits <= 1) return;                          // its rows are finished (or were given up)
    const int rows = min(u.rows - u.r0, 256), h = unit % P.span.kv_heads;
    auto add = [&](int row, int first, int step, float4& acc) {
        return add_partials(
            P, splits, first, step, lane, [&](int c) { return unit_slot(c0 + c, c == 0) * 256 + row; }, acc);
    };
    if (splits <= 8) {
        for (int row = cta * 8 + warp; row < rows; row += P.join_ctas * 8) {
            float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
            const float sum = add(row, 0, 1, acc);
            store_out(P, u.b, h, u.r0 + row, 4 * lane, acc, sum);
        }
        return;
    }
    for (int row = cta; row < rows; row += P.join_ctas) {
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        const float sum = add(row, warp, 8, acc);
        __syncthreads();                              // (the row before has been read)
        part[warp][lane] = acc;
        __syncthreads();
        if (warp) continue;
#pragma unroll
        for (int c = 1; c < 8; ++c) {
            const float4 y = part[c][lane];
            acc.x += y.x; acc.y += y.y; acc.z += y.z; acc.w += y.w;
        }
        store_out(P, u.b, h, u.r0 + row, 4 * lane, acc, sum);
    }
}

template <int NB>
cudaLaunchConfig_t rows_config(unsigned grid, int cluster, cudaLaunchAttribute (&attr)[2], cudaStream_t stream) {
    cudaLaunchConfig_t cfg = kv4_config(grid, kDecThreads, sizeof(RowsSmem<NB>), attr, stream);
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    return cfg;
}

// What a device runs at once: CTAs of the rows kernel, clusters of 2, 4 and 8
// of them (slot i: 2^i CTAs).  Asked once per device.
struct RowsFit {
    int at_once[PerDeviceOnce::kMaxDevices][4];
};
template <int NB>
int rows_fit(const int** at_once) {
    static PerDeviceOnce setup;
    static RowsFit fit;
    const int rc = setup([](int dev) -> int {
        KVP_CUDA(cudaFuncSetAttribute(attn_kv4_rows_kernel<NB>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                      (int)sizeof(RowsSmem<NB>)));
        for (int i = 0; i < 4; ++i) {
            cudaLaunchAttribute attr[2];
            const cudaLaunchConfig_t cfg = rows_config<NB>(1024, 1 << i, attr, nullptr);
            int n = 0;
            if (i == 0) {
                int sms = 0;
                KVP_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, attn_kv4_rows_kernel<NB>, kDecThreads,
                                                                       sizeof(RowsSmem<NB>)));
                KVP_CUDA(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
                n *= sms;
            } else {
                KVP_CUDA(cudaOccupancyMaxActiveClusters(&n, attn_kv4_rows_kernel<NB>, &cfg));
            }
            fit.at_once[dev][i] = n;
        }
        return KVP_OK;
    });
    int dev = 0;
    if (rc == KVP_OK) KVP_CUDA(cudaGetDevice(&dev));
    *at_once = fit.at_once[dev];
    return rc;
}

template <int NB>
int launch_rows(const Kv4Params& P, unsigned grid, cudaStream_t stream) {
    cudaLaunchAttribute attr[2];
    const cudaLaunchConfig_t cfg = rows_config<NB>(grid, P.cluster ? P.splits : 1, attr, stream);
    KVP_CUDA(cudaLaunchKernelEx(&cfg, attn_kv4_rows_kernel<NB>, P));
    return KVP_OK;
}

int sm_count() {
    int n = 148, dev = 0;
    if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
    return n > 0 ? n : 148;
}

}  // namespace

int launch_attn_kv4(const Kv4Span& s, const Kv4Attn& a, int* d_status, cudaStream_t stream) {
    const int rc = check_kv4_attn(s, a);
    if (rc != KVP_OK || s.rows == 0 || s.batch == 0) return rc;
    Kv4Params P;
    std::memset(&P, 0, sizeof P);
    P.span = s;
    P.attn = a;
    P.status = d_status;
    P.group = a.heads / s.kv_heads;
    P.max_rows = s.rows * P.group;
    const long long cap = (long long)s.map_stride * kKv4PageRows;
    // beyond the capacity a window or a sink hides nothing and a frame is all
    P.tokens = a.tokens;
    P.window_rows = a.window ? std::min<long long>((long long)a.window * a.tokens, 1LL << 31) : 0;
    P.sink_rows = (int)std::min<long long>((long long)a.sinks * a.tokens, cap);
    P.scale_log2 = 1.4426950408889634f / sqrtf((float)kKv4Head);
    P.rise = kRise / P.scale_log2;
    P.inv_group = 1.f / (float)P.group;

    // Keys that the rows of one tile can see, at most (starts on the device: the
    // capacity's).
    auto keys_of = [&](int tile_rows) {
        const long long all = s.starts ? cap : (long long)s.start + s.rows;
        return a.window ? std::min(all, tile_rows / P.group + 2 + (long long)a.tokens + P.window_rows + P.sink_rows)
                        : all;
    };
    // Up to 16 rows of a K/V head fit the N side of the mma.sync kernel; more go
    // through it 16 at a time as long as that is quicker.  It takes a thousand
    // 16-row x 32-key steps in 1.5 us after 7 us, the tcgen05 kernel a thousand
    // of 256 rows in 4.1 us after 17 (12 heads x 4064 keys, 64 rows: 17.7 us and
    // 27.2; 2 x 8 heads x 9064 keys, 32 rows: 19.3 and 37.0, 64 rows: 31.5 and
    // 38.5; 16 x 8 heads x 8064 keys, 32 rows: 97 and 145, 64 rows: 190 and 147).
    const double heads_k = (double)s.batch * s.kv_heads / kKeys * 1e-3;
    const bool tiles = P.max_rows > 16 &&
                       7 + (P.max_rows + 15) / 16 * heads_k * keys_of(16) * 1.5 >
                           17 + (P.max_rows + 255) / 256 * heads_k * keys_of(256) * 4.1;
    const int nb = P.max_rows > 8 ? 2 : 1, tile_rows = tiles ? 256 : 8 * nb;
    P.row_tiles = (P.max_rows + tile_rows - 1) / tile_rows;
    const long long units = (long long)s.batch * s.kv_heads * P.row_tiles;
    long long grid = units, slots = 0;   // slots: rows of the workspace
    const long long keys = keys_of(tile_rows);
    if (tiles) {
        // Units whose number does not divide over the SMs can be cut: the CTAs
        // share all units' pages evenly, for two pieces more a CTA, their partial
        // rows and the join, about 6 pages' time and a twentieth for each unit (12
        // heads x 1560 rows over 9360 keys, 84 units: 121 us, whole 167; over 3120
        // keys 60 and 63; 8 x 3 heads x 2000 rows, causal, 192 units: 72 and 45; 3
        // frames over 10920 of 12 heads, 228 units: 367 and 430).  Whole units,
        // longest first, take as long as the longest of each round, or the even
        // share and what the last ones stick out.
        P.splits = 1;
        const int sms = sm_count();
        const long long start = s.starts ? std::max(0LL, cap - s.rows) : s.start, pairs = (long long)s.batch * P.row_tiles;
        auto cost = [&](long long unit) {             // of a unit in the list (unit_of)
            const long long r0 = (P.row_tiles - 1 - unit / s.kv_heads / s.batch) * 256;
            const long long f0 = (start + r0 / P.group) / a.tokens * a.tokens + a.tokens;
            const long long last = start + (std::min<long long>(r0 + 256, P.max_rows) - 1) / P.group;
            const long long f1 = last / a.tokens * a.tokens + a.tokens;
            const long long lo = P.window_rows ? std::max(0LL, f0 - P.window_rows) / kKv4PageRows : 0;
            const long long hi = (std::min(f1, start + s.rows) + kKv4PageRows - 1) / kKv4PageRows;
            return hi - lo + std::min<long long>((P.sink_rows + kKv4PageRows - 1) / kKv4PageRows, lo) + kKv4UnitCost;
        };
        constexpr int kSamples = 16;
        double share = 0, rounds = 0;
        for (int i = 0; i < kSamples; ++i) share += (double)cost((2 * i + 1) * units / (2 * kSamples));
        share *= (double)units / (kSamples * sms);
        if (units < 8 * sms)
            for (long long u = 0; u < units; u += sms) rounds += (double)cost(u);
        P.chunked = units < 8 * sms && pairs <= kKv4ChunkPairs &&
                    units * (s.map_stride + kKv4UnitCost) < 0x7fffffffLL &&
                    std::min(rounds, share + (double)cost(units - 1)) > share + 6 + units / 20.0;
        if (P.chunked) {
            grid = sms;
            P.ctas = sms;
            slots = 2 * 256 * grid;
            // eight CTAs an SM, at least sixteen a unit (few units are in many pieces)
            P.join_ctas = (int)std::max(16LL, std::min(128LL, 8 * sms / units));
        }
    } else {
        const int* at_once = nullptr;
        const int rf = nb == 1 ? rows_fit<1>(&at_once) : rows_fit<2>(&at_once);
        if (rf != KVP_OK) return rf;
        // As many splits as the device runs at once (one more CTA would wait for
        // a second round: 37 us against 25 at 32768 keys x 12 heads), with a
        // step for each warp of a split at least.
        const long long steps = (keys + kKeys - 1) / kKeys;
        // Beyond 32 of them two steps for each warp: a long join costs more than
        // it saves (60000 keys of one head: 48 splits 13.4 us, 235 17.3).
        const long long most = std::max(std::min(32LL, (steps + kWarps - 1) / kWarps), steps / (4 * kWarps));
        const long long want = std::max<long long>(1, std::min(at_once[0] / units, most));
        // Splits that are a cluster join without workspace and second launch,
        // which is worth two steps more a warp (4099 keys x 12 heads: 8 in a
        // cluster 8.0 us, 12 and a join 8.4 and a second launch's host time;
        // 16 sequences of 8191 x 8 heads: 2 in a cluster 34.4, 2 and a join
        // 36.3; 32768 x 12 heads: 8 in a cluster 27.2, 24 and a join 20.0).
        auto a_warp = [&](long long c) { return (steps + c * kWarps - 1) / (c * kWarps); };
        int c = 0;
        for (int i = 3; i > 0 && !c; --i)
            if ((1 << i) <= want && units <= at_once[i]) c = 1 << i;
        P.cluster = c > 0 && a_warp(c) <= a_warp(want) + 2;
        P.splits = P.cluster ? c : (int)want;
        grid = units * P.splits;
        // (units * want is at most what the device runs at once)
        if (P.splits > 1 && !P.cluster) slots = (long long)s.batch * s.kv_heads * P.max_rows * P.splits;
    }
    if (grid > 0x7fffffffLL) {
        set_error("attn_kv4: too many rows for one launch");
        return KVP_ERR_ARG;
    }
    void* ws = nullptr;
    if (slots > 0) {
        const size_t rows_bytes = (size_t)slots * (kKv4Head + 2) * sizeof(float);
        cudaMemPool_t pool = nullptr;
        KVP_CUDA(workspace_pool(&pool));
        const size_t unit_bytes = P.chunked ? (size_t)(1 + units) * sizeof(int) : 0;
        KVP_CUDA(cudaMallocFromPoolAsync(&ws, rows_bytes + unit_bytes, pool, stream));
        P.ws_o = static_cast<float*>(ws);
        P.ws_ml = P.ws_o + slots * kKv4Head;
        P.ws_unit = reinterpret_cast<int*>(P.ws_ml + slots * 2);
    }
    int launched = tiles     ? launch_kv4_tiles(P, (unsigned)grid, stream)
                   : nb == 1 ? launch_rows<1>(P, (unsigned)grid, stream)
                             : launch_rows<2>(P, (unsigned)grid, stream);
    if (ws) {
        if (launched == KVP_OK) {
            cudaLaunchAttribute early;
            cudaLaunchConfig_t cfg = kv4_config(1, 256, 0, &early, stream);
            // a few splits: one warp a row; many: eight share them
            const long long rows = slots / P.splits;
            const bool many = P.splits > 8;
            cfg.gridDim = dim3((unsigned)(tiles ? units * P.join_ctas : many ? rows : (rows + 7) / 8));
            const cudaError_t e = tiles  ? cudaLaunchKernelEx(&cfg, attn_kv4_join_units_kernel, P)
                                  : many ? cudaLaunchKernelEx(&cfg, attn_kv4_join_kernel<8>, P)
                                         : cudaLaunchKernelEx(&cfg, attn_kv4_join_kernel<1>, P);
            if (e != cudaSuccess) launched = cuda_status(e, "attn_kv4 join");
        }
        const cudaError_t e = cudaFreeAsync(ws, stream);
        if (e != cudaSuccess && launched == KVP_OK) launched = cuda_status(e, "attn_kv4 workspace");
    }
    return launched;
}

}  // namespace kvp
