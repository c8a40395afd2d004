// Attention over the 4-bit K/V cache for many query rows: tcgen05 tensor
// cores, the cache expanded to 16 bits on its way into shared memory.
//
// Bound by the two products: 4 * 128 flops a (query row, key), against 144
// bytes a key that every 256 query rows read again from L2.  CTA = two
// 128-row query tiles of one K/V head (rows r = i * group + g, so grouped
// heads fill a tile) x a range of 128-key pages, one such unit after the
// other (Kv4Unit).  Warp roles (384 threads):
//   warps 0, 2, 3   expand the cache: units of 32 rows of K or V in turn,
//                   16-byte words from global memory (one unit ahead), fields
//                   to bf16 (K) and fp16 (V) in registers, 16-byte stores into
//                   the 128B-swizzled tiles that TMA would write from bf16 rows (K
//                   K-major, V MN-major); the words of half the lanes change
//                   places so that no store conflicts
//   warp 1          TMEM and the single-thread MMA issuer: S0_j, PV1_{j-1},
//                   S1_j, PV0_j
//   warps 4-7, 8-11 softmax of query tile 0 and 1, a row a thread, P kept in
//                   TMEM, the running max raised only where a tile has hidden
//                   keys or a row's sum overgrows
// TMEM: S0 | S1 | O0 | O1, 128 columns each; P overlays S's first 64.
// Every wait is bounded (sm100_ptx.h).
//
// One frame of 1560 rows over 32760 keys x 12 heads takes 344 us (913 TFLOP/s
// of products that are needed, 55 % of what a large bf16 GEMM reaches), three
// frames with a window of six and the first one kept 367, a token-causal
// prompt of 4097 rows x 24 heads on 8 with a window of 1024 94.1.  A page takes a
// CTA about 3500 cycles, 2048 of them MMAs: a query tile's S, its exponentials
// (1500; 1310 alone, 1024 of them MUFU's) and its PV follow one another, and
// what lies between them counts: 240 cycles before the exponentials, 280 from
// them to the issuer.  The roles' code shares one instruction cache: the seldom
// paths are loops, which made the frames 3 % faster and the prompt, a third of
// whose pages have hidden keys, 2 % slower.  Measured and slower: S in halves of
// 64 keys that land under the other half's softmax (+22 %), two threads a row
// (+15 %), an eighth of the exponentials on the FMA pipes (+1 to 3 %).
#include <cstring>

#include "attn_kv4.cuh"
#include "attn_mma_sm100.cuh"
#include "attn_softmax_sm100.cuh"
#include "kv4.h"

namespace kvp {

namespace {

using namespace ptx;
using namespace attn_dev;
using namespace kv4_dev;

constexpr int kThreads = 384;
constexpr int kBN = kKv4PageRows;             // keys of a tile
constexpr int kKStages = 2, kVStages = 3;
constexpr uint32_t kPanel = 128 * 128;        // one [128 rows][64 bf16] swizzled panel
constexpr uint32_t kTileBytes = 2 * kPanel;
constexpr int kRegsLow = 104, kRegsHigh = 200;   // warps 0-3, 4-11
static_assert(kRegsLow * 128 + 2 * kRegsHigh * 128 <= 65536, "register split exceeds the SM");
constexpr float kRedoSum = 32768.f;           // a tile row sum above this (2^8 shifted by kPShift) takes the new max
constexpr float kRaise = 1.f;                  // and a score above the max by this
constexpr int kUnits = 8;                     // of a tile: K rows 0-31, 32-63, .., then V's
constexpr int kExpanders = 3;

// Where a CTA is in its list of units, in costs: a unit costs kKv4UnitCost and
// its pages.  off: in the unit, left: what the CTA still takes, pos: in the list.
// Each role holds its own and moves it on by itself.
struct Work {
    int pair, head, off, left, pos;
};

// A piece for the softmax, which holds little of it in registers.  An expander,
// which is ahead, makes the entries (a piece's dozen divisions are 1,400 cycles
// that would stand between two pieces).
struct Turn {
    int batch, head, start, end, rows, row0, u0, n_tiles, rot, na, b0, two, partial, free_n, tile0;
    int qi0, qg0;               // row row0 is query head qg0 of the group, of the sequence's row qi0
};
constexpr int kTurns = 4;

struct __align__(1024) Smem {
    uint8_t q[2][kTileBytes];
    uint8_t k[kKStages][kTileBytes];
    uint8_t v[kVStages][kTileBytes];
    uint64_t bar_q[2];
    uint64_t bar_kfull[kKStages], bar_kempty[kKStages];
    uint64_t bar_vfull[kVStages], bar_vempty[kVStages];
    uint64_t bar_s_full[2];     // S_q(j) landed (and, by issue order, PV_q(j-1) too)
    uint64_t bar_p_full[2];     // P_q(j) in TMEM, S_q(j) read, O_q rescaled
    uint64_t bar_o_done[2];     // last PV_q landed
    uint64_t bar_turn[kTurns], bar_turn_empty[kTurns];
    uint64_t bar_mma_done;      // every issued MMA landed (TMEM may be freed)
    uint32_t tmem_base;
    int abort_flag;
    int scan[kThreads / 32];
    Work first;                 // where the CTA begins
    volatile int bad[8];        // K/V tile i of the CTA: its page is not in the pool (slot i % 8)
    Turn turn[kTurns];          // piece i: slot i % kTurns; n_tiles 0 ends the list
};

// Bits [0, n) set.
__device__ __forceinline__ uint32_t below(int n) { return n >= 32 ? 0xffffffffu : n <= 0 ? 0u : (1u << n) - 1u; }

__device__ __forceinline__ uint32_t next_word(uint32_t (&vis)[4]) {   // four calls go round
    const uint32_t v = vis[0];
    vis[0] = vis[1];
    vis[1] = vis[2];
    vis[2] = vis[3];
    vis[3] = v;
    return v;
}
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(
            addr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
// 128 columns of an S row of which vis says which are visible (32 a word; a
// warp's rows agree on most words): their max, and P with its sum, word by word.
// A hidden key's weight is 0: everything on MUFU, whose 2^-inf is 0.
__device__ __forceinline__ void load_visible(uint32_t s_addr, uint32_t vis, uint32_t (&y)[32]) {
    KVP_TMEM_LD32(s_addr, y);
    KVP_TMEM_WAIT_LD_DEP(y);
    if (__any_sync(0xffffffffu, vis != 0xffffffffu)) {
#pragma unroll
        for (int c = 0; c < 32; ++c)
            if (!(vis >> c & 1u)) y[c] = 0xFF800000u;   // -inf
    }
}
__device__ __forceinline__ float max_visible(uint32_t s_addr, uint32_t (&vis)[4]) {
    float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll 1
    for (int h = 0; h < 4; ++h) {
        const uint32_t v = next_word(vis);
        if (__all_sync(0xffffffffu, v == 0u)) continue;
        uint32_t y[32];
        load_visible(s_addr + 32 * h, v, y);
#pragma unroll
        for (int c = 0; c < 32; ++c) mx[c & 3] = fmaxf(mx[c & 3], __uint_as_float(y[c]));
    }
    return fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
}
// P goes to its place as it is made (columns [16 h, 16 h + 16): S's words h / 2
// and before, which have been read).
__device__ __forceinline__ float exp_visible(uint32_t s_addr, float m, float sl2, uint32_t (&vis)[4]) {
    float sum = 0.f;
#pragma unroll 1
    for (int h = 0; h < 4; ++h) {
        const uint32_t v = next_word(vis);
        uint32_t p[16];
        if (__all_sync(0xffffffffu, v == 0u)) {
#pragma unroll
            for (int c = 0; c < 16; ++c) p[c] = 0u;
        } else {
            uint32_t y[32];
            load_visible(s_addr + 32 * h, v, y);
            float part[2] = {0.f, 0.f};
#pragma unroll
            for (int c = 0; c < 32; c += 2) {
                const float p0 = ex2_approx(fmaf(__uint_as_float(y[c]), sl2, -m));
                const float p1 = ex2_approx(fmaf(__uint_as_float(y[c + 1]), sl2, -m));
                part[0] += p0;
                part[1] += p1;
                p[c >> 1] = pack_f16(p0, p1);
            }
            sum += part[0] + part[1];
        }
        tmem_st16(s_addr + 16 * h, p);
    }
    return sum;
}

// A word's eight values, K in bf16 and V in fp16, and a lane's four words as
// four 16-byte chunks of a tile.
__device__ __forceinline__ uint4 values(uint32_t w, const Scale2& s) {
    return make_uint4(field<0>(w, s), field<1>(w, s), field<2>(w, s), field<3>(w, s));
}
__device__ __forceinline__ uint4 values(uint32_t w, const VScale2& s) {
    return make_uint4(vfield<0>(w, s), vfield<1>(w, s), vfield<2>(w, s), vfield<3>(w, s));
}
template <class S>
__device__ __forceinline__ void expand4(uint8_t* tile, const uint32_t (&off)[4], uint32_t w0, uint32_t w1, uint32_t w2,
                                        uint32_t w3, const S& s01, const S& s23) {
    *reinterpret_cast<uint4*>(tile + off[0]) = values(w0, s01);
    *reinterpret_cast<uint4*>(tile + off[1]) = values(w1, s01);
    *reinterpret_cast<uint4*>(tile + off[2]) = values(w2, s23);
    *reinterpret_cast<uint4*>(tile + off[3]) = values(w3, s23);
}

constexpr int kMinPages = 2;                  // of a CTA's share, beside a unit's own cost

__device__ __forceinline__ void init_barriers(Smem& sm) {
    for (int q = 0; q < 2; ++q) {
        mbar_init(&sm.bar_q[q], 128);
        mbar_init(&sm.bar_s_full[q], 1);
        mbar_init(&sm.bar_p_full[q], 128);
        mbar_init(&sm.bar_o_done[q], 1);
    }
    for (int i = 0; i < kKStages; ++i) {
        mbar_init(&sm.bar_kfull[i], kUnits / 2);
        mbar_init(&sm.bar_kempty[i], 1);
    }
    for (int i = 0; i < kVStages; ++i) {
        mbar_init(&sm.bar_vfull[i], kUnits / 2);
        mbar_init(&sm.bar_vempty[i], 1);
    }
    for (int i = 0; i < kTurns; ++i) {
        mbar_init(&sm.bar_turn[i], 1);
        mbar_init(&sm.bar_turn_empty[i], 8);
    }
    mbar_init(&sm.bar_mma_done, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    fence_proxy_async_smem();
}

// A CTA's piece of a unit: its pages [u0, u0 + n_tiles).
// Its tiles go round from the first that every row sees whole: that gives each
// row its max, and the tiles with hidden keys need one pass like the others.
struct Piece {
    Kv4Unit u;
    int u0, n_tiles, rot;
    bool two;                                 // the second query tile has rows
    __device__ __forceinline__ Piece(const Kv4Params& P, const Work& w) {
        u = unit_of(P, w.pair);
        u0 = max(w.off - kKv4UnitCost, 0);
        n_tiles = max(min(w.off + w.left - kKv4UnitCost, u.pages) - u0, 0);   // (0: the list ends before the first page)
        two = u.r0 + 128 < u.rows;
        rot = free0() < free1() ? free0() : 0;
    }
    // tiles [free0, free1) in the order of their pages: every row sees them whole
    __device__ __forceinline__ int free0() const {
        return max(u.na + (u.last.lo + kBN - 1) / kBN - u.b0 - u0, 0);
    }
    __device__ __forceinline__ int free1() const { return min(u.na + u.first.hi / kBN - u.b0 - u0, n_tiles); }
    __device__ __forceinline__ int page_pos(int j) const {   // position page of tile j
        j += rot;
        const int i = u0 + (j < n_tiles ? j : j - n_tiles);
        return i < u.na ? i : i - u.na + u.b0;
    }
};

// The next piece of the list after one of a unit of `pages`.
__device__ __forceinline__ void advance(const Kv4Params& P, Work& w, int pages) {
    const int cost = min(kKv4UnitCost + pages - w.off, w.left);
    w.left -= cost;
    w.pos += cost;
    w.off = 0;
    if (++w.head == P.span.kv_heads && w.left > 0) {
        w.head = 0;
        do ++w.pair;
        while (unit_of(P, w.pair).pages == 0);        // left > 0: there is one
    }
}

// Row row0 + i (i < 256) of a piece: query head g of the group, the sequence's
// row.  (t + 1/2) / group is 2^-9 from an integer at least where group is below
// 256, far from fp32's rounding; above it the quotient is 0 or 1.
struct RowOf {
    int row, g;
};
__device__ __forceinline__ RowOf row_of(const Kv4Params& P, int qi0, int qg0, int i) {
    const int t = qg0 + i;
    const int q = P.group < 256 ? (int)(((float)t + 0.5f) * P.inv_group) : t >= P.group ? 1 : 0;
    return RowOf{qi0 + q, t - q * P.group};
}

__global__ void __launch_bounds__(kThreads, 1) attn_kv4_sm100_kernel(const __grid_constant__ Kv4Params P) {
    extern __shared__ uint8_t smem_raw[];
    cudaGridDependencySynchronize();              // (kv4_config)
    if (P.chunked) cudaTriggerProgrammaticLaunchCompletion();   // the join may be launched; it waits for the data
    if (reinterpret_cast<uintptr_t>(smem_raw) & 1023) {
        if (threadIdx.x == 0) atomicOr(P.status, KVP_STATUS_ALIGN);
        return;
    }
    Smem& sm = *reinterpret_cast<Smem*>(smem_raw);
    const Kv4Span& s = P.span;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    // Where this CTA's work begins, and how many pages it takes.
    int left = 0;
    if (P.chunked) {
        // prefix sums of the pairs' costs, three pairs a thread
        const int pairs = P.row_tiles * s.batch;
        int n[3], mine = 0;
#pragma unroll
        for (int i = 0; i < 3; ++i) {
            const int p = 3 * (int)threadIdx.x + i;
            n[i] = p < pairs ? unit_of(P, p).pages : 0;
            if (n[i] > 0) n[i] += kKv4UnitCost;
            mine += n[i];
        }
        int upto = mine;
#pragma unroll
        for (int d = 1; d < 32; d *= 2) {
            const int v = __shfl_up_sync(0xffffffffu, upto, d);
            if (lane >= d) upto += v;
        }
        if (lane == 31) sm.scan[warp] = upto;
        __syncthreads();
        int before = upto - mine, all = 0;
        for (int w = 0; w < kThreads / 32; ++w) {
            if (w < warp) before += sm.scan[w];
            all += sm.scan[w];
        }
        all *= s.kv_heads;
        const int chunk = max((all + (int)gridDim.x - 1) / (int)gridDim.x, kKv4UnitCost + kMinPages);
        const int pos = (int)min((long long)blockIdx.x * chunk, (long long)all);
        left = min(chunk, all - pos);
        if (blockIdx.x == 0 && threadIdx.x == 0) P.ws_unit[0] = chunk;
#pragma unroll
        for (int i = 0; i < 3; ++i) {
            const int r = pos - before * s.kv_heads;   // into this pair's kv_heads units
            if (left > 0 && r >= 0 && r < n[i] * s.kv_heads) {
                sm.first = Work{3 * (int)threadIdx.x + i, r / n[i], r % n[i], left, pos};
            }
            before += n[i];
        }
    } else {
        const int pair = (int)(blockIdx.x / (uint32_t)s.kv_heads);
        left = unit_of(P, pair).pages;
        if (left > 0) left += kKv4UnitCost;
        if (threadIdx.x == 0) sm.first = Work{pair, (int)(blockIdx.x % (uint32_t)s.kv_heads), 0, left, 0};
    }
    // the refused sequences are reported once
    if (threadIdx.x == 0)
        for (int i = (int)blockIdx.x; i < s.batch; i += (int)gridDim.x)
            if (unit_of(P, i).refused) atomicOr(P.status, KVP_STATUS_MAP);
    if (left == 0) return;
    if (threadIdx.x == 0) {
        sm.abort_flag = 0;
        init_barriers(sm);
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                         smem_u32(&sm.tmem_base)), "r"(512));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sm.tmem_base;

    // Every role goes through the pieces by itself; the barriers' phases run on
    // from one to the next, so that the first tiles of a piece are expanded
    // while the one before ends.
    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsLow));
        Work w = sm.first;
        if (warp != 1) {
            // ============================ expanders ===========================
            const int g = lane >> 2, t = lane & 3;
            // K: row g of a block, quarter t, words in the order i ^ (t & 2).
            // V: rows 2t and 2t + 1, group g, words of a row in the order e ^ (g & 1).
            uint32_t koff[4], voff[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                koff[i] = (t >> 1) * kPanel + g * 128 + ((((t & 1) * 4) ^ (t & 2) ^ g ^ i) << 4);
                voff[i] = (g >> 2) * kPanel + (2 * t + (i >> 1)) * 128 +
                          ((((g & 3) * 2) ^ (g & 1) ^ (2 * t) ^ (i >> 1) ^ (i & 1)) << 4);
            }
            const uint32_t page_bytes = (uint32_t)s.kv_heads * kKv4PageHeadBytes;
            const int turn0 = warp == 0 ? 0 : warp - 1;    // its first unit of a piece
            // slot `turn` is free: the eight softmax warps are done with the piece before
            auto next_turn = [&](int turn) {
                return warp_wait(&sm.bar_turn_empty[turn % kTurns], (uint32_t)(turn / kTurns & 1) ^ 1u, sm, P.status);
            };
            bool ok = true;
            int turn = 0;
            for (int tile0 = 0; ok && w.left > 0;) {
                const Piece pc(P, w);
                if (pc.n_tiles == 0) break;
                if (warp == 0) ok = next_turn(turn);
                if (!ok) break;
                if (warp == 0 && lane == 0) {
                    Turn& t = sm.turn[turn % kTurns];
                    t.batch = pc.u.b;
                    t.head = w.head;
                    t.start = pc.u.start;
                    t.end = pc.u.end;
                    t.rows = pc.u.rows;
                    t.row0 = pc.u.r0;
                    t.u0 = pc.u0;
                    t.n_tiles = pc.n_tiles;
                    t.rot = pc.rot;
                    t.na = pc.u.na;
                    t.b0 = pc.u.b0;
                    t.two = pc.two;
                    t.partial = pc.n_tiles < pc.u.pages;
                    t.free_n = max(pc.free1() - pc.free0(), 0);
                    t.tile0 = tile0;
                    t.qi0 = pc.u.r0 / P.group;
                    t.qg0 = pc.u.r0 % P.group;
                    if (P.chunked && pc.u0 == 0)
                        P.ws_unit[1 + w.pair * s.kv_heads + w.head] = w.pos - w.off + kKv4UnitCost;
                    mbar_arrive(&sm.bar_turn[turn % kTurns]);
                }
                ++turn;
                const int units = pc.n_tiles * kUnits;
                const uint8_t* pool = static_cast<const uint8_t*>(s.pages) + w.head * kKv4PageHeadBytes;
                auto lookup = [&](int n) { return n < units ? page_of(s, pc.u.b, pc.page_pos(n / kUnits)) : 0; };
                uint4 c[4];
                uint32_t sc[4];
                auto load = [&](int n, int page) {
                    const int part = (n >> 2) & 1;
                    const uint8_t* p = pool + (unsigned long long)(uint32_t)max(page, 0) * page_bytes +
                                       (n & 3) * 4 * kKv4BlockBytes;
                    const uint8_t* at = p + (part ? kKv4VCode : 0) + lane * 16;
                    const uint8_t* ps = p + (part ? kKv4VScale : kKv4KScale) + lane * 2;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        c[i] = *reinterpret_cast<const uint4*>(at + i * kKv4BlockBytes);
                        sc[i] = *reinterpret_cast<const uint16_t*>(ps + i * kKv4BlockBytes);
                    }
                };
                int n = turn0, page = lookup(n), page1 = lookup(n + kExpanders);
                load(n, page);
                for (; n < units; n += kExpanders) {
                    const bool bad = page < 0;
                    page = page1;
                    page1 = lookup(n + 2 * kExpanders);
                    uint4 cc[4];
                    uint32_t ss[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        cc[i] = c[i];
                        ss[i] = sc[i];
                    }
                    if (n + kExpanders < units) load(n + kExpanders, page);
                    const int j = tile0 + n / kUnits, part = (n >> 2) & 1;
                    const int st = part ? j % kVStages : j % kKStages;
                    const uint32_t ph = (uint32_t)(part ? j / kVStages : j / kKStages) & 1u;
                    if (!warp_wait(part ? &sm.bar_vempty[st] : &sm.bar_kempty[st], ph ^ 1u, sm, P.status)) {
                        ok = false;
                        break;
                    }
                    if (n % kUnits == 0 && lane == 0) {
                        sm.bad[j % 8] = bad;
                        if (bad) atomicOr(P.status, KVP_STATUS_MAP);
                    }
                    // 8 rows are 1024 bytes of a panel
                    uint8_t* tile = (part ? sm.v[st] : sm.k[st]) + (n & 3) * 4 * 1024;
                    if (part) {
                        const bool swap = g & 1;
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const VScale2 s0 = vscale2(__byte_perm(ss[i], 0, 0x4040));
                            const VScale2 s1 = vscale2(__byte_perm(ss[i], 0, 0x4141));
                            expand4(tile + i * 1024, voff, swap ? cc[i].y : cc[i].x, swap ? cc[i].x : cc[i].y,
                                    swap ? cc[i].w : cc[i].z, swap ? cc[i].z : cc[i].w, s0, s1);
                        }
                    } else {
                        const bool swap = t & 2;
                        const uint32_t lo = swap ? 0x4141 : 0x4040, hi = swap ? 0x4040 : 0x4141;
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const Scale2 s0 = scale2(__byte_perm(ss[i], 0, lo));
                            const Scale2 s1 = scale2(__byte_perm(ss[i], 0, hi));
                            expand4(tile + i * 1024, koff, swap ? cc[i].z : cc[i].x, swap ? cc[i].w : cc[i].y,
                                    swap ? cc[i].x : cc[i].z, swap ? cc[i].y : cc[i].w, s0, s1);
                        }
                    }
                    fence_proxy_async_smem();   // each lane's stores, before the arrival that covers them
                    __syncwarp();
                    if (lane == 0) mbar_arrive(part ? &sm.bar_vfull[st] : &sm.bar_kfull[st]);
                }
                tile0 += pc.n_tiles;
                advance(P, w, pc.u.pages);
            }
            if (warp == 0 && ok && next_turn(turn) && lane == 0) {
                sm.turn[turn % kTurns].n_tiles = 0;
                mbar_arrive(&sm.bar_turn[turn % kTurns]);
            }
        } else {
            // ============================ MMA issuer ==========================
            if (lane == 0) {
                constexpr uint32_t idS = idesc_bf16(false);
                constexpr uint32_t idO = idesc_f16(true);
                constexpr uint64_t kStageDesc = kTileBytes >> 4;
                const uint64_t dq0 = sw128_desc(smem_u32(sm.q[0]), 16, 1024);
                const uint64_t dq1 = sw128_desc(smem_u32(sm.q[1]), 16, 1024);
                const uint64_t dk = sw128_desc(smem_u32(sm.k[0]), 16, 1024);
                const uint64_t dv = sw128_desc(smem_u32(sm.v[0]), kPanel, 1024);
                const uint32_t s0_tm = tmem, s1_tm = tmem + 128u, o0_tm = tmem + 256u, o1_tm = tmem + 384u;
                uint32_t ks = 0, kph = 0, vs = 0, vph = 0, pvs = 0;
                uint32_t q0_ph = 0, q1_ph = 0, p0_ph = 0, p1_ph = 0;
                bool ok = true;
                while (ok && w.left > 0) {
                    const Piece pc(P, w);
                    const int n_tiles = pc.n_tiles;
                    const bool two = pc.two;
                    if (n_tiles == 0) break;
                    ok = mbar_wait(&sm.bar_q[0], q0_ph, sm, P.status);
                    if (ok && two) ok = mbar_wait(&sm.bar_q[1], q1_ph, sm, P.status);
                    bool k_known = false;
                    // While the first six MMAs of a GEMM are queued, the barriers of
                    // the next GEMM are tested without blocking.
                    for (int j = 0; ok && j < n_tiles; ++j) {
                        if (!k_known && !(ok = mbar_wait(&sm.bar_kfull[ks], kph, sm, P.status))) break;
                        tc_fence_after();
                        const uint64_t kd = dk + ks * kStageDesc;
                        const bool pv1 = two && j > 0;
                        tc_gemm_ss_head(s0_tm, dq0, kd, idS);
                        const bool pv1_ready = pv1 && mbar_test(&sm.bar_p_full[1], p1_ph);
                        tc_gemm_ss_tail(s0_tm, dq0, kd, idS);
                        tc_commit(&sm.bar_s_full[0]);
                        if (pv1) {
                            if (!pv1_ready && !(ok = mbar_wait(&sm.bar_p_full[1], p1_ph, sm, P.status))) break;
                            tc_fence_after();
                            const uint64_t vd = dv + pvs * kStageDesc;
                            tc_gemm_ts_head(o1_tm, s1_tm, vd, idO, j > 1 ? 1u : 0u);
                            tc_gemm_ts_tail(o1_tm, s1_tm, vd, idO);
                            p1_ph ^= 1u;
                        }
                        bool pv0_ready = false;
                        if (two) {
                            tc_gemm_ss_head(s1_tm, dq1, kd, idS);
                            pv0_ready = mbar_test(&sm.bar_vfull[vs], vph) && mbar_test(&sm.bar_p_full[0], p0_ph);
                            tc_gemm_ss_tail(s1_tm, dq1, kd, idS);
                            tc_commit(&sm.bar_s_full[1]);
                        }
                        const uint32_t ks_n = ks + 1 == kKStages ? 0u : ks + 1;
                        const uint32_t kph_n = ks + 1 == kKStages ? kph ^ 1u : kph;
                        if (!pv0_ready && !(ok = mbar_wait(&sm.bar_vfull[vs], vph, sm, P.status) &&
                                                 mbar_wait(&sm.bar_p_full[0], p0_ph, sm, P.status))) break;
                        tc_fence_after();
                        const uint64_t vd = dv + vs * kStageDesc;
                        tc_gemm_ts_head(o0_tm, s0_tm, vd, idO, j > 0 ? 1u : 0u);
                        k_known = j + 1 < n_tiles && mbar_test(&sm.bar_kfull[ks_n], kph_n);
                        tc_gemm_ts_tail(o0_tm, s0_tm, vd, idO);
                        p0_ph ^= 1u;
                        pvs = vs;
                        if (++vs == kVStages) { vs = 0; vph ^= 1u; }
                        ks = ks_n;
                        kph = kph_n;
                    }
                    if (ok) {
                        tc_commit(&sm.bar_o_done[0]);
                        if (two && (ok = mbar_wait(&sm.bar_p_full[1], p1_ph, sm, P.status))) {
                            tc_fence_after();
                            const uint64_t vd = dv + pvs * kStageDesc;
                            tc_gemm_ts_head(o1_tm, s1_tm, vd, idO, n_tiles > 1 ? 1u : 0u);
                            tc_gemm_ts_tail(o1_tm, s1_tm, vd, idO);
                            tc_commit(&sm.bar_o_done[1]);
                            p1_ph ^= 1u;
                            q1_ph ^= 1u;
                        }
                        q0_ph ^= 1u;
                    }
                    advance(P, w, pc.u.pages);
                }
                // Drain: every issued MMA lands before TMEM is freed.
                tc_commit(&sm.bar_mma_done);
                const unsigned long long t0 = globaltimer();
                while (!mbar_try_wait(&sm.bar_mma_done, 0) && globaltimer() - t0 < kWaitNs) {
                }
            }
            __syncwarp();
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsHigh));
        // ========================== softmax + epilogue ========================
        const int qt = (warp - 4) >> 2;
        const int row = (warp & 3) * 32 + lane;        // query row in tile == TMEM lane
        const uint32_t s_tm = tmem + ((uint32_t)((warp & 3) * 32) << 16) + 128u * qt;
        const uint32_t o_tm = s_tm + 256u;
        uint32_t s_ph = 0, o_ph = 0;
        bool ok = true;
        for (int turn = 0; ok; ++turn) {
            if (!warp_wait(&sm.bar_turn[turn % kTurns], (uint32_t)(turn / kTurns) & 1u, sm, P.status)) break;
            const volatile Turn& pc = sm.turn[turn % kTurns];
            const int n_tiles = pc.n_tiles;
            if (n_tiles == 0) break;
            if (qt == 1 && !pc.two) {                      // this query tile has no rows
                __syncwarp();
                if (lane == 0) mbar_arrive(&sm.bar_turn_empty[turn % kTurns]);
                continue;
            }
            const int h = pc.head, r0 = pc.row0, rows = pc.rows, qi0 = pc.qi0, qg0 = pc.qg0;
            const bool releaser = (threadIdx.x & 127) == 0 && qt == pc.two;
            // A row past the last (Q is 0, never stored) takes every key; a warp of
            // such rows does no softmax.
            Sees mine = {0, 0};
            {
                // Q: this warp's 32 rows, two rows a pass, 16 lanes on a row's 256 bytes;
                // rows past the last are zero
                const int mine0 = 128 * qt + (warp & 3) * 32, rw = r0 + mine0, sub = lane >> 4, chunk = lane & 15;
                const __nv_bfloat16* src = static_cast<const __nv_bfloat16*>(P.attn.q) +
                                           pc.batch * P.attn.q_batch_stride +
                                           (long long)h * P.group * kKv4Head + 8 * chunk;
                uint8_t* dst = sm.q[qt] + (chunk >> 3) * kPanel;
#pragma unroll
                for (int k = 0; k < 32; k += 2) {
                    const bool in = rw + sub + k < rows;
                    const RowOf y = row_of(P, qi0, qg0, mine0 + sub + k);
                    const __nv_bfloat16* at = src + y.row * P.attn.q_row_stride + (long long)y.g * kKv4Head;
                    cp_async16(dst + sw128_off((warp & 3) * 32 + sub + k, chunk & 7), in ? at : P.attn.q,
                               in ? 16u : 0u);
                }
                cp_async_wait_all();
                fence_proxy_async_smem();
                mbar_arrive(&sm.bar_q[qt]);
                if (rw + lane < rows) mine = sees(P, pc.start + row_of(P, qi0, qg0, mine0 + lane).row, pc.end);
                else if (rw < rows) mine.hi = 0x7fffffff;
            }
            float m_run = -INFINITY, l_run = 0.f;          // m in log2 units
            bool warm = false;                             // every row of the warp has seen a key
            const int free_n = pc.free_n, tile0 = pc.tile0;
            for (int j = 0; j < n_tiles; ++j) {
                if (!warp_wait(&sm.bar_s_full[qt], s_ph, sm, P.status)) { ok = false; break; }
                s_ph ^= 1u;
                tc_fence_after();
                // (the flag is written before the K tile is full, which S waits for; the
                // tile that takes its slot cannot begin before this one's P is there)
                const bool bad = sm.bad[(tile0 + j) % 8];
                // S landing for the last query tile of a step means every MMA issued
                // before has landed: K(j) and V(j-1) are no longer read.
                if (releaser) {
                    mbar_arrive(&sm.bar_kempty[(tile0 + j) % kKStages]);
                    if (j > 0) mbar_arrive(&sm.bar_vempty[(tile0 + j - 1) % kVStages]);
                }
                if (__all_sync(0xffffffffu, mine.hi == 0)) {   // no row: what P's columns hold is never stored
                    tc_fence_before();
                    mbar_arrive(&sm.bar_p_full[qt]);
                    continue;
                }
                uint32_t vis[4] = {0xffffffffu, 0xffffffffu, 0xffffffffu, 0xffffffffu};
                bool gone = false, some_gone = false;      // (a row that sees nothing here)
                bool plain = warm;                         // each row sees all or nothing, and has a max
                if (__builtin_expect(bad || j >= free_n, 0)) {
                    // columns [0, sink) and [lo, hi) are visible
                    int u = j + pc.rot;
                    u = pc.u0 + (u < n_tiles ? u : u - n_tiles);
                    const int key0 = (u < pc.na ? u : u - pc.na + pc.b0) * kBN;
                    const int hi = bad ? 0 : mine.hi - key0;
                    const int sink = P.sink_rows - key0, lo = mine.lo - key0;
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        vis[e] = below(hi - 32 * e) & (~below(lo - 32 * e) | below(sink - 32 * e));
                    const bool whole = (vis[0] & vis[1] & vis[2] & vis[3]) == 0xffffffffu;
                    gone = (vis[0] | vis[1] | vis[2] | vis[3]) == 0u;
                    some_gone = __any_sync(0xffffffffu, gone);
                    plain = __all_sync(0xffffffffu, gone || (whole && m_run != -INFINITY)) &&
                            !__all_sync(0xffffffffu, gone);
                }
                // P (fp16: off by 2^-11 of itself at most, or 2^-32 of the largest;
                // the sum keeps 32 bits) -> the first 64 columns of S_q, key 2c in
                // the low half.  Nearly every tile goes the first way, against the
                // running max, which is laid out without a jump (700 cycles stood
                // between S and the first exponential before).
                float rsum = 0.f;
                if (__builtin_expect(plain, 1)) {
                    uint32_t pk[64];
                    rsum = exp_row<false, 4, 0u, true>(s_tm, m_run - kPShift, P.scale_log2, kBN, pk);
                    if (__builtin_expect(some_gone, 0)) {
                        if (gone) {
                            rsum = 0.f;
#pragma unroll
                            for (int c = 0; c < 64; ++c) pk[c] = 0u;
                        }
                    }
                    plain = __all_sync(0xffffffffu, rsum <= kRedoSum);
                    if (__builtin_expect(plain, 1)) {
                        KVP_TMEM_ST32(s_tm, pk);
                        KVP_TMEM_ST32(s_tm + 32, (pk + 32));
                    }
                }
                if (__builtin_expect(!plain, 0)) {
                    // Hidden keys, a row's first key or a sum that overgrows (some
                    // score is above the max by 1 then): the tile's max first.
                    const float top = max_visible(s_tm, vis) * P.scale_log2;
                    const float m_new = top > m_run + kRaise ? top : m_run;
                    // (a row without keys keeps max -inf: subtract 0)
                    rsum = exp_visible(s_tm, (m_new == -INFINITY ? 0.f : m_new) - kPShift, P.scale_log2, vis);
                    const float alpha = m_new == m_run ? 1.f : ex2_approx(m_run - m_new);
                    l_run *= alpha;
                    m_run = m_new;
                    warm = __all_sync(0xffffffffu, m_run != -INFINITY);
                    if (j > 0 && __any_sync(0xffffffffu, alpha != 1.f)) {
                        // O_q holds PV_q(j-1) (complete: it was issued before S_q(j))
#pragma unroll 1
                        for (int c4 = 0; c4 < 4; ++c4) {
                            uint32_t o[32];
                            KVP_TMEM_LD32(o_tm + 32 * c4, o);
                            KVP_TMEM_WAIT_LD_DEP(o);
#pragma unroll
                            for (int c = 0; c < 32; ++c)
                                o[c] = __float_as_uint(__uint_as_float(o[c]) * alpha);
                            KVP_TMEM_ST32(o_tm + 32 * c4, o);
                        }
                    }
                }
                l_run += rsum;
                tmem_wait_st();
                tc_fence_before();
                mbar_arrive(&sm.bar_p_full[qt]);
            }
            // A warp's rows go out through its own rows of the Q tile (every S
            // has landed): a row's 128 bytes by eight lanes, four rows a store.
            const int er = pc.rows, r = pc.row0 + 128 * qt + row;
            const bool partial = pc.partial;
            if (!ok || !warp_wait(&sm.bar_o_done[qt], o_ph, sm, P.status)) {
                ok = false;
                break;
            }
            o_ph ^= 1u;
            tc_fence_after();
            if (releaser) mbar_arrive(&sm.bar_vempty[(tile0 + n_tiles - 1) % kVStages]);
            uint8_t* stage = sm.q[qt] + (warp & 3) * 32 * 128;
            const int rw = r - lane, sub = lane >> 3, chunk = lane & 7;
            const float inv = l_run == 0.f ? 0.f : kVUnit / l_run;      // a row without keys is 0
            // row rw + sub + 4 i of the workspace or of the output
            const long long slot = unit_slot((int)blockIdx.x, pc.u0 == 0) * 256 + 128 * qt + (warp & 3) * 32;
            if (partial)
                *reinterpret_cast<float2*>(P.ws_ml + (slot + lane) * 2) = make_float2(m_run, l_run);
            uint8_t* ws = reinterpret_cast<uint8_t*>(P.ws_o + (slot + sub) * kKv4Head) + 16 * chunk;
            uint8_t* out = reinterpret_cast<uint8_t*>(static_cast<__nv_bfloat16*>(P.attn.out) +
                                                      pc.batch * P.attn.out_batch_stride +
                                                      (long long)h * P.group * kKv4Head) + 16 * chunk;
            const int step = partial ? 32 : 64;                         // dims that make 128 bytes
#pragma unroll 1
            for (int c0 = 0; c0 < kKv4Head; c0 += step) {
                uint32_t o[32];
                KVP_TMEM_LD32(o_tm + c0, o);
                KVP_TMEM_WAIT_LD_DEP(o);
                if (partial) {
#pragma unroll
                    for (int c = 0; c < 8; ++c)
                        *reinterpret_cast<uint4*>(stage + lane * 128 + ((c ^ (lane & 7)) << 4)) =
                            make_uint4(__float_as_uint(__uint_as_float(o[4 * c]) * kVUnit),
                                       __float_as_uint(__uint_as_float(o[4 * c + 1]) * kVUnit),
                                       __float_as_uint(__uint_as_float(o[4 * c + 2]) * kVUnit),
                                       __float_as_uint(__uint_as_float(o[4 * c + 3]) * kVUnit));
                } else {
#pragma unroll 1
                    for (int e = 0; e < 2; ++e) {
                        if (e) {
                            KVP_TMEM_LD32(o_tm + c0 + 32, o);
                            KVP_TMEM_WAIT_LD_DEP(o);
                        }
#pragma unroll
                        for (int c = 0; c < 4; ++c) {
                            uint4 y;
                            y.x = pack_bf16(__uint_as_float(o[8 * c]) * inv, __uint_as_float(o[8 * c + 1]) * inv);
                            y.y = pack_bf16(__uint_as_float(o[8 * c + 2]) * inv, __uint_as_float(o[8 * c + 3]) * inv);
                            y.z = pack_bf16(__uint_as_float(o[8 * c + 4]) * inv, __uint_as_float(o[8 * c + 5]) * inv);
                            y.w = pack_bf16(__uint_as_float(o[8 * c + 6]) * inv, __uint_as_float(o[8 * c + 7]) * inv);
                            *reinterpret_cast<uint4*>(stage + lane * 128 + (((4 * e + c) ^ (lane & 7)) << 4)) = y;
                        }
                    }
                }
                __syncwarp();
#pragma unroll 4
                for (int i = 0; i < 8; ++i) {
                    const int k = 4 * i + sub;
                    const uint4 y = *reinterpret_cast<const uint4*>(stage + k * 128 + ((chunk ^ (k & 7)) << 4));
                    uint8_t* dst = ws + i * (4 * kKv4Head * 4) + c0 * 4;
                    if (!partial) {
                        const RowOf x = row_of(P, qi0, qg0, 128 * qt + (warp & 3) * 32 + k);
                        dst = out + (x.row * P.attn.out_row_stride + (long long)x.g * kKv4Head + c0) * 2;
                    }
                    if (rw + k < er) *reinterpret_cast<uint4*>(dst) = y;
                }
                __syncwarp();
            }
            tc_fence_before();                             // O is read: the next piece may begin to fill it
            if (lane == 0) mbar_arrive(&sm.bar_turn_empty[turn % kTurns]);
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 1) {
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
    }
}

}  // namespace

int launch_kv4_tiles(const Kv4Params& P, unsigned grid, cudaStream_t stream) {
    static PerDeviceOnce setup;
    const int smem = (int)sizeof(Smem);
    const int rc = setup([&](int dev) -> int {
        int optin = 0;
        KVP_CUDA(cudaDeviceGetAttribute(&optin, cudaDevAttrMaxSharedMemoryPerBlockOptin, dev));
        if (smem > optin) {
            set_error("attn_kv4: needs %d B of shared memory per block, device allows %d", smem, optin);
            return KVP_ERR_UNSUPPORTED;
        }
        // setmaxnreg.inc waits until the warpgroup's registers exist in the
        // CTA's pool: refuse a build whose launch pool is smaller than the split.
        cudaFuncAttributes fa;
        KVP_CUDA(cudaFuncGetAttributes(&fa, attn_kv4_sm100_kernel));
        if ((long long)fa.numRegs * kThreads < (long long)kRegsLow * 128 + 2LL * kRegsHigh * 128) {
            set_error("attn_kv4: kernel built with %d registers per thread, the register split needs %d",
                      fa.numRegs, (kRegsLow * 128 + 2 * kRegsHigh * 128 + kThreads - 1) / kThreads);
            return KVP_ERR_UNSUPPORTED;
        }
        KVP_CUDA(cudaFuncSetAttribute(attn_kv4_sm100_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
        return KVP_OK;
    });
    if (rc != KVP_OK) return rc;
    cudaLaunchAttribute early;
    const cudaLaunchConfig_t cfg = kv4_config(grid, kThreads, (size_t)smem, &early, stream);
    KVP_CUDA(cudaLaunchKernelEx(&cfg, attn_kv4_sm100_kernel, P));
    return KVP_OK;
}

}  // namespace kvp
