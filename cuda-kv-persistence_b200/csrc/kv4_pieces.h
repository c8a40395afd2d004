// Which CTAs hold the pieces of a cut unit (Kv4Unit in attn_kv4.cuh).  Plain
// C++, for the join kernel and the CPU test.
#pragma once

#ifdef __CUDACC__
#define KVP_HOST_DEVICE __host__ __device__ __forceinline__
#else
#define KVP_HOST_DEVICE inline
#endif

namespace kvp {

struct Kv4Pieces {
    int first, count;   // CTAs [first, first + count); count 0: nothing to join
};

// A unit of `pages` pages whose first one is at `page` in a list that `ctas`
// CTAs take `chunk` at a time.  Both come from the workspace, where the kernel
// before wrote them; if it gave up (a wait that ran out) they may be anything,
// and no CTA outside [0, ctas) may follow from them.
KVP_HOST_DEVICE Kv4Pieces kv4_pieces(int chunk, int page, int pages, int ctas) {
    if (chunk <= 0 || page < 0 || pages <= 0) return Kv4Pieces{0, 0};
    const int first = page / chunk;
    const long long last = ((long long)page + pages - 1) / chunk;
    if (last >= ctas) return Kv4Pieces{0, 0};
    return Kv4Pieces{first, (int)last - first + 1};
}

}  // namespace kvp
