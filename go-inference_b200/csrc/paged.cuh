// paged.cuh — what the paged-cache kernels share: the cache's addressing, the visibility of keys, and the
// argument checks of their entry points.
#pragma once
#include "common.cuh"

#include <initializer_list>

namespace lthn {

// lthn_paged_kv with its default strides filled in.
struct PagedCache {
    uint16_t* k;
    uint16_t* v;
    const int32_t* table;
    int64_t page_stride, row_stride, head_stride;
    int pages, page_size, table_stride, seqs, kv_heads;
    int capacity;        // rows the table can name for a sequence, at most 2^26
    // position / page_size for positions below 2^27: (position * div_mul) >> div_shift, with div_shift = 27 + ceil(log2 page_size) and
    // div_mul = ceil(2^div_shift / page_size); the product's error, position * (div_mul * page_size - 2^div_shift), stays below 2^div_shift
    uint32_t div_mul, div_shift;
    uint32_t* status;
};

// Score options with the defaults filled in. Scores are kept in units of log2, so that a weight is one ex2.
struct AttnOpts {
    float scale;         // softmax scale
    float softcap;       // 0: none; at most 2^126, also in units of the raw product
    const float* slopes;
    int window;          // 0: none
    const int32_t* prefix;
};

// Host: checks of the arguments every call has, and the fill-in. `name` is the entry point, for messages.
int32_t paged_check_cache(const char* name, const lthn_paged_kv* c, PagedCache* out);
int32_t paged_check_options(const char* name, const lthn_attn_options* o, int head_dim, AttnOpts* out);
// An argument that the kernels read or write through. NULL ones are skipped: the optional arguments.
struct PagedPtr {
    const char* what;
    const void* p;
    int align;           // bytes
    bool pinned;         // page-locked host memory serves too (not where TMA or wide copies go through it)
};
// Every pointer is aligned and memory that the current device can reach: a host pointer or another GPU's would fault in the kernel.
int32_t paged_check_pointers(const char* name, std::initializer_list<PagedPtr> list);
int paged_sm_count();

#ifdef __CUDACC__
// what a raw product is multiplied with to be in units of the cap; finite, so that a product of zero stays zero under the smallest caps
__device__ __forceinline__ float paged_cap_in(const AttnOpts& o) { return fminf(o.scale / o.softcap, 3.402823466e38f); }
__device__ __forceinline__ int paged_entry(const PagedCache& c, int pos) { return (int)(((uint64_t)(uint32_t)pos * c.div_mul) >> c.div_shift); }
__device__ __forceinline__ int paged_row(const PagedCache& c, int pos) { return pos - paged_entry(c, pos) * c.page_size; }

// Element offset of kv head 0 of a row of a page, or -1 (and the status bit) for a page outside the pool.
__device__ __forceinline__ int64_t paged_offset(const PagedCache& c, int page, int in_page) {
    if ((unsigned)page >= (unsigned)c.pages) {
        atomicOr(c.status, LTHN_STATUS_PAGED);
        return -1;
    }
    return page * c.page_stride + in_page * c.row_stride;
}

// a sequence's length, cut at what the table can name
__device__ __forceinline__ int paged_length(const PagedCache& c, int len) {
    if (len > c.capacity) {
        atomicOr(c.status, LTHN_STATUS_PAGED);
        return c.capacity;
    }
    return max(len, 0);
}

// The key tiles (of TILE keys) that queries at positions [q0, q1] of a sequence may look at: tiles [0, na) hold the
// prefix, tiles [b, b + n - na) the rest; piece i of n is tile i (i < na) or b + i - na.
struct KeyTiles {
    int na, b, n;
    __device__ __forceinline__ int tile(int i) const { return i < na ? i : b + i - na; }
};
template <int TILE>
__device__ __forceinline__ KeyTiles key_tiles(int q0, int q1, int len, int prefix, int window) {
    KeyTiles t;
    const int p = min(max(prefix, 0), len);
    t.na = (p + TILE - 1) / TILE;
    const int lo = window > 0 ? max(0, q0 - window + 1) : 0;   // first key the oldest query's window holds
    const int hi = min(q1 + 1, len);                           // behind the last key the newest query sees
    t.b = max(t.na, lo / TILE);
    t.n = t.na + max(0, (hi + TILE - 1) / TILE - t.b);
    return t;
}

// Inclusive scan over the block of one count per thread; returns the total. sh: one word per warp.
template <int WARPS>
__device__ __forceinline__ int paged_block_scan(int v, int& incl, int* sh) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    incl = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += u;
    }
    __syncthreads();
    if (lane == 31) sh[warp] = incl;
    __syncthreads();
    int total = 0;
#pragma unroll
    for (int w = 0; w < WARPS; w++) {
        if (w < warp) incl += sh[w];
        total += sh[w];
    }
    return total;
}

__device__ __forceinline__ uint32_t pack_bf16x2(float lo, float hi) {
    uint32_t d;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
    return d;
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// 16 bytes global -> shared; bytes = 0 writes zeros and reads nothing
__device__ __forceinline__ void cp_async16_zfill(uint32_t dst, const void* src, int bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void paged_cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void paged_cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void ldmatrix_x4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
// Bounded wait on an mbarrier phase: try_wait parks the thread for a while each time; after 0.2 s of wall time it gives up.
__device__ __forceinline__ bool paged_wait(uint64_t* bar, uint32_t parity) {
    uint32_t done = 0;
    uint64_t t0 = 0;
    for (uint32_t it = 0;; ++it) {
        asm volatile("{\n\t.reg .pred p;\n\t"
                     "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
                     "selp.u32 %0, 1, 0, p;\n\t}"
                     : "=r"(done) : "r"(smem_u32(bar)), "r"(parity) : "memory");
        if (done) return true;
        if ((it & 63) == 63) {
            uint64_t now;
            asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(now));
            if (t0 == 0) t0 = now;
            else if (now - t0 > 200000000ull) return false;
        }
    }
}

// Asks for the launch of a waiting CTA to be cancelled; the answer (16 bytes) comes by mbarrier. After a refusal no CTA asks again.
__device__ __forceinline__ void paged_try_cancel(void* answer, uint64_t* bar) {
    asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];"
                 ::"r"(smem_u32(answer)), "r"(smem_u32(bar)) : "memory");
}
// the block index that now is this CTA's to do, -1: none
__device__ __forceinline__ int paged_cancelled(const void* answer) {
    int x;
    asm volatile("{\n\t.reg .b128 h;\n\t.reg .pred p;\n\tld.shared.b128 h, [%1];\n\tmov.b32 %0, -1;\n\t"
                 "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, h;\n\t"
                 "@p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %0, h;\n\t}" : "=r"(x) : "r"(smem_u32(answer)) : "memory");
    return x;
}
#endif

}  // namespace lthn
