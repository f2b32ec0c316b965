// paged_prefill.cu — attention of packed prompt chunks over the paged KV cache on the Blackwell tensor cores.
//
//   out = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m),   s_j = cap(q.k_j scale) - slope |i - j|,   m = max_j s_j
//
// 4*D flops per visible (query, key) pair against 4*D bytes of K and V per key and tile of query rows: bound by the tensor pipe
// for prompts, by HBM for a few rows against a long context.
//
// Rows. The query rows of a tile are the (token, query head) pairs of one kv head, token by token, as many whole tokens as 128
// rows hold, so the heads that share K and V share their loads, a chunk of a few tokens still fills a tile, and the
// queries of a tile are one TMA box per 64 head dimensions. A CTA works on one or two tiles of 128 rows (two: two accumulators of head_dim columns fit the tensor memory beside two score tiles for head_dim 64 and 128) and on
// BN keys at a time.
//
//   softmax warps   two warpgroups, one per score buffer, one thread per row: tcgen05.ld the row's BN scores, mask, maximum, ex2,
//                   sum - all within the thread - and tcgen05.st the weights as bf16 over the scores they came from.
//   issuer          one warp: S = Q K^T (both operands in shared memory), O += P V (P in tensor memory, V in shared
//                   memory as an N-major operand, so it is stored as it comes). There are two score buffers. Unit u uses
//                   buffer u & 1 and the issue order is S(0) S(1) | O(0) S(2) | O(1) S(3) | ..., so that the tensor pipe
//                   works on one buffer while the other's softmax runs. With two row tiles the buffers belong to them;
//                   with one they alternate over its key tiles, and the warpgroups pass the running maximum of a row to one
//                   another (the sums stay apart until the end), which leaves only load and maximum in sequence.
//   loaders         three warps fetch the queries of a segment and fill a ring of K and V tiles in the 128-byte swizzle. Where the page size is a multiple of 8 (the
//                   swizzle's row group) by tiled TMA, one box per page, 64 head dimensions and gcd(page size, BN) rows. V rows
//                   that nobody sees must be zeros (they may hold NaN, which a weight of zero would not silence), so a V
//                   tile with such rows - the last of a sequence, the first of a window - and pools of other page
//                   sizes come row by row with cp.async of 16 bytes, zero-filled; unseen K rows may hold anything, their
//                   scores are replaced. 8192 tokens of 32 heads: 1007 us with cp.async throughout, 541 us with TMA.
//
// The running maximum is only moved when a row's grew by more than 2^8: until then weights are up to 2^8, which neither
// their bf16 rounding (relative) nor the f32 sums mind, and O in tensor memory needs no correction. A move multiplies
// O by 2^(old - new) through registers; after the first tiles it is rare.
//
// Work. The key tiles of all (row tile, kv head) pairs form one list, weighted by what they cost; CTA c of C (one per SM) takes the
// c-th C-th of it, whatever the lengths are, and walks through its segments without stopping: the loaders are at the next
// segment's queries and keys while the softmax warps finish the last one. A pair that lies within one CTA is finished there; otherwise each
// CTA that holds part of it leaves (maximum, sum, unnormalised output) in its slot of the workspace - at most two such
// parts, its first and its last segment - and a second kernel joins them. (One CTA per tile, longest first, spent 7 us of
// each CTA on its start and end; cut into equal chunks, the few rows of drafts against long contexts of different lengths took
// two waves where the work was one.)
//
// Every wait is bounded: on a time-out the roles record it in the device status word, drain what they have in flight, free
// the tensor memory and return.
#include "paged.cuh"

#include <cuda.h>

#include <algorithm>
#include <mutex>
#include <numeric>

namespace lthn {

struct PrefillArgs {
    PagedCache c;
    int box;             // rows of a TMA box, 0: rows are copied one by one
    int rows_first;      // the tensor maps' dimensions are (dim, row, head, page), else (dim, head, row, page)
    AttnOpts o;
    const uint16_t* q;
    uint16_t* out;
    int64_t q_stride, out_stride;
    const int32_t *q_start, *lens;
    float* lse;
    uint32_t* wait_status;
    int seqs, total_q, Hq, G;
    int tokens;          // of a row tile: 128 / G
    int q_box;           // queries by TMA (their row stride is a multiple of head_dim), else copied row by row
    float4* part;        // [2*CTAs][D/4][rows] unnormalised outputs, four columns each
    float2* ml;          // [2*CTAs][rows] maximum (log2 units) and sum
    int4* desc;          // [CTAs] the pair that begins in the CTA and ends in another: sequence, tile, head, last CTA (-1: none)
};

// The rows of sequence s, made safe: within [0, total_q).
__device__ __forceinline__ int2 prefill_span(const PrefillArgs& a, int s) {
    const int b = a.q_start[s], e = a.q_start[s + 1];
    if (b < 0 || e < b || e > a.total_q) {
        atomicOr(a.c.status, LTHN_STATUS_PAGED);
        return make_int2(0, 0);
    }
    return make_int2(b, e - b);
}

// The tokens of one or two row tiles of a sequence.
struct PfTile {
    int2 span;           // the sequence's rows of q: first, count
    int len, pos0;       // keys; position of the first query
    int prefix;
    int tok0;            // first token of the tile
    int qlo, qhi;        // positions of its first and last token
    KeyTiles kt;
    bool two;            // both row tiles have tokens
};
template <int NQ, int BN>
__device__ __forceinline__ PfTile prefill_tile(const PrefillArgs& a, int seq, int tile) {
    PfTile t;
    t.span = prefill_span(a, seq);
    t.len = paged_length(a.c, a.lens[seq]);
    t.pos0 = t.len - t.span.y;
    t.prefix = a.o.prefix ? min(max(a.o.prefix[seq], 0), t.len) : 0;
    t.tok0 = tile * NQ * a.tokens;
    t.qlo = t.pos0 + t.tok0;
    t.qhi = t.pos0 + min(t.tok0 + NQ * a.tokens, t.span.y) - 1;
    t.kt = key_tiles<BN>(t.qlo, t.qhi, t.len, t.prefix, a.o.window);
    t.two = NQ == 2 && t.span.y - t.tok0 > a.tokens;
    return t;
}
// What a (tile, head) pair costs: about 0.6 us per unit. A key tile of two row tiles keeps the tensor pipe busier than one of one; the start covers
// the first scores, the last output and its way to memory.
constexpr int PF_ONE = 2, PF_TWO = 3, PF_START = 6;
constexpr int PF_LEAST = 8;   // units of a CTA below which fewer CTAs are used: every part holds a key tile
static_assert(PF_LEAST >= 2 * PF_TWO, "a range within a pair holds a whole key tile");
__device__ __forceinline__ int pf_key_cost(const PfTile& t) { return t.two ? PF_TWO : PF_ONE; }
__device__ __forceinline__ int pf_cost(const PfTile& t) { return PF_START + t.kt.n * pf_key_cost(t); }
// the key tiles that lie before unit v of a pair
__device__ __forceinline__ int pf_tiles_before(const PfTile& t, int v) { return v <= PF_START ? 0 : (v - PF_START) / pf_key_cost(t); }

// The walk of a CTA through its segments; every role makes its own.
template <int NQ, int BN>
struct PfWalk {
    PfTile t;
    int seq, tile, head, v, cost;
    int64_t u, u1;
    int i0, n, take;     // segment: key tiles [i0, i0 + n) of the pair
    __device__ __forceinline__ void start(const PrefillArgs& a, int seq_, int tile_, int64_t base, int64_t u0, int64_t end) {
        seq = seq_; tile = tile_; u = u0; u1 = end;
        t = prefill_tile<NQ, BN>(a, seq, tile);
        cost = pf_cost(t);
        head = (int)((u0 - base) / cost);
        v = (int)((u0 - base) - (int64_t)head * cost);
    }
    __device__ __forceinline__ bool more() const { return u < u1; }
    // false: nothing to do in this one
    __device__ __forceinline__ bool segment() {
        take = (int)min((int64_t)(cost - v), u1 - u);
        i0 = pf_tiles_before(t, v);
        n = pf_tiles_before(t, v + take) - i0;
        return n > 0 || (t.kt.n == 0 && v == 0);
    }
    __device__ __forceinline__ bool whole() const { return n == t.kt.n; }
    __device__ __forceinline__ void next(const PrefillArgs& a) {
        u += take;
        v += take;
        if (v < cost || u >= u1) return;
        v = 0;
        if (++head < a.c.kv_heads) return;
        head = 0;
        tile++;
        if (tile * NQ * (int64_t)a.tokens >= t.span.y) {
            tile = 0;
            do seq++; while (seq < a.seqs && prefill_span(a, seq).y == 0);
            if (seq >= a.seqs) { u = u1; return; }       // only if the lengths changed under the call
        }
        t = prefill_tile<NQ, BN>(a, seq, tile);
        cost = pf_cost(t);
    }
};

// ---- tcgen05 wrappers (cta_group::1) ---------------------------------------------------------------
__device__ __forceinline__ void pf_tmem_alloc(uint32_t* smem_dst, uint32_t ncols) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(smem_dst)), "r"(ncols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void pf_tmem_dealloc(uint32_t taddr, uint32_t ncols) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols) : "memory");
}
__device__ __forceinline__ void pf_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void pf_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void pf_fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
// Issued by one lane, but from code that the whole warp runs: the operands are then known to be the same for all lanes and live in
// uniform registers, where the instruction wants them (from a one-lane branch each issue costs several register moves).
__device__ __forceinline__ void pf_mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p, e;\n\telect.sync _|e, 0xffffffff;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void pf_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p, e;\n\telect.sync _|e, 0xffffffff;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
                 ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void pf_commit(uint64_t* bar) {
    asm volatile("{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\t"
                 "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void pf_tma_3d(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, uint64_t* bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
                 ::"r"(dst), "l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void pf_tma_4d(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, int c3, uint64_t* bar) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
                 ::"r"(dst), "l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void pf_arrive(uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void pf_ld32(uint32_t taddr, float* f) {
    uint32_t* r = (uint32_t*)f;
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr) : "memory");
}
__device__ __forceinline__ void pf_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void pf_st32(uint32_t taddr, const float* f) {
    const uint32_t* r = (const uint32_t*)f;
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
        "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
        "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};"
        ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
          "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]),
          "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]),
          "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]) : "memory");
}
__device__ __forceinline__ void pf_st16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
        ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
          "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]) : "memory");
}
__device__ __forceinline__ void pf_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Bounded wait on an mbarrier phase: try_wait parks the thread for a while each time; after 0.2 s of wall time it gives up.
__device__ __forceinline__ bool pf_wait(uint64_t* bar, uint32_t parity) {
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

// Shared-memory operands in the 128-byte swizzle: slabs of 64 elements, rows 128 bytes apart, 8-row groups 1024.
// K-major (Q and K): a K = 16 step is 32 bytes further in the slab.
__device__ __forceinline__ uint64_t pf_desc_k(uint32_t addr) {
    return (uint64_t)((addr & 0x3FFFFu) >> 4) | ((uint64_t)1 << 16) | ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
// N-major (V: rows are keys = the MMA's K, 64 head dimensions each): 8-key groups 1024 bytes apart (stride offset), the next 64
// head dimensions one slab further (leading offset); a K = 16 step is 16 rows = 2048 bytes.
__device__ __forceinline__ uint64_t pf_desc_n(uint32_t addr, uint32_t slab) {
    return (uint64_t)((addr & 0x3FFFFu) >> 4) | ((uint64_t)(slab >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) |
           ((uint64_t)2 << 61);
}

__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
// the n lowest bits of a word, n of any size and sign
__device__ __forceinline__ uint32_t low_bits(int n) { return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u; }
// two f32 operations in one instruction
__device__ __forceinline__ uint64_t pack2(float lo, float hi) {
    uint64_t d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(lo), "f"(hi));
    return d;
}
__device__ __forceinline__ void unpack2(uint64_t v, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ float rcp_approx(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

template <int D>
struct PfCfg {
    static constexpr int NQ = D == 256 ? 1 : 2;              // row tiles per CTA
    static constexpr int BN = D == 256 ? 64 : 128;           // keys per tile
    static constexpr int ROWS = NQ * 128;
    static constexpr int SM_WARPS = 8;                       // softmax warps
    static constexpr int WARPS = SM_WARPS + 4;               // + issuer + three loaders
    static constexpr int THREADS = WARPS * 32;
    static constexpr int Q_BYTES = 128 * D * 2;              // one row tile
    static constexpr int KV_BYTES = BN * D * 2;
    static constexpr int SLAB = BN * 128;                    // bytes of 64 head dimensions of a K or V tile
    static constexpr int ST = D == 64 ? 8 : 5;
    static constexpr int RING = NQ * Q_BYTES;                // offsets in shared memory
    static constexpr int OFFS = RING + ST * KV_BYTES;        // [2][BN] row offsets
    static constexpr int BARS = OFFS + 2 * BN * 8;
    static constexpr int ROW_MAX = BARS + 512;               // one row tile: the rows' running maximum
    static constexpr int TOTAL = ROW_MAX + 512;
    static constexpr int S_COLS = BN;                        // tensor memory: two score buffers, then the outputs at column 256
    static constexpr int LAG = 2;                            // ring slots in flight behind the one being filled
    static_assert(LAG <= ST - 3, "a slot is handed over before the one that frees its successor is waited for");
    static_assert(TOTAL <= 232448, "shared memory of a CTA");
};

// FEAT bit 0: tanh cap, bit 1: distance bias
template <int D, int FEAT>
__global__ void __launch_bounds__(PfCfg<D>::THREADS, 1) paged_prefill_kernel(const __grid_constant__ CUtensorMap q_map, const __grid_constant__ CUtensorMap k_map,
                                                                       const __grid_constant__ CUtensorMap v_map, const PrefillArgs a) {
    using C = PfCfg<D>;
    constexpr int BN = C::BN, ST = C::ST, ROWS = C::ROWS;
    constexpr float LOG2E = 1.4426950408889634f;
    extern __shared__ __align__(1024) unsigned char pf_smem[];
    uint64_t* full = (uint64_t*)(pf_smem + C::BARS);         // [ST] loaders -> issuer
    uint64_t* empty = full + ST;                             // [ST] issuer's commit -> loaders
    uint64_t* s_full = empty + ST;                           // [2] scores are there
    uint64_t* p_full = s_full + 2;                           // [2] weights are there, O is corrected
    uint64_t* o_done = p_full + 2;                           // [2] per row tile: O(u) has been added, all but the last
    uint64_t* o_last = o_done + 2;                           // [2] the last has (a barrier of its own: with one row tile the softmax
                                                             //     may be two units ahead, which a parity cannot tell from none)
    uint64_t* turn = o_last + 2;                             // [4] one row tile: the maximum of key tile j is out, per 32 rows
    uint64_t* q_full = turn + 4;                             // queries of a segment
    uint64_t* q_empty = q_full + 1;                          // its last scores are done
    uint64_t* meet = q_empty + 1;                            // both softmax warpgroups (a barrier whose wait is bounded)
    uint64_t* drain = meet + 1;
    uint32_t* tmem_slot = (uint32_t*)(drain + 1);
    int* scan = (int*)(tmem_slot + 2);                       // WARPS words, then sequence, tile and (64 bits) first unit of the first tile
    static_assert((2 * ST + 20) * 8 + (C::WARPS + 4) * 4 <= 512, "barriers and scan words");

    pdl_trigger();
    const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);

    // ---- this CTA's part of the work ------------------------------------------------------------------
    int* first = (int*)(pf_smem + C::RING);                  // first tile of each sequence
    int T = 0;
    for (int s0 = 0; s0 < a.seqs; s0 += C::THREADS) {
        const int s = s0 + tid;
        const int c = s < a.seqs ? (prefill_span(a, s).y + C::NQ * a.tokens - 1) / (C::NQ * a.tokens) : 0;
        int incl;
        const int total = paged_block_scan<C::WARPS>(c, incl, scan);
        if (s < a.seqs) first[s] = T + incl - c;
        T += total;
    }
    __syncthreads();
    auto find = [&](int t) {                                 // the last sequence that begins at or before tile t (empty ones begin with the next)
        int lo = 0, hi = a.seqs - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (first[mid] <= t) lo = mid;
            else hi = mid - 1;
        }
        return lo;
    };
    auto cost_of = [&](int t) {
        if (t >= T) return 0;
        const int s = find(t);
        return pf_cost(prefill_tile<C::NQ, BN>(a, s, t - first[s]));
    };
    int incl, mine = cost_of(tid);
    int part = paged_block_scan<C::WARPS>(mine, incl, scan);
    int64_t U = part;
    for (int t0 = C::THREADS; t0 < T; t0 += C::THREADS) {
        int x;
        U += paged_block_scan<C::WARPS>(cost_of(t0 + tid), x, scan);
    }
    U *= a.c.kv_heads;
    const int ctas = (int)max((int64_t)1, min((int64_t)gridDim.x, U / PF_LEAST));
    if (T == 0 || (int)blockIdx.x >= ctas) {
        if (tid == 0) a.desc[blockIdx.x] = make_int4(0, 0, 0, -1);
        return;
    }
    const int64_t u0 = U * blockIdx.x / ctas, u1 = U * (blockIdx.x + 1) / ctas;
    int64_t* first_unit = (int64_t*)(scan + C::WARPS + 2);
    int64_t base = 0;
    for (int t0 = 0;;) {
        if ((base + part) * a.c.kv_heads > u0) {
            const int64_t b = (base + incl - mine) * a.c.kv_heads;
            if (mine > 0 && b <= u0 && b + (int64_t)mine * a.c.kv_heads > u0) {
                const int s = find(t0 + tid);
                scan[C::WARPS] = s;
                scan[C::WARPS + 1] = t0 + tid - first[s];
                *first_unit = b;
            }
            break;
        }
        base += part;
        t0 += C::THREADS;
        mine = cost_of(t0 + tid);
        part = paged_block_scan<C::WARPS>(mine, incl, scan);
    }

    if (tid == 0) {
        for (int s = 0; s < ST; s++) { mbar_init(&full[s], 96); mbar_init(&empty[s], 1); }
        for (int b = 0; b < 2; b++) { mbar_init(&s_full[b], 1); mbar_init(&p_full[b], 128); mbar_init(&o_done[b], 1); mbar_init(&o_last[b], 1); }
        for (int w = 0; w < 4; w++) mbar_init(&turn[w], 1);
        mbar_init(q_full, 96);
        mbar_init(q_empty, 1);
        mbar_init(meet, C::SM_WARPS * 32);
        mbar_init(drain, 1);
        mbar_fence_init();
    }
    if (warp == C::SM_WARPS) pf_tmem_alloc(tmem_slot, 512);
    pf_fence_before();
    __syncthreads();
    pf_fence_after();
    const uint32_t tmem = *tmem_slot;
    const uint32_t smem = smem_u32(pf_smem);
    PfWalk<C::NQ, BN> wk;
    wk.start(a, scan[C::WARPS], scan[C::WARPS + 1], *first_unit, u0, u1);
    const PfTile& t = wk.t;
    bool ok = true;

    // ring slots of the K and V tile of key tile j of a segment, in the order of their last use
    auto k_slot = [&](int j) { return t.two ? 2 * j : j < 2 ? j : 2 * j - 1; };
    auto v_slot = [&](int j) { return t.two ? 2 * j + 1 : j == wk.n - 1 ? 2 * wk.n - 1 : 2 * j + 2; };

    if (warp < C::SM_WARPS) {
        // ================================ softmax ================================
        asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
        const int wg = warp >> 2;                            // score buffer = warpgroup
        const int wr = (warp & 3) * 32, r = wr + lane;       // row within the row tile = tensor memory lane
        const int r_token = r / a.G, r_head = r - r_token * a.G;
        const uint32_t lanes = tmem + ((uint32_t)wr << 16);
        const uint32_t s_addr = lanes + wg * C::S_COLS;
        // plain scores stay as the product left them, the others are brought to log2 units first
        const float c1 = FEAT ? 1.0f : a.o.scale * LOG2E;
        const float cap2 = a.o.softcap * LOG2E, cin = FEAT & 1 ? 2.0f * LOG2E * a.o.scale / a.o.softcap : a.o.scale * LOG2E;
        float* row_max = (float*)(pf_smem + C::ROW_MAX);     // one row tile only
        int uses = 0;                                        // of this warpgroup's score buffer
        int turns = 0, done0 = 0, done1 = 0, last0 = 0, last1 = 0, meets = 0;  // phases the barriers have gone through
        auto pair_sync = [&] {
            pf_arrive(meet);
            const bool met = __all_sync(0xffffffffu, pf_wait(meet, meets++ & 1));
            ok = ok && met;
        };
        for (; wk.more() && ok; wk.next(a)) {
        if (!wk.segment()) continue;
        const bool two = t.two;
        const int n = wk.n, i0 = wk.i0, qt = two ? wg : 0, len = t.len;
        const int token = t.tok0 + qt * a.tokens + r_token;  // of the sequence
        const bool live = r_token < a.tokens && token < t.span.y;
        const int head = wk.head * a.G + r_head;
        const int qpos = t.pos0 + token;
        // visible: key < pre, or klo <= key < khi
        const int pre = t.prefix, khi = min(qpos + 1, len), klo = a.o.window > 0 ? qpos - a.o.window + 1 : 0;
        const float slope = (FEAT & 2) && live ? a.o.slopes[head] * LOG2E : 0.f;
        const uint32_t o_addr = lanes + 256 + qt * D;
        float m = -INFINITY, l = 0.f;                        // reference maximum (units of the scores), sum relative to it

        for (int j = two ? 0 : wg; j < n; j += two ? 1 : 2) {
            ok = __all_sync(0xffffffffu, pf_wait(&s_full[wg], uses & 1));
            if (!ok) break;
            uses++;
            pf_fence_after();
            float s[BN];
#pragma unroll
            for (int x = 0; x < BN; x += 32) pf_ld32(s_addr + x, s + x);
            pf_ld_wait();
            const int k0 = t.kt.tile(i0 + j) * BN;
            if (FEAT & 1) {
                // cap tanh(x scale / cap) = cap (1 - 2 / (1 + e^(2 x scale / cap)))
#pragma unroll
                for (int x = 0; x < BN; x++) s[x] = fmaf(-2.0f * cap2, rcp_approx(1.0f + ex2(s[x] * cin)), cap2);
            }
            if (FEAT & 2) {
                const float gap = (float)(qpos - k0);
#pragma unroll
                for (int x = 0; x < BN; x++) s[x] = fmaf(-slope, fabsf(gap - (float)x), FEAT & 1 ? s[x] : s[x] * cin);
            }
            const bool all = !live || k0 + BN <= pre || (k0 >= klo && k0 + BN <= khi);
            if (!__all_sync(0xffffffffu, all)) {
                const int p = pre - k0, lo = klo - k0, hi = khi - k0;
#pragma unroll
                for (int x0 = 0; x0 < BN; x0 += 32) {
                    const uint32_t seen = low_bits(p - x0) | (low_bits(hi - x0) & ~low_bits(lo - x0));
#pragma unroll
                    for (int x = 0; x < 32; x++) s[x0 + x] = seen >> x & 1 ? s[x0 + x] : -INFINITY;
                }
            }
            float mx[4];                                     // four chains
#pragma unroll
            for (int x = 0; x < 4; x++) mx[x] = max3(s[x], s[x + 4], s[x + 8]);
#pragma unroll
            for (int x = 12; x + 8 <= BN; x += 8)
#pragma unroll
                for (int e = 0; e < 4; e++) mx[e] = max3(mx[e], s[x + e], s[x + 4 + e]);
            static_assert((BN - 12) % 8 == 4, "the last four scores");
            mx[0] = max3(mx[0], s[BN - 4], s[BN - 3]);
            mx[1] = max3(mx[1], s[BN - 2], s[BN - 1]);
            if (!two && j > 0) {                             // the row's maximum so far, from the other warpgroup
                ok = __all_sync(0xffffffffu, pf_wait(&turn[warp & 3], (turns + j - 1) & 1));
                if (!ok) break;
                const float mo = row_max[r];
                if (mo != m) {                               // it has moved: this warpgroup's sum follows
                    l = m == -INFINITY ? 0.f : l * ex2((m - mo) * c1);
                    m = mo;
                }
                __syncwarp();
            }
            const float mnew = live ? max3(fmaxf(m, mx[0]), mx[1], fmaxf(mx[2], mx[3])) : m;   // a row without a query holds anything
            const bool move = __any_sync(0xffffffffu, (mnew - m) * c1 > 8.0f);
            const float mold = m;
            if (move) {
                l = m == -INFINITY ? 0.f : l * ex2((m - mnew) * c1);
                m = mnew;
            }
            if (!two) {
                row_max[r] = m;
                __syncwarp();
                if (lane == 0) pf_arrive(&turn[warp & 3]);
                __syncwarp();
            }
            if (move && j > 0) {
                const float alpha = mold == -INFINITY ? 0.f : ex2((mold - mnew) * c1);
                ok = __all_sync(0xffffffffu, pf_wait(&o_done[qt], ((qt ? done1 : done0) + j - 1) & 1));
                if (!ok) break;
                pf_fence_after();
#pragma unroll
                for (int x = 0; x < D; x += 32) {
                    float o[32];
                    pf_ld32(o_addr + x, o);
                    pf_ld_wait();
#pragma unroll
                    for (int e = 0; e < 32; e++) o[e] *= alpha;
                    pf_st32(o_addr + x, o);
                }
            }
            const float neg = m == -INFINITY ? 0.f : -m * c1;
            const uint64_t c2 = pack2(c1, c1), n2 = pack2(neg, neg);
            uint64_t sum[2] = {0, 0};
#pragma unroll
            for (int x = 0; x < BN; x += 32) {
                uint32_t w[16];
#pragma unroll
                for (int e = 0; e < 32; e += 2) {
                    float p0, p1;
                    unpack2(fma2(pack2(s[x + e], s[x + e + 1]), c2, n2), p0, p1);
                    p0 = ex2(p0);
                    p1 = ex2(p1);
                    sum[e / 2 & 1] = add2(sum[e / 2 & 1], pack2(p0, p1));
                    w[e / 2] = pack_bf16x2(p0, p1);
                }
                pf_st16(s_addr + x / 2, w);
            }
            pf_st_wait();
            pf_fence_before();
            pf_arrive(&p_full[wg]);
            float l0, l1;
            unpack2(add2(sum[0], sum[1]), l0, l1);
            l += l0 + l1;
        }
        if (ok && n > 0) ok = __all_sync(0xffffffffu, pf_wait(&o_last[qt], (qt ? last1 : last0) & 1));
        int x0 = 0, x1 = D;                                  // output columns of this warpgroup
        if (!two && n > 0) {
            // the two sums of a row meet, relative to the last maximum; each warpgroup stores half of the columns
            if (ok) ok = __all_sync(0xffffffffu, pf_wait(&turn[warp & 3], (turns + n - 1) & 1));
            const float mo = row_max[r];
            l = m == -INFINITY ? 0.f : l * ex2((m - mo) * c1);
            m = mo;
            pair_sync();
            if (wg == 1) row_max[r] = l;
            pair_sync();
            if (wg == 0) { l += row_max[r]; row_max[r] = l; }
            pair_sync();
            l = row_max[r];
            x0 = wg * (D / 2);
            x1 = x0 + D / 2;
            turns += n;
        }
        if (n > 0) {
            if (two) { done1 += n - 1; last1++; }
            done0 += n - 1;
            last0++;
        }
        if (ok) {
            pf_fence_after();
            const int64_t tok = t.span.x + token;
            const float m2 = m * c1;                         // log2 units (c1 > 0)
            const float inv = l > 0.f ? 1.0f / l : 0.f;
            uint16_t* dst = a.out + tok * a.out_stride + (int64_t)head * D;
            const bool whole = wk.whole();
            const int slot = 2 * blockIdx.x + (i0 > 0 ? 0 : 1);
            float4* part = a.part + (int64_t)slot * (D / 4) * ROWS + qt * 128 + r;
#pragma unroll 1
            for (int x = x0; x < x1; x += 32) {
                float o[32];
                __syncwarp();                                // the stores below are not made by all lanes, the loads have to be
                if (n > 0) {
                    pf_ld32(o_addr + x, o);
                    pf_ld_wait();
                } else {
#pragma unroll
                    for (int e = 0; e < 32; e++) o[e] = 0.f;
                }
                if (!live) continue;
                if (whole) {
#pragma unroll
                    for (int e = 0; e < 32; e += 8)
                        *(uint4*)(dst + x + e) = make_uint4(pack_bf16x2(o[e] * inv, o[e + 1] * inv), pack_bf16x2(o[e + 2] * inv, o[e + 3] * inv),
                                                            pack_bf16x2(o[e + 4] * inv, o[e + 5] * inv), pack_bf16x2(o[e + 6] * inv, o[e + 7] * inv));
                } else {
#pragma unroll
                    for (int e = 0; e < 32; e += 4) part[(x + e) / 4 * ROWS] = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
                }
            }
            if (live && x0 == 0) {
                if (!whole) a.ml[slot * ROWS + qt * 128 + r] = make_float2(m2, l);
                else if (a.lse) a.lse[tok * a.Hq + head] = (m2 + log2f(l)) * 0.6931471805599453f;
            }
        }
        if (!two && n > 0) pair_sync();                      // both have read O before the next segment's first weights let it be replaced
        }
        if (!ok && lane == 0) atomicOr(a.wait_status, 1u << 26);
    } else if (warp == C::SM_WARPS) {
        // ================================ issuer ================================
        asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
        // f32 accumulators, bf16 operands, M = 128; S: N = BN, both K-major; O: N = D, B is N-major
        const uint32_t idesc = (1u << 4) | (1u << 7) | (1u << 10) | ((128u >> 4) << 24);
        const uint32_t idesc_s = idesc | ((uint32_t)(BN >> 3) << 17), idesc_o = idesc | (1u << 16) | ((uint32_t)(D >> 3) << 17);
        int slot0 = 0, segments = 0;                         // ring slots and segments so far
        uint32_t uses = 0;                                   // bit b: parity of the uses of score buffer b
        int4 begun = make_int4(0, 0, 0, -1);
        for (; wk.more() && ok; wk.next(a)) {
            if (!wk.segment()) continue;
            const bool two = t.two;
            const int n = wk.n, units = two ? 2 * n : n;
            if (wk.i0 == 0 && !wk.whole())
                begun = make_int4(wk.seq, wk.tile, wk.head, (int)(((wk.u - wk.v + wk.cost) * ctas + U - 1) / U) - 1);
            if (n == 0) continue;
            ok = __all_sync(0xffffffffu, pf_wait(q_full, segments & 1));
            auto scores = [&](int u) {
                const int j = two ? u >> 1 : u, qt = two ? u & 1 : 0, slot = slot0 + k_slot(j), st = slot % ST;
                ok = __all_sync(0xffffffffu, pf_wait(&full[st], (slot / ST) & 1));
                if (!ok) return;
                pf_fence_after();
                const uint32_t qa = smem + qt * C::Q_BYTES, kb = smem + C::RING + st * C::KV_BYTES, d = tmem + (u & 1) * C::S_COLS;
#pragma unroll
                for (int x = 0; x < D / 16; x++)
                    pf_mma_ss(d, pf_desc_k(qa + (x >> 2) * (128 * 128) + (x & 3) * 32), pf_desc_k(kb + (x >> 2) * C::SLAB + (x & 3) * 32), idesc_s, x > 0);
                pf_commit(&s_full[u & 1]);
                if (!two || qt == 1) pf_commit(&empty[st]);
                if (u == units - 1) pf_commit(q_empty);
            };
            if (ok) scores(0);
            if (ok && units > 1) scores(1);
            for (int u = 0; u < units && ok; u++) {
                const int j = two ? u >> 1 : u, qt = two ? u & 1 : 0, slot = slot0 + v_slot(j), st = slot % ST;
                ok = __all_sync(0xffffffffu, pf_wait(&full[st], (slot / ST) & 1) && pf_wait(&p_full[u & 1], uses >> (u & 1) & 1));
                if (!ok) break;
                uses ^= 1u << (u & 1);
                pf_fence_after();
                const uint32_t vb = smem + C::RING + st * C::KV_BYTES, pa = tmem + (u & 1) * C::S_COLS, d = tmem + 256 + qt * D;
#pragma unroll
                for (int x = 0; x < BN / 16; x++) pf_mma_ts(d, pa + x * 8, pf_desc_n(vb + x * 2048, C::SLAB), idesc_o, j > 0 || x > 0);
                if (!two || qt == 1) pf_commit(&empty[st]);
                pf_commit(j == n - 1 ? &o_last[qt] : &o_done[qt]);   // the last commit of all is one that is waited for
                if (u + 2 < units) scores(u + 2);
            }
            slot0 += 2 * n;
            segments++;
        }
        if (!ok) {
            if (lane == 0) atomicOr(a.wait_status, 1u << 25);
            pf_commit(drain);                                // nothing of this CTA may still run when its memory is given back
            pf_wait(drain, 0);
        }
        if (lane == 0) a.desc[blockIdx.x] = begun;
        __syncwarp();
    } else {
        // ================================ loaders ================================
        asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
        const int lw = warp - C::SM_WARPS - 1;
        constexpr int NX = (BN / 4 + 2) / 3 * 4;             // rows of a warp: every third group of four
        constexpr int PER = (NX + 31) / 32;
        int64_t* offs = (int64_t*)(pf_smem + C::OFFS);
        const int boxes = a.box ? BN / a.box : 0;
        int slot0 = 0, segments = 0, handed = 0;             // ring slots and segments so far, slots handed over (copied rows only)
        for (; wk.more() && ok; wk.next(a)) {
        if (!wk.segment()) continue;
        const int n = wk.n, i0 = wk.i0, len = t.len, prefix = t.prefix, qhi = t.qhi;
        if (n == 0) continue;
        const int32_t* trow = a.c.table + (int64_t)wk.seq * a.c.table_stride;
        const uint16_t* kbase = a.c.k + wk.head * a.c.head_stride;
        const uint16_t* vbase = a.c.v + wk.head * a.c.head_stride;
        const int lo = a.o.window > 0 ? max(0, t.qlo - a.o.window + 1) : 0;
        auto row_of = [&](int x) { return (x >> 2) * 12 + lw * 4 + (x & 3); };
        auto key_of = [&](int j, int x) {                    // -1: a row nobody sees
            const int rr = row_of(x), key = t.kt.tile(i0 + j) * BN + rr;
            return x < NX && rr < BN && key < len && (key < prefix || (key >= lo && key <= qhi)) ? key : -1;
        };
        auto free_slot = [&](int slot) {
            ok = __all_sync(0xffffffffu, pf_wait(&empty[slot % ST], ((slot / ST) & 1) ^ 1));
            return ok;
        };
        // ---- row by row ----
        int page[PER];                                       // of this lane's rows of the next tile
        auto fetch_pages = [&](int j) {
#pragma unroll
            for (int e = 0; e < PER; e++) {
                const int key = j < n ? key_of(j, lane + 32 * e) : -1;
                page[e] = key >= 0 ? trow[paged_entry(a.c, key)] : 0;
            }
        };
        auto set_offsets = [&](int j) {
#pragma unroll
            for (int e = 0; e < PER; e++) {
                const int x = lane + 32 * e, key = key_of(j, x);
                if (x < NX && row_of(x) < BN) offs[(j & 1) * BN + row_of(x)] = key >= 0 ? paged_offset(a.c, page[e], paged_row(a.c, key)) : -1;
            }
            __syncwarp();
        };
        auto copy_rows = [&](int slot, const uint16_t* src, int j) {
            const int64_t* off = offs + (j & 1) * BN;
            const uint32_t dst = smem + C::RING + slot % ST * C::KV_BYTES;
            constexpr int CPR = D / 8, RPI = 32 / CPR, B = 4;    // 16-byte chunks per row, rows per instruction, instructions at once
            const int c = lane % CPR;
            src += c * 8;
#pragma unroll 1
            for (int x0 = 0; x0 < NX; x0 += RPI * B) {
                int64_t o[B];
#pragma unroll
                for (int b = 0; b < B; b++) {
                    const int x = x0 + b * RPI + lane / CPR;
                    o[b] = x < NX && row_of(x) < BN ? off[row_of(x)] : -2;
                }
#pragma unroll
                for (int b = 0; b < B; b++) {
                    const int rr = row_of(x0 + b * RPI + lane / CPR);
                    if (o[b] > -2)
                        cp_async16_zfill(dst + (c >> 3) * C::SLAB + rr * 128 + (((c & 7) ^ (rr & 7)) << 4), src + max(o[b], (int64_t)0), o[b] < 0 ? 0 : 16);
                }
            }
            paged_cp_commit();
        };
        // ---- by pages: lane i looks after box i of a tile ----
        int box_page = 0;
        auto box_key = [&](int j) {                          // -1: nobody sees a row of the box
            const int key = t.kt.tile(i0 + j) * BN + lane * a.box;
            return j < n && lane < boxes && key < len && (key < prefix || (key + a.box > lo && key <= qhi)) ? key : -1;
        };
        auto fetch_box_page = [&](int j) {
            const int key = box_key(j);
            return key >= 0 ? trow[paged_entry(a.c, key)] : 0;
        };
        auto copy_boxes = [&](int slot, const CUtensorMap* map, int j, int pages_of_tile) {
            const int key = box_key(j);
            const int in_page = key >= 0 ? paged_row(a.c, key) : -1;
            const int st = slot % ST, total = boxes * (D / 64), x = lane * 3 + lw;
            const int bx = min(x / (D / 64), 31), slab = x % (D / 64);
            const int pg = __shfl_sync(0xffffffffu, pages_of_tile, bx), row = __shfl_sync(0xffffffffu, in_page, bx);
            if (x < total && row >= 0) {
                mbar_expect_tx(&full[st], a.box * 128);
                pf_tma_4d(smem + C::RING + st * C::KV_BYTES + slab * C::SLAB + bx * a.box * 128, map, slab * 64, a.rows_first ? row : wk.head,
                          a.rows_first ? wk.head : row, pg, &full[st]);
            } else {
                pf_arrive(&full[st]);
            }
            __syncwarp();
        };
        // rows copied one by one are handed over when they have landed: LAG slots later where every slot is copied so
        auto hand_over = [&](int slot) {
            if (a.box) {
                paged_cp_wait<0>();
                pf_fence_async();
                pf_arrive(&full[slot % ST]);
            } else if (slot - handed >= C::LAG) {
                paged_cp_wait<C::LAG>();
                pf_fence_async();
                pf_arrive(&full[handed++ % ST]);
            }
        };
        // The segment's queries, when the last scores of the segment before are done: by TMA, or each warp every third 32 rows, of which
        // lane i knows where row i lies.
        auto load_queries = [&] {
            if (!a.box) {                                    // nothing may be waited for here that waits for a slot in flight
                paged_cp_wait<0>();
                pf_fence_async();
                while (handed < slot0 + k_slot(0) + 1) pf_arrive(&full[handed++ % ST]);
            }
            ok = __all_sync(0xffffffffu, pf_wait(q_empty, (segments & 1) ^ 1));
            if (!ok) return;
            const int tiles = t.two ? 2 : 1;
            if (a.q_box) {                                   // tokens behind the sequence's last are somebody else's, or zeros: never stored
                if (lw == 0 && lane < tiles * (D / 64)) {
                    const int qt = lane / (D / 64), slab = lane % (D / 64);
                    mbar_expect_tx(q_full, a.tokens * a.G * 128);
                    pf_tma_3d(smem + qt * C::Q_BYTES + slab * (128 * 128), &q_map, slab * 64, wk.head * a.G, t.span.x + t.tok0 + qt * a.tokens, q_full);
                } else {
                    pf_arrive(q_full);
                }
                __syncwarp();
                return;
            }
            constexpr int CPR = D / 8, RPI = 32 / CPR;       // 16-byte chunks per row, rows per instruction
            const int c = lane % CPR;
            for (int g0 = lw * 32; g0 < tiles * 128; g0 += 96) {
                const int rr0 = g0 & 127, mine = rr0 + lane, tk = mine / a.G, token = t.tok0 + (g0 >> 7) * a.tokens + tk;
                const int64_t at = tk < a.tokens && token < t.span.y
                                       ? (t.span.x + token) * a.q_stride + (int64_t)(wk.head * a.G + mine - tk * a.G) * D : -1;
                const uint32_t qs = smem + (g0 >> 7) * C::Q_BYTES;
#pragma unroll 8
                for (int i = 0; i < 32; i += RPI) {
                    const int x = i + lane / CPR, rr = rr0 + x;
                    const int64_t o = __shfl_sync(0xffffffffu, at, x);
                    cp_async16_zfill(qs + (c >> 3) * (128 * 128) + rr * 128 + (((c & 7) ^ (rr & 7)) << 4), a.q + (o < 0 ? 0 : o) + c * 8, o < 0 ? 0 : 16);
                }
            }
            paged_cp_commit();
            paged_cp_wait<0>();
            pf_fence_async();
            pf_arrive(q_full);
        };
        static_assert(16 * (D / 64) <= 96, "a lane issues one box");
        int v_page = 0, v_page2 = 0;                         // box pages of the K tiles whose V tile is still to come
        auto fill_k = [&](int j) {
            const int slot = slot0 + k_slot(j);
            if (!a.box) {
                set_offsets(j);
                fetch_pages(j + 1);
                if (!free_slot(slot)) return;
                copy_rows(slot, kbase, j);
            } else {
                const int pages_of_tile = box_page;
                box_page = fetch_box_page(j + 1);
                v_page2 = v_page;
                v_page = pages_of_tile;
                if (!free_slot(slot)) return;
                if (__all_sync(0xffffffffu, box_key(j) < 0 || (unsigned)pages_of_tile < (unsigned)a.c.pages)) {
                    copy_boxes(slot, &k_map, j, pages_of_tile);
                    return;
                }
                fetch_pages(j);                              // a bad page: reported, and zeros
                set_offsets(j);
                copy_rows(slot, kbase, j);
            }
            hand_over(slot);
        };
        auto fill_v = [&](int j) {
            const int slot = slot0 + v_slot(j);
            if (!free_slot(slot)) return;
            if (a.box) {
                const int pages_of_tile = t.two || j == n - 1 ? v_page : v_page2;
                const int k0 = t.kt.tile(i0 + j) * BN;
                const bool whole = k0 + BN <= len && (k0 + BN <= prefix || (k0 >= lo && k0 + BN - 1 <= qhi));
                if (whole && __all_sync(0xffffffffu, box_key(j) < 0 || (unsigned)pages_of_tile < (unsigned)a.c.pages)) {
                    copy_boxes(slot, &v_map, j, pages_of_tile);
                    return;
                }
                fetch_pages(j);
                set_offsets(j);
            }
            copy_rows(slot, vbase, j);
            hand_over(slot);
            __syncwarp();                                    // the offsets may be replaced
        };
        if (a.box) box_page = fetch_box_page(0);
        else fetch_pages(0);
        fill_k(0);
        if (ok) load_queries();
        if (t.two) {
            for (int j = 0; j < n && ok; j++) {
                fill_v(j);
                if (ok && j + 1 < n) fill_k(j + 1);
            }
        } else {
            if (ok && n > 1) fill_k(1);
            for (int j = 0; j < n && ok; j++) {
                fill_v(j);
                if (ok && j + 2 < n) fill_k(j + 2);
            }
        }
        slot0 += 2 * n;
        segments++;
        }
        // hand over the last slots
        paged_cp_wait<0>();
        if (ok && !a.box) {
            pf_fence_async();
            while (handed < slot0) pf_arrive(&full[handed++ % ST]);
        } else if (!ok && lane == 0) {
            atomicOr(a.wait_status, 1u << 24);
        }
        __syncwarp();
    }
    pf_fence_before();
    __syncthreads();
    if (warp == C::SM_WARPS) pf_tmem_dealloc(tmem, 512);
}

// Joins the parts of the pair that begins in CTA blockIdx.x and ends in another: a lane is a row, a thread 8 columns of it.
template <int D>
__global__ void __launch_bounds__(256) paged_prefill_join_kernel(const PrefillArgs a) {
    pdl_wait();
    constexpr int ROWS = PfCfg<D>::ROWS;
    const int4 ds = a.desc[blockIdx.x];
    if (ds.w < 0) return;
    const int item = blockIdx.y * 256 + threadIdx.x, r = item % ROWS, col = item / ROWS;
    const int2 span = prefill_span(a, ds.x);
    const int r_token = (r & 127) / a.G, token = (ds.y * PfCfg<D>::NQ + (r >> 7)) * a.tokens + r_token;
    if (r_token >= a.tokens || token >= span.y) return;
    float m = -INFINITY, l = 0.f, x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int c = blockIdx.x; c <= ds.w; c++) {
        const int slot = 2 * c + (c == (int)blockIdx.x ? 1 : 0);
        const float2 ml = a.ml[slot * ROWS + r];
        const float4* src = a.part + ((int64_t)slot * (D / 4) + 2 * col) * ROWS + r;
        const float4 p = src[0], q = src[ROWS];
        const float nm = fmaxf(m, ml.x), ref = nm == -INFINITY ? 0.f : nm;
        const float e0 = ex2(m - ref), e1 = ex2(ml.x - ref);     // -inf -> 0
        m = nm;
        l = l * e0 + ml.y * e1;
        x[0] = x[0] * e0 + p.x * e1; x[1] = x[1] * e0 + p.y * e1; x[2] = x[2] * e0 + p.z * e1; x[3] = x[3] * e0 + p.w * e1;
        x[4] = x[4] * e0 + q.x * e1; x[5] = x[5] * e0 + q.y * e1; x[6] = x[6] * e0 + q.z * e1; x[7] = x[7] * e0 + q.w * e1;
    }
    const float inv = l > 0.f ? 1.0f / l : 0.f;
    const int64_t tok = span.x + token;
    const int head = ds.z * a.G + (r & 127) - r_token * a.G;
    *(uint4*)(a.out + tok * a.out_stride + (int64_t)head * D + col * 8) =
        make_uint4(pack_bf16x2(x[0] * inv, x[1] * inv), pack_bf16x2(x[2] * inv, x[3] * inv), pack_bf16x2(x[4] * inv, x[5] * inv), pack_bf16x2(x[6] * inv, x[7] * inv));
    if (a.lse && col == 0) a.lse[tok * a.Hq + head] = (m + log2f(l)) * 0.6931471805599453f;
}

struct PrefillPlan { int ctas; size_t part, ml, desc, total; };
// one CTA per SM, fewer where the work (bounded by max_ctx keys per sequence) has fewer parts
static PrefillPlan prefill_plan(int D, int kv_heads, int seqs, int total_q, int q_heads, int max_ctx) {
    PrefillPlan p;
    const int rows = D == 256 ? 128 : 256, bn = D == 256 ? 64 : 128, tokens = rows / 128 * (128 / (q_heads / kv_heads));
    const int64_t tiles = std::min<int64_t>((int64_t)total_q / tokens + seqs, total_q);   // each sequence may end in one of its own
    const int64_t units = tiles * kv_heads * (PF_START + ((int64_t)max_ctx + bn - 1) / bn * (rows == 256 ? PF_TWO : PF_ONE));
    p.ctas = (int)std::max<int64_t>(1, std::min<int64_t>(paged_sm_count(), units / PF_LEAST));
    auto up = [](size_t b) { return (b + 255) & ~(size_t)255; };
    p.part = up((size_t)2 * p.ctas * rows * D * 4);
    p.ml = up((size_t)2 * p.ctas * rows * 8);
    p.desc = up((size_t)p.ctas * 16);
    p.total = p.part + p.ml + p.desc;
    return p;
}

typedef CUresult (*EncodeTiled)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
static EncodeTiled encode_tiled() {
    static EncodeTiled fn = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        return cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess
                   ? (EncodeTiled)p : nullptr;
    }();
    return fn;
}
// Tensor maps of the pools with boxes of 64 head dimensions by gcd(page size, bn) rows. False where the pool has no such form (page
// sizes that are not multiples of 8 rows, strides that do not nest): its rows are copied one by one.
static bool prefill_maps(const PagedCache& c, int D, int bn, CUtensorMap* km, CUtensorMap* vm, int* box, int* rows_first) {
    if (c.page_size % 8 || !encode_tiled()) return false;
    *box = std::gcd(c.page_size, bn);
    *rows_first = c.row_stride < c.head_stride;
    const int64_t s1 = *rows_first ? c.row_stride : c.head_stride, s2 = *rows_first ? c.head_stride : c.row_stride, s3 = c.page_stride;
    const int64_t n1 = *rows_first ? c.page_size : c.kv_heads, n2 = *rows_first ? c.kv_heads : c.page_size;
    if (s1 < D || s2 % s1 || s3 % s2 || s2 < s1 * n1 || s3 < s2 * n2 || s3 >= (int64_t)1 << 39) return false;
    const cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)n1, (cuuint64_t)n2, (cuuint64_t)std::max(1, c.pages)};
    const cuuint64_t strides[3] = {(cuuint64_t)s1 * 2, (cuuint64_t)s2 * 2, (cuuint64_t)s3 * 2};
    const cuuint32_t boxes[4] = {64, *rows_first ? (cuuint32_t)*box : 1, *rows_first ? 1 : (cuuint32_t)*box, 1}, es[4] = {1, 1, 1, 1};
    for (int i = 0; i < 2; i++)
        if (encode_tiled()(i ? vm : km, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, i ? c.v : c.k, dims, strides, boxes, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
                           CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
            return false;
    return true;
}

// Tensor map of the queries: boxes of 64 head dimensions by the G heads of a kv head by the tokens of a row tile.
static bool prefill_q_map(const PrefillArgs& a, int D, CUtensorMap* qm) {
    if (a.q_stride % D || a.q_stride >= (int64_t)1 << 38 || !encode_tiled()) return false;
    const cuuint64_t dims[3] = {(cuuint64_t)D, (cuuint64_t)a.Hq, (cuuint64_t)a.total_q};
    const cuuint64_t strides[2] = {(cuuint64_t)D * 2, (cuuint64_t)a.q_stride * 2};
    const cuuint32_t boxes[3] = {64, (cuuint32_t)a.G, (cuuint32_t)a.tokens}, es[3] = {1, 1, 1};
    return encode_tiled()(qm, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, (void*)a.q, dims, strides, boxes, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int D, int FEAT>
static int32_t launch_prefill(cudaStream_t s, PrefillArgs a, int ctas) {
    using C = PfCfg<D>;
    static uint32_t attr_devs = 0;
    static std::mutex mu;
    int dev = 0;
    LTHN_CUDA_TRY(cudaGetDevice(&dev));
    {
        std::lock_guard<std::mutex> lk(mu);
        if (!(attr_devs >> (dev & 31) & 1)) {
            LTHN_CUDA_TRY(cudaFuncSetAttribute(paged_prefill_kernel<D, FEAT>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::TOTAL));
            attr_devs |= 1u << (dev & 31);
        }
    }
    CUtensorMap qm = {}, km = {}, vm = {};
    a.q_box = prefill_q_map(a, D, &qm);
    if (!prefill_maps(a.c, D, C::BN, &km, &vm, &a.box, &a.rows_first)) a.box = 0;
    paged_prefill_kernel<D, FEAT><<<ctas, C::THREADS, C::TOTAL, s>>>(qm, km, vm, a);
    LTHN_CUDA_TRY(cudaGetLastError());
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(ctas, C::ROWS * (D / 8) / 256); cfg.blockDim = dim3(256); cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at; cfg.numAttrs = 1;
    LTHN_CUDA_TRY(cudaLaunchKernelEx(&cfg, paged_prefill_join_kernel<D>, a));
    return LTHN_OK;
}
template <int D>
static int32_t launch_prefill_feat(cudaStream_t s, const PrefillArgs& a, int ctas) {
    const int f = (a.o.softcap > 0.f ? 1 : 0) | (a.o.slopes ? 2 : 0);
    return f == 0 ? launch_prefill<D, 0>(s, a, ctas) : f == 1 ? launch_prefill<D, 1>(s, a, ctas) : f == 2 ? launch_prefill<D, 2>(s, a, ctas) : launch_prefill<D, 3>(s, a, ctas);
}

}  // namespace lthn

using namespace lthn;

static int32_t prefill_check(const lthn_paged_kv* cache, int32_t seqs, int32_t total_q, int32_t q_heads, int32_t max_ctx, PagedCache* c) {
    int32_t rc;
    if ((rc = paged_check_cache("paged_prefill_attention", cache, c))) return rc;
    LTHN_REQUIRE(seqs >= 0 && total_q >= 0 && max_ctx >= 0, "paged_prefill_attention: negative size");
    LTHN_REQUIRE(seqs <= 32768, "paged_prefill_attention: at most 32768 sequences per call");
    LTHN_REQUIRE(seqs <= cache->seqs, "paged_prefill_attention: more sequences than the page table has");
    LTHN_REQUIRE(q_heads > 0 && q_heads <= 65535 && q_heads % cache->kv_heads == 0, "paged_prefill_attention: q_heads must be a positive multiple of kv_heads");
    LTHN_REQUIRE(q_heads / cache->kv_heads <= 128, "paged_prefill_attention: at most 128 query heads per kv head");
    LTHN_REQUIRE(total_q <= 1 << 30, "paged_prefill_attention: too many query rows");
    return LTHN_OK;
}
extern "C" {

int32_t lthn_paged_prefill_attention_workspace(const lthn_paged_kv* cache, int32_t seqs, int32_t total_q, int32_t q_heads, int32_t max_ctx,
                                               size_t* bytes) {
    clear_error();
    LTHN_REQUIRE(bytes != nullptr, "paged_prefill_attention_workspace: bytes is NULL");
    PagedCache c;
    int32_t rc;
    if ((rc = prefill_check(cache, seqs, total_q, q_heads, max_ctx, &c))) return rc;
    *bytes = prefill_plan(cache->head_dim, cache->kv_heads, seqs, total_q, q_heads, max_ctx ? std::min(max_ctx, c.capacity) : c.capacity).total;
    return LTHN_OK;
}

int32_t lthn_paged_prefill_attention(void* stream, const lthn_paged_kv* cache, const lthn_attn_options* options, const uint16_t* q,
                                     int64_t q_stride, const int32_t* q_start, const int32_t* kv_lens, int32_t seqs, int32_t total_q,
                                     int32_t q_heads, int32_t max_ctx, uint16_t* out, int64_t out_stride, float* lse, void* workspace,
                                     size_t workspace_bytes) {
    clear_error();
    const char* me = "paged_prefill_attention";
    PrefillArgs a = {};
    int32_t rc;
    if ((rc = prefill_check(cache, seqs, total_q, q_heads, max_ctx, &a.c))) return rc;
    const int D = cache->head_dim;
    if ((rc = paged_check_options(me, options, D, &a.o))) return rc;
    if (seqs == 0 || total_q == 0) return LTHN_OK;
    LTHN_REQUIRE(q && out && q_start && kv_lens && workspace, "paged_prefill_attention: NULL pointer");
    a.q_stride = q_stride ? q_stride : (int64_t)q_heads * D;
    a.out_stride = out_stride ? out_stride : (int64_t)q_heads * D;
    LTHN_REQUIRE(((a.q_stride | a.out_stride) & 7) == 0, "paged_prefill_attention: strides must be multiples of 8 elements");
    LTHN_REQUIRE(a.q_stride >= (int64_t)q_heads * D && a.out_stride >= (int64_t)q_heads * D, "paged_prefill_attention: rows of q or out would overlap");
    LTHN_REQUIRE((((uintptr_t)q | (uintptr_t)out | (uintptr_t)workspace) & 15) == 0, "paged_prefill_attention: q, out and workspace must be 16-byte aligned");
    const PrefillPlan p = prefill_plan(D, cache->kv_heads, seqs, total_q, q_heads, max_ctx ? std::min(max_ctx, a.c.capacity) : a.c.capacity);
    LTHN_REQUIRE(workspace_bytes >= p.total, "paged_prefill_attention: workspace too small");
    if ((rc = paged_check_device(me, "the cache", cache->k))) return rc;
    if ((rc = paged_check_device(me, "q", q))) return rc;
    a.q = q; a.out = out; a.q_start = q_start; a.lens = kv_lens; a.lse = lse;
    a.seqs = seqs; a.total_q = total_q; a.Hq = q_heads; a.G = q_heads / cache->kv_heads;
    a.tokens = 128 / a.G;
    a.part = (float4*)workspace;
    a.ml = (float2*)((char*)workspace + p.part);
    a.desc = (int4*)((char*)workspace + p.part + p.ml);
    a.wait_status = device_status_word();
    a.c.status = device_paged_status_word();
    if (!a.c.status) return fail(LTHN_ERR_CUDA, "paged_prefill_attention: no device status word");
    if (D == 64) return launch_prefill_feat<64>((cudaStream_t)stream, a, p.ctas);
    if (D == 128) return launch_prefill_feat<128>((cudaStream_t)stream, a, p.ctas);
    return launch_prefill_feat<256>((cudaStream_t)stream, a, p.ctas);
}

}  // extern "C"
