// paged_prefill.cu — attention of packed prompt chunks over the paged KV cache on the Blackwell tensor cores.
//
//   out = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m),   s_j = cap(q.k_j scale) - slope |i - j|,   m = max_j s_j
//
// 4*D flops per visible (query, key) pair against 4*D bytes of K and V per key and tile of query rows: bound by the tensor pipe
// for prompts, by HBM for a few rows against a long context.
//
// Rows. The query rows of a tile are the (token, query head) pairs of one kv head, token by token, as many whole tokens as
// 128 rows hold, so the heads that share K and V share their loads, a chunk of a few tokens still fills a tile, and the
// queries of a tile are one TMA box per 64 head dimensions. A CTA works on BN keys at a time and on one tile of 128 rows,
// or two for head_dim 64 and 128, where two accumulators fit the tensor memory beside two score tiles.
//
//   softmax warps   two warpgroups, one per score buffer, one thread per row: tcgen05.ld the row's BN scores, mask, maximum, ex2,
//                   sum - all within the thread - and tcgen05.st the weights as bf16 over the scores they came from.
//   issuer          one warp: S = Q K^T (both operands in shared memory), O += P V (P in tensor memory, V in shared
//                   memory as an N-major operand, so it is stored as it comes). There are two score buffers. Unit u uses
//                   buffer u & 1 and the issue order is S(0) S(1) | O(0) S(2) | O(1) S(3) | ..., so that the tensor pipe
//                   works on one buffer while the other's softmax runs. With two row tiles the buffers belong to them;
//                   with one they alternate over its key tiles, and the warpgroups pass the running maximum of a row to one
//                   another (the sums stay apart until the end), which leaves only load and maximum in sequence.
//   loaders         three warps fetch the queries of an item and fill a ring of K and V tiles in the 128-byte swizzle. Where
//                   the page size is a multiple of 8 (the swizzle's row group) by tiled TMA, one box per page, 64 head
//                   dimensions and gcd(page size, BN) rows. V rows that nobody sees must be zeros (they may hold NaN,
//                   which a weight of zero would not silence), so a V tile with such rows - the last of a sequence, the
//                   first of a window - and pools of other page sizes come row by row with cp.async of 16 bytes,
//                   zero-filled; unseen K rows may hold anything, their scores are replaced. 8192 tokens of 32 heads: 1007 us with cp.async throughout, 541 us with TMA
//                   as it was then; pages of other sizes still cost about twice.
//
// Weights are rounded to bf16 (2^-8 each, the size of the rounding of the output) because the second product takes one type for both operands
// and V is bf16; a second product with the remainders, as in the one-token kernel, would cost half as much again of what bounds long prompts.
// The sums take the weights before that rounding.
//
// The running maximum is only moved when a row's grew by more than 2^8: until then weights are up to 2^8, which neither
// their bf16 rounding (relative) nor the f32 sums mind, and O in tensor memory needs no correction. A move multiplies
// O by 2^(old - new) through registers; after the first tiles it is rare.
//
// Work. An item is (row tile, kv head, chunk of its key tiles); the grid has one CTA per item, the longest first, but only as many
// run as there are SMs: a CTA that is through with loading an item cancels the launch of a waiting one
// (clusterlaunchcontrol) and takes its item over, so barriers, tensor memory and pipeline stay up and the loads of the next item run under
// the last products and the output of this one. One of the loader warps does this and publishes the item to the other
// roles. (One CTA per item spent 7 us of each on its start and end: 7 packed chunks of up to 1500 tokens took 201 us against 186. A fixed
// even share per CTA of a list weighted by cost loses more than that: what a key tile costs depends on its mask and on who shares it in L2.)
// Where there are few items the keys of a tile are cut into chunks, which leave (maximum, sum, unnormalised output)
// in the workspace for a second kernel to join.
//
// Every wait is bounded: on a time-out the roles record it in the device status word and leave; when all have, the loaders wait for the
// boxes and the answer that are still on their way to this CTA's shared memory and the issuer for its products, then the tensor memory is
// freed and the CTA returns.
#include "paged.cuh"

#include <cuda.h>

#include <algorithm>
#include <cmath>
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
    int out_sectors;     // the rows of out lie on 32-byte boundaries
    int q_box;           // queries by TMA (their row stride is a multiple of head_dim), else copied row by row
    int tiles;           // upper bound of the row tiles of all sequences
    int chunks;          // chunks per row tile and kv head
    int chunk_tiles;     // key tiles per chunk, unless the lengths call for others
    int levels, sms;     // key tiles of max_ctx
    int give_up;         // tests: a role that never starts (1 softmax, 2 issuer, 3 one of the loaders), so that the others' waits run out
    float4* part;        // [tiles*kv_heads*chunks][D/4][rows] unnormalised outputs, four columns each
    float2* ml;          // [tiles*kv_heads*chunks][rows] maximum (log2 units) and sum
    int4* desc;          // [tiles] sequence, tile of the sequence, chunks in use
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

// What the roles need to know of an item; one lies in shared memory while the next is worked out.
struct PfItem {
    int seq, head;       // head < 0: no more items
    int first, tokens;   // the sequence's rows of q
    int len, pos0;       // keys; position of the first query
    int prefix;
    int tok0;            // first token of the row tiles
    int qlo, qhi;        // positions of their first and last token
    int two;             // both row tiles have tokens
    KeyTiles kt;
    int i0, n;           // key tiles [i0, i0 + n) of kt; n = 0 where nobody sees anything
    int part;            // place in the workspace, -1: not cut, the output is final
};
// What a call says of a sequence.
struct PfSeq { int first, tokens, len, prefix; };
__device__ __forceinline__ PfSeq prefill_seq(const PrefillArgs& a, int s) {
    PfSeq q = {0, 0, 0, 0};
    if (s >= a.seqs) return q;
    const int len = a.lens[s], prefix = a.o.prefix ? a.o.prefix[s] : 0;
    const int2 span = prefill_span(a, s);
    q.first = span.x;
    q.tokens = span.y;
    q.len = paged_length(a.c, len);
    q.prefix = min(max(prefix, 0), q.len);
    return q;
}
template <int NQ, int BN>
__device__ __forceinline__ PfItem prefill_tile(const PrefillArgs& a, const PfSeq& q, int seq, int tile) {
    PfItem t;
    t.seq = seq;
    t.first = q.first;
    t.tokens = q.tokens;
    t.len = q.len;
    t.pos0 = t.len - t.tokens;
    t.prefix = q.prefix;
    t.tok0 = tile * NQ * a.tokens;
    t.qlo = t.pos0 + t.tok0;
    t.qhi = t.pos0 + min(t.tok0 + NQ * a.tokens, t.tokens) - 1;
    t.kt = key_tiles<BN>(t.qlo, t.qhi, t.len, t.prefix, a.o.window);
    t.two = NQ == 2 && t.tokens - t.tok0 > a.tokens;
    return t;
}

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
__device__ __forceinline__ void pf_prefetch_map(const CUtensorMap* map) { asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory"); }
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
// 32 bytes of a lane to global memory
__device__ __forceinline__ void pf_store_sector(void* p, const uint32_t (&w)[8]) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
                 ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7]) : "memory");
}
__device__ __forceinline__ void pf_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

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
__device__ __forceinline__ int warp_sum_int(int v) { return (int)__reduce_add_sync(0xffffffffu, (unsigned)v); }
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
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
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

constexpr float CAP_SMALL = 64.0f, CAP_NEAR = 0.3f;

// FEAT bit 0: tanh cap of at most CAP_SMALL, bit 1: distance bias, bit 2: a larger cap
// 168 registers a thread at launch, and spills of 48 to 260 bytes; head_dim 64 under a large cap has the most.
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
    uint64_t* p_half = s_full + 2;                           // [2] the first half of the weights is there, O is corrected
    uint64_t* p_full = p_half + 2;                           // [2] the other half is
    uint64_t* o_done = p_full + 2;                           // [2] per row tile: O(u) has been added, all but the last
    uint64_t* o_last = o_done + 2;                           // [2] the last has (a barrier of its own: with one row tile the softmax
                                                             //     may be two units ahead, which a parity cannot tell from none)
    uint64_t* turn = o_last + 2;                             // [4] one row tile: the maximum of key tile j is out, per 32 rows
    uint64_t* q_full = turn + 4;                             // queries of an item
    uint64_t* q_empty = q_full + 1;                          // its last scores are done
    uint64_t* meet = q_empty + 1;                            // both softmax warpgroups (a barrier whose wait is bounded)
    uint64_t* drain = meet + 1;
    uint64_t* item_full = drain + 1;                         // [2] the item is there
    uint64_t* item_empty = item_full + 2;                    // [2] everybody has read it
    uint64_t* answered = item_empty + 2;
    uint32_t* tmem_slot = (uint32_t*)(answered + 1);
    unsigned char* answer = pf_smem + C::BARS + 320;         // 16 bytes
    PfItem* items = (PfItem*)(answer + 16);                  // [2]
    int* gave_up = (int*)(items + 2);                        // [8] whether a role has; then, of each loader warp that has left, the ring slots and
                                                             //     the queries it had arrived for; the question without an answer, -1: none
    static_assert((2 * ST + 23) * 8 + 8 <= 320 && 336 + 2 * sizeof(PfItem) + 32 <= 512, "barriers, items and what is left behind");

    const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
    pdl_trigger();                                           // of the join, which waits for the end of this grid
    PfSeq seq_here = {0, 0, 0, 0};                           // the last warp, which finds the items: sequence `lane`
    if (warp == C::SM_WARPS + 1 && lane < 3 && (lane < 2 ? a.box : a.q_box)) pf_prefetch_map(lane == 0 ? &k_map : lane == 1 ? &v_map : &q_map);
    if (warp == C::WARPS - 1) seq_here = prefill_seq(a, lane);
    if (tid == 0) {
        for (int s = 0; s < ST; s++) { mbar_init(&full[s], 96); mbar_init(&empty[s], 1); }
        for (int b = 0; b < 2; b++) {
            mbar_init(&s_full[b], 1); mbar_init(&p_half[b], 128); mbar_init(&p_full[b], 128);
            mbar_init(&o_done[b], 1); mbar_init(&o_last[b], 1);
            mbar_init(&item_full[b], 1); mbar_init(&item_empty[b], C::WARPS);
        }
        for (int w = 0; w < 4; w++) mbar_init(&turn[w], 1);
        mbar_init(q_full, 96);
        mbar_init(q_empty, 1);
        mbar_init(meet, C::SM_WARPS * 32);
        mbar_init(drain, 1);
        mbar_init(answered, 1);
        gave_up[0] = 0;
        for (int x = 1; x < 8; x++) gave_up[x] = -1;
        mbar_fence_init();
    }
    if (warp == C::SM_WARPS) pf_tmem_alloc(tmem_slot, 512);
    pf_fence_before();
    __syncthreads();
    pf_fence_after();
    const uint32_t tmem = *tmem_slot;
    const uint32_t smem = smem_u32(pf_smem);
    bool ok = true;
    PfItem t;
    int items_read = 0;
    // the next item for this warp; false: there are no more
    auto next_item = [&] {
        const int b = items_read & 1;
        ok = __all_sync(0xffffffffu, paged_wait(&item_full[b], (items_read >> 1) & 1));
        if (!ok) return false;
        t = items[b];
        __syncwarp();
        if (lane == 0) pf_arrive(&item_empty[b]);
        items_read++;
        return t.head >= 0;
    };

    // The j-th key tile of an item. A distance bias lets scores rise towards the query, and with them the maximum at every tile, so
    // those go from the newest keys to the oldest (4 drafts on contexts up to 40000: 61 us against 59).
    auto tile_at = [&](int j) { return t.kt.tile(FEAT & 2 ? t.i0 + t.n - 1 - j : t.i0 + j); };
    // ring slots of the K and V tile of key tile j of an item, in the order of their last use
    auto k_slot = [&](int j) { return t.two ? 2 * j : j < 2 ? j : 2 * j - 1; };
    auto v_slot = [&](int j) { return t.two ? 2 * j + 1 : j == t.n - 1 ? 2 * t.n - 1 : 2 * j + 2; };

    if (warp < C::SM_WARPS) {
        // ================================ softmax ================================
        asm volatile("setmaxnreg.inc.sync.aligned.u32 200;");
        const int wg = warp >> 2;                            // score buffer = warpgroup
        const int wr = (warp & 3) * 32, r = wr + lane;       // row within the row tile = tensor memory lane
        const int r_token = r / a.G, r_head = r - r_token * a.G;
        const uint32_t lanes = tmem + ((uint32_t)wr << 16);
        const uint32_t s_addr = lanes + wg * C::S_COLS;
        // plain scores and those under a large cap stay in units of the product, the others are brought to log2 units first
        const float c1 = FEAT & 3 ? 1.0f : a.o.scale * LOG2E;
        const float u_in = paged_cap_in(a.o), e_in = 2.0f * LOG2E * fminf(u_in, 1e38f), cap = FEAT & 4 ? a.o.softcap / a.o.scale : a.o.softcap * LOG2E;
        auto far_from_zero = [&](float x) { return fmaf(-2.0f * cap, rcp_approx(1.0f + ex2(x * e_in)), cap); };
        float* row_max = (float*)(pf_smem + C::ROW_MAX);     // one row tile only
        int uses = 0;                                        // of this warpgroup's score buffer
        int turns = 0, done0 = 0, done1 = 0, last0 = 0, last1 = 0, meets = 0;  // phases the barriers have gone through
        if (a.give_up == 1) ok = false;
        auto pair_sync = [&] {
            pf_arrive(meet);
            const bool met = __all_sync(0xffffffffu, paged_wait(meet, meets++ & 1));
            ok = ok && met;
        };
        while (ok && next_item()) {
            const bool two = t.two;
            const int n = t.n, qt = two ? wg : 0, len = t.len;
            const int token = t.tok0 + qt * a.tokens + r_token;  // of the sequence
            const bool live = r_token < a.tokens && token < t.tokens;
            const int head = t.head * a.G + r_head;
            const int qpos = t.pos0 + token;
            // visible: key < pre, or klo <= key < khi
            const int pre = t.prefix, khi = min(qpos + 1, len), klo = a.o.window > 0 ? qpos - a.o.window + 1 : 0;
            const float slope = (FEAT & 2) && live ? a.o.slopes[head] * LOG2E : 0.f;
            const uint32_t o_addr = lanes + 256 + qt * D;
            float m = -INFINITY, l = 0.f;                        // reference maximum (units of the scores), sum relative to it

            for (int j = two ? 0 : wg; j < n; j += two ? 1 : 2) {
                ok = __all_sync(0xffffffffu, paged_wait(&s_full[wg], uses & 1));
                if (!ok) break;
                uses++;
                pf_fence_after();
                float s[BN];
#pragma unroll
                for (int x = 0; x < BN; x += 32) pf_ld32(s_addr + x, s + x);
                pf_ld_wait();
                const int k0 = tile_at(j) * BN;
                if (FEAT & 1) {
                    // cap tanh(x / cap) = cap (1 - 2 / (1 + e^(2 x / cap))), off by 1.6 * 2^-23 of the cap: 1.2e-5 at most up to CAP_SMALL
#pragma unroll
                    for (int x = 0; x < BN; x++) s[x] = far_from_zero(s[x]);
                }
                if (FEAT & 4) {
                    // Large caps: an error relative to the score, not to the cap. Where |u| = |x / cap| < CAP_NEAR: x + x u^2 P(u^2), with P the fit of
                    // (tanh(u) / u - 1) / u^2 of least error there (2^-24.5 of tanh u, 2^-23.4 with the f32 roundings). Beyond, the form above,
                    // whose error is 2^-20.5 of the score or less there.
                    float top[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int x = 0; x < BN; x += 8)
#pragma unroll
                        for (int e = 0; e < 4; e++) top[e] = max3(top[e], fabsf(s[x + e]), fabsf(s[x + 4 + e]));
                    const bool near = fmaxf(max3(top[0], top[1], top[2]), top[3]) * u_in < CAP_NEAR;
                    const uint64_t in2 = pack2(u_in, u_in);
                    const uint64_t p1 = pack2(-0.33333287f, -0.33333287f), p2 = pack2(0.13323873f, 0.13323873f), p3 = pack2(-0.051132675f, -0.051132675f);
                    auto near_zero = [&](float x0, float x1, float& y0, float& y1) {
                        const uint64_t x = pack2(x0, x1), u = mul2(x, in2), w = mul2(u, u);
                        unpack2(fma2(x, mul2(w, fma2(w, fma2(w, p3, p2), p1)), x), y0, y1);
                    };
                    if (__all_sync(0xffffffffu, near)) {
#pragma unroll
                        for (int x = 0; x < BN; x += 2) near_zero(s[x], s[x + 1], s[x], s[x + 1]);
                    } else {
#pragma unroll
                        for (int x = 0; x < BN; x += 2) {
                            float y0, y1;
                            near_zero(s[x], s[x + 1], y0, y1);
                            s[x] = fabsf(s[x]) * u_in < CAP_NEAR ? y0 : far_from_zero(s[x]);
                            s[x + 1] = fabsf(s[x + 1]) * u_in < CAP_NEAR ? y1 : far_from_zero(s[x + 1]);
                        }
                    }
                }
                if (FEAT & 2) {
                    const float gap = (float)(qpos - k0);
#pragma unroll
                    for (int x = 0; x < BN; x++) s[x] = fmaf(-slope, fabsf(gap - (float)x), FEAT & 1 ? s[x] : s[x] * (a.o.scale * LOG2E));
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
                    ok = __all_sync(0xffffffffu, paged_wait(&turn[warp & 3], (turns + j - 1) & 1));
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
                    ok = __all_sync(0xffffffffu, paged_wait(&o_done[qt], ((qt ? done1 : done0) + j - 1) & 1));
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
                    if (x == BN / 2 - 32 || x == BN - 32) {      // the product with V begins with the first half
                        pf_st_wait();
                        pf_fence_before();
                        pf_arrive(x == BN - 32 ? &p_full[wg] : &p_half[wg]);
                    }
                }
                float l0, l1;
                unpack2(add2(sum[0], sum[1]), l0, l1);
                l += l0 + l1;
            }
            if (ok && n > 0) ok = __all_sync(0xffffffffu, paged_wait(&o_last[qt], (qt ? last1 : last0) & 1));
            int x0 = 0, x1 = D;                                  // output columns of this warpgroup
            if (!two && n > 0) {
                // the two sums of a row meet, relative to the last maximum; each warpgroup stores half of the columns
                if (ok) ok = __all_sync(0xffffffffu, paged_wait(&turn[warp & 3], (turns + n - 1) & 1));
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
                const int64_t tok = t.first + token;
                const float m2 = m * c1;                         // log2 units (c1 > 0)
                const float inv = l > 0.f ? 1.0f / l : 0.f;
                uint16_t* dst = a.out + tok * a.out_stride + (int64_t)head * D;
                const bool whole = t.part < 0;
                float4* part = a.part + (int64_t)t.part * (D / 4) * ROWS + qt * 128 + r;
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
                        for (int e = 0; e < 32; e += 16) {
                            uint32_t w[8];
#pragma unroll
                            for (int p = 0; p < 8; p++) w[p] = pack_bf16x2(o[e + 2 * p] * inv, o[e + 2 * p + 1] * inv);
                            if (a.out_sectors) {             // 7 packed chunks: 180 us in 16-byte stores, 175.5 in whole sectors
                                pf_store_sector(dst + x + e, w);
                            } else {
                                *(uint4*)(dst + x + e) = make_uint4(w[0], w[1], w[2], w[3]);
                                *(uint4*)(dst + x + e + 8) = make_uint4(w[4], w[5], w[6], w[7]);
                            }
                        }
                    } else {
#pragma unroll
                        for (int e = 0; e < 32; e += 4) part[(x + e) / 4 * ROWS] = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
                    }
                }
                if (live && x0 == 0) {
                    if (!whole) a.ml[(int64_t)t.part * ROWS + qt * 128 + r] = make_float2(m2, l);
                    else if (a.lse) a.lse[tok * a.Hq + head] = (m2 + log2f(l)) * 0.6931471805599453f;
                }
            }
            if (!two && n > 0) pair_sync();                      // both have read O before the next item's first weights let it be replaced
        }
        if (!ok && lane == 0) {
            gave_up[0] = 1;
            atomicOr(a.wait_status, 1u << 26);
        }
    } else if (warp == C::SM_WARPS) {
        // ================================ issuer ================================
        asm volatile("setmaxnreg.dec.sync.aligned.u32 104;");
        // f32 accumulators, bf16 operands, M = 128; S: N = BN, both K-major; O: N = D, B is N-major
        const uint32_t idesc = (1u << 4) | (1u << 7) | (1u << 10) | ((128u >> 4) << 24);
        const uint32_t idesc_s = idesc | ((uint32_t)(BN >> 3) << 17), idesc_o = idesc | (1u << 16) | ((uint32_t)(D >> 3) << 17);
        int slot0 = 0, seen = 0;                             // ring slots and items with keys so far
        uint32_t uses = 0;                                   // bit b: parity of the uses of score buffer b
        if (a.give_up == 2) ok = false;
        while (ok && next_item()) {
            const bool two = t.two;
            const int n = t.n, units = two ? 2 * n : n;
            if (n == 0) continue;
            ok = __all_sync(0xffffffffu, paged_wait(q_full, seen & 1));
            auto scores = [&](int u) {
                const int j = two ? u >> 1 : u, qt = two ? u & 1 : 0, slot = slot0 + k_slot(j), st = slot % ST;
                ok = __all_sync(0xffffffffu, paged_wait(&full[st], (slot / ST) & 1));
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
                const uint32_t vb = smem + C::RING + st * C::KV_BYTES, pa = tmem + (u & 1) * C::S_COLS, d = tmem + 256 + qt * D;
                ok = __all_sync(0xffffffffu, paged_wait(&full[st], (slot / ST) & 1) && paged_wait(&p_half[u & 1], uses >> (u & 1) & 1));
                if (!ok) break;
                pf_fence_after();
#pragma unroll
                for (int x = 0; x < BN / 32; x++) pf_mma_ts(d, pa + x * 8, pf_desc_n(vb + x * 2048, C::SLAB), idesc_o, j > 0 || x > 0);
                ok = __all_sync(0xffffffffu, paged_wait(&p_full[u & 1], uses >> (u & 1) & 1));
                if (!ok) break;
                pf_fence_after();
                uses ^= 1u << (u & 1);
#pragma unroll
                for (int x = BN / 32; x < BN / 16; x++) pf_mma_ts(d, pa + x * 8, pf_desc_n(vb + x * 2048, C::SLAB), idesc_o, 1u);
                if (!two || qt == 1) pf_commit(&empty[st]);
                pf_commit(j == n - 1 ? &o_last[qt] : &o_done[qt]);   // the last commit of all is one that is waited for
                if (u + 2 < units) scores(u + 2);
            }
            slot0 += 2 * n;
            seen++;
        }
        if (!ok && lane == 0) {
            gave_up[0] = 1;
            atomicOr(a.wait_status, 1u << 25);
        }
        __syncwarp();
    } else {
        // ================================ loaders ================================
        asm volatile("setmaxnreg.dec.sync.aligned.u32 104;");
        const int lw = warp - C::SM_WARPS - 1;
        constexpr int NX = (BN / 4 + 2) / 3 * 4;             // rows of a warp: every third group of four
        constexpr int PER = (NX + 31) / 32;
        int64_t* offs = (int64_t*)(pf_smem + C::OFFS);
        const int boxes = a.box ? BN / a.box : 0;
        int slot0 = 0, seen = 0, handed = 0;                 // ring slots and items with keys so far, slots handed over (copied rows only)
        // ---- the last of the three warps also finds the items ----
        const bool finder = lw == 2;
        int tiles_here = 0, tiles = 0, published = 0, asked = 0;  // row tiles of sequence `lane`, of all sequences; items, questions so far
        int levels = 0, chunk_tiles = a.chunk_tiles;         // key tiles of the longest sequence, of a chunk
        auto tiles_in = [&](int tokens) { return (tokens + C::NQ * a.tokens - 1) / (C::NQ * a.tokens); };
        auto tiles_of = [&](int sq) { return sq < a.seqs ? tiles_in(prefill_span(a, sq).y) : 0; };
        auto warp_scan = [&](int v) {
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int u = __shfl_up_sync(0xffffffffu, v, o);
                if (lane >= o) v += u;
            }
            return v;
        };
        // Item `id` in `x`; false: there is no such tile or chunk. First chunks come before second ones, so that what is left of a tile's
        // keys comes last, and the row tiles in the order of their last key, the farthest first; with more than 32 sequences that
        // holds within a sequence only.
        auto look_up = [&](int id, PfItem& x) {
            const int rest = id / a.c.kv_heads, chunk = rest / a.tiles, tile_id = rest % a.tiles;
            if (tile_id >= tiles) {
                if (a.chunks > 1 && chunk == 0 && id % a.c.kv_heads == 0 && lane == 0) a.desc[tile_id] = make_int4(0, 0, 0, 0);
                return false;
            }
            int want = tiles - 1 - tile_id, sq = 0, count = tiles_here;
            if (a.seqs > 1 && a.seqs <= 32) {
                // the tile's level, the key tile that its last token is in: more than tile_id tiles are at level lo or behind, not so at hi
                int lo = 0, hi = levels + 1, at_lo = tiles_here, at_hi = 0, before = 0;
                while (hi - lo > 1) {
                    const int mid = (lo + hi) >> 1, token = (mid - 1) * BN - (seq_here.len - seq_here.tokens);   // of this lane's sequence, first of the level
                    int there = token < 0 ? tiles_here : token >= seq_here.tokens ? 0 : tiles_here;
                    if (there > 1 && token > 0) there -= token / (C::NQ * a.tokens);
                    const int total = warp_sum_int(there);
                    if (total > tile_id) { lo = mid; at_lo = there; }
                    else { hi = mid; at_hi = there; before = total; }
                }
                const int incl = warp_scan(at_lo - at_hi), rank = tile_id - before;
                sq = __ffs(__ballot_sync(0xffffffffu, incl > rank)) - 1;
                want = __shfl_sync(0xffffffffu, tiles_here - 1 - at_hi + incl - (at_lo - at_hi), sq) - rank;
            } else {
                for (int s0 = 0;; s0 += 32, count = tiles_of(s0 + lane)) {
                    const int incl = warp_scan(count), total = __shfl_sync(0xffffffffu, incl, 31);
                    if (want < total) {
                        const int l = __ffs(__ballot_sync(0xffffffffu, incl > want)) - 1;
                        want -= __shfl_sync(0xffffffffu, incl - count, l);
                        sq = s0 + l;
                        break;
                    }
                    want -= total;
                    if (s0 + 32 >= a.seqs) return false;     // only if q_start changed under the call
                }
            }
            PfSeq of;
            if (sq < 32) {
                of.first = __shfl_sync(0xffffffffu, seq_here.first, sq);
                of.tokens = __shfl_sync(0xffffffffu, seq_here.tokens, sq);
                of.len = __shfl_sync(0xffffffffu, seq_here.len, sq);
                of.prefix = __shfl_sync(0xffffffffu, seq_here.prefix, sq);
            } else {
                of = prefill_seq(a, sq);
            }
            x = prefill_tile<C::NQ, BN>(a, of, sq, want);
            x.head = id % a.c.kv_heads;
            const int per = max(chunk_tiles, (x.kt.n + a.chunks - 1) / a.chunks);     // also where max_ctx was too small
            const int used = a.chunks > 1 ? max(1, (x.kt.n + per - 1) / per) : 1;
            if (a.chunks > 1 && chunk == 0 && x.head == 0 && lane == 0) a.desc[tile_id] = make_int4(sq, want, used, 0);
            if (chunk >= used) return false;
            x.i0 = chunk * per;
            x.n = a.chunks > 1 ? min(per, x.kt.n - x.i0) : x.kt.n;
            x.part = used > 1 ? (tile_id * a.c.kv_heads + x.head) * a.chunks + chunk : -1;
            return true;
        };
        auto publish = [&](const PfItem& x) {
            const int b = published & 1;
            ok = ok && __all_sync(0xffffffffu, paged_wait(&item_empty[b], ((published >> 1) & 1) ^ 1));
            if (!ok) return;
            if (lane == 0) {
                items[b] = x;
                pf_arrive(&item_full[b]);
            }
            published++;
            __syncwarp();
        };
        auto find_next = [&] {
            PfItem x;
            for (;;) {
                if (lane == 0) {
                    pf_fence_async();                        // the last answer has been read
                    mbar_expect_tx(answered, 16);
                    paged_try_cancel(answer, answered);
                }
                __syncwarp();
                ok = ok && __all_sync(0xffffffffu, paged_wait(answered, asked & 1));
                if (!ok) {
                    if (lane == 0) gave_up[7] = asked;
                    return;
                }
                asked++;
                const int id = paged_cancelled(answer);
                __syncwarp();
                if (id < 0) {
                    x.head = -1;
                    break;
                }
                if (look_up(id, x)) break;
            }
            publish(x);
        };
        if (finder) {
            tiles_here = tiles_in(seq_here.tokens);
            for (int s0 = 0; s0 < a.seqs; s0 += 32) tiles += warp_sum_int(s0 ? tiles_of(s0 + lane) : tiles_here);
            levels = (int)__reduce_max_sync(0xffffffffu, (unsigned)((seq_here.len + BN - 1) / BN));
            if (a.chunks > 1 && a.seqs <= 32 && tiles * a.c.kv_heads <= a.sms && (a.seqs > 1 || levels * 8 < a.levels * 7)) {
                // lengths other than max_ctx say better how to cut: the shortest chunks, 256 keys at least, with which all run at once
                const int n1 = tiles_here ? prefill_tile<C::NQ, BN>(a, seq_here, lane, tiles_here - 1).kt.n : 0;
                const int n0 = tiles_here > 1 ? prefill_tile<C::NQ, BN>(a, seq_here, lane, 0).kt.n : n1;
                int hi = (int)__reduce_max_sync(0xffffffffu, (unsigned)max(n0, n1)), lo = max(256 / BN, (hi + a.chunks - 1) / a.chunks);
                const float mean = 0.5f * (n0 + n1);
                while (lo < hi) {
                    const int mid = (lo + hi) >> 1;
                    const float each = mean * (1.0f / mid);  // chunks of a tile; of those of several tiles the last is half full on average
                    const int mine = (int)ceilf(tiles_here > 1 ? tiles_here * (each + 0.5f) : each);
                    if (warp_sum_int(mine) * a.c.kv_heads <= a.sms) hi = mid;
                    else lo = mid + 1;
                }
                chunk_tiles = lo;
            }
            PfItem x;
            if (look_up(blockIdx.x, x)) publish(x);
            else find_next();
        }
        if (a.give_up == 3 && lw == 1) ok = false;
        while (ok && next_item()) {
            const int n = t.n, len = t.len, prefix = t.prefix, qhi = t.qhi;
            if (n == 0) {
                if (finder) find_next();
                continue;
            }
            const int32_t* trow = a.c.table + (int64_t)t.seq * a.c.table_stride;
            const uint16_t* kbase = a.c.k + t.head * a.c.head_stride;
            const uint16_t* vbase = a.c.v + t.head * a.c.head_stride;
            const int lo = a.o.window > 0 ? max(0, t.qlo - a.o.window + 1) : 0;
            auto row_of = [&](int x) { return (x >> 2) * 12 + lw * 4 + (x & 3); };
            auto key_of = [&](int j, int x) {                    // -1: a row nobody sees
                const int rr = row_of(x), key = tile_at(j) * BN + rr;
                return x < NX && rr < BN && key < len && (key < prefix || (key >= lo && key <= qhi)) ? key : -1;
            };
            auto left_at = [&](int slot, int queries) {
                if (lane == 0) { gave_up[1 + lw] = slot; gave_up[4 + lw] = queries; }
            };
            auto free_slot = [&](int slot) {
                ok = __all_sync(0xffffffffu, paged_wait(&empty[slot % ST], ((slot / ST) & 1) ^ 1));
                if (!ok) left_at(slot, slot > slot0 ? seen + 1 : seen);   // (slots are filled in their order, the queries come behind the first)
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
                const int key = tile_at(j) * BN + lane * a.box;
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
                    pf_tma_4d(smem + C::RING + st * C::KV_BYTES + slab * C::SLAB + bx * a.box * 128, map, slab * 64, a.rows_first ? row : t.head,
                              a.rows_first ? t.head : row, pg, &full[st]);
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
            // The item's queries, when the last scores of the item before are done: by TMA, or each warp every third 32 rows, of which
            // lane i knows where row i lies.
            auto load_queries = [&] {
                if (!a.box) {                                    // nothing may be waited for here that waits for a slot in flight
                    paged_cp_wait<0>();
                    pf_fence_async();
                    while (handed < slot0 + k_slot(0) + 1) pf_arrive(&full[handed++ % ST]);
                }
                ok = __all_sync(0xffffffffu, paged_wait(q_empty, (seen & 1) ^ 1));
                if (!ok) {
                    left_at(slot0 + 1, seen);
                    return;
                }
                const int row_tiles = t.two ? 2 : 1;
                if (a.q_box) {                                   // tokens behind the sequence's last are somebody else's, or zeros: never stored
                    if (lw == 0 && lane < row_tiles * (D / 64)) {
                        const int qt = lane / (D / 64), slab = lane % (D / 64);
                        mbar_expect_tx(q_full, a.tokens * a.G * 128);
                        pf_tma_3d(smem + qt * C::Q_BYTES + slab * (128 * 128), &q_map, slab * 64, t.head * a.G, t.first + t.tok0 + qt * a.tokens, q_full);
                    } else {
                        pf_arrive(q_full);
                    }
                    __syncwarp();
                    return;
                }
                constexpr int CPR = D / 8, RPI = 32 / CPR;       // 16-byte chunks per row, rows per instruction
                const int c = lane % CPR;
                for (int g0 = lw * 32; g0 < row_tiles * 128; g0 += 96) {
                    const int rr0 = g0 & 127, mine = rr0 + lane, tk = mine / a.G, token = t.tok0 + (g0 >> 7) * a.tokens + tk;
                    const int64_t at = tk < a.tokens && token < t.tokens
                                           ? (t.first + token) * a.q_stride + (int64_t)(t.head * a.G + mine - tk * a.G) * D : -1;
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
                    const int k0 = tile_at(j) * BN;
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
            seen++;
            if (finder && ok) find_next();                       // all loads of this item are on their way
        }
        // hand over the last slots
        paged_cp_wait<0>();
        if (ok && !a.box) {
            pf_fence_async();
            while (handed < slot0) pf_arrive(&full[handed++ % ST]);
        } else if (!ok && lane == 0) {
            gave_up[0] = 1;
            atomicOr(a.wait_status, 1u << 24);
        }
        if (lane == 0 && gave_up[1 + lw] < 0) { gave_up[1 + lw] = slot0; gave_up[4 + lw] = seen; }   // it left between two items
        __syncwarp();
    }
    pf_fence_before();
    __syncthreads();
    if (gave_up[0]) {
        // Nothing of this CTA may still run or be written when its memory is given back. A phase of `full` takes the arrivals of all
        // three warps: those that left earlier make up for what the others have arrived for since. That is at most ST slots, one of each
        // stage, and one item's queries: a stage is filled again, as are the queries, only after all three had arrived for it.
        if (warp == C::SM_WARPS) {
            pf_commit(drain);                                // all products
            paged_wait(drain, 0);
        } else if (warp > C::SM_WARPS) {
            const int lw = warp - C::SM_WARPS - 1, *slots = gave_up + 1, *queries = gave_up + 4;
            if (a.box) {                                     // (rows copied one by one have been waited for)
                const int last = max(slots[0], max(slots[1], slots[2]));
                for (int s = slots[lw]; s < last; s++) pf_arrive(&full[s % ST]);
                for (int s = max(last - ST, 0); s < last; s++) paged_wait(&full[s % ST], (s / ST) & 1);
            }
            if (a.q_box) {
                const int last = max(queries[0], max(queries[1], queries[2]));
                if (queries[lw] < last) pf_arrive(q_full);
                if (last > 0) paged_wait(q_full, (last - 1) & 1);
            }
            if (lw == 2 && gave_up[7] >= 0) paged_wait(answered, gave_up[7] & 1);
        }
        __syncthreads();
    }
    if (warp == C::SM_WARPS) pf_tmem_dealloc(tmem, 512);
}

// Joins the chunks of a row tile. A lane is a row, a warp 8 columns of 32 rows and every CG-th chunk; with CG > 1 the warps of a column group
// meet in shared memory. CG = 1 for up to 8 chunks: no barrier, few CTAs (4 chunks of 68 tiles: 3 us, 17 with CG = 8). CG = 8
// above, where its CTAs run in two waves at most: one thread's chain of loads over the chunks would take longer than the CTAs it saves
// (18 chunks of 16 tiles: 3 us less).
template <int D, int CG>
__global__ void __launch_bounds__(256) paged_prefill_join_kernel(const PrefillArgs a) {
    constexpr int ROWS = PfCfg<D>::ROWS, GROUPS = 8 / CG;        // column groups of a CTA
    __shared__ float2 s_ml[CG > 1 ? 8 : 1][32];
    __shared__ float s_x[CG > 1 ? 8 : 1][8][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, kvh = blockIdx.y;
    constexpr int PER_ROWS = D / 8 / GROUPS;                     // CTAs per 32 rows
    const int r = blockIdx.z / PER_ROWS * 32 + lane, col = blockIdx.z % PER_ROWS * GROUPS + warp / CG;
    pdl_wait();
    const int4 ds = a.desc[blockIdx.x];
    if (ds.z <= 1 || ds.z > a.chunks || (unsigned)ds.x >= (unsigned)a.seqs || (unsigned)ds.y >= (unsigned)a.tiles) return;   // (a CTA that gave up)
    const int2 span = prefill_span(a, ds.x);
    const int r_token = (r & 127) / a.G, token = (ds.y * PfCfg<D>::NQ + (r >> 7)) * a.tokens + r_token;
    const bool live = r_token < a.tokens && token < span.y;
    const int64_t first = ((int64_t)blockIdx.x * a.c.kv_heads + kvh) * a.chunks;
    float m = -INFINITY, l = 0.f, x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (live) {
#pragma unroll 4
        for (int c = warp % CG; c < ds.z; c += CG) {
            const float2 ml = a.ml[(first + c) * ROWS + r];
            const float4* src = a.part + ((first + c) * (D / 4) + 2 * col) * ROWS + r;
            const float4 p = src[0], q = src[ROWS];
            const float nm = fmaxf(m, ml.x), ref = nm == -INFINITY ? 0.f : nm;
            const float e0 = ex2(m - ref), e1 = ex2(ml.x - ref);     // -inf -> 0
            m = nm;
            l = l * e0 + ml.y * e1;
            x[0] = x[0] * e0 + p.x * e1; x[1] = x[1] * e0 + p.y * e1; x[2] = x[2] * e0 + p.z * e1; x[3] = x[3] * e0 + p.w * e1;
            x[4] = x[4] * e0 + q.x * e1; x[5] = x[5] * e0 + q.y * e1; x[6] = x[6] * e0 + q.z * e1; x[7] = x[7] * e0 + q.w * e1;
        }
    }
    if (CG > 1) {
        s_ml[warp % 8][lane] = make_float2(m, l);
#pragma unroll
        for (int e = 0; e < 8; e++) s_x[warp % 8][e][lane] = x[e];
        __syncthreads();
        if (warp > 0) return;
#pragma unroll
        for (int w = 0; w < CG; w++) m = fmaxf(m, s_ml[w][lane].x);
        const float ref = m == -INFINITY ? 0.f : m;
        l = 0.f;
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] = 0.f;
#pragma unroll
        for (int w = 0; w < CG; w++) {
            const float2 ml = s_ml[w][lane];
            const float e1 = ex2(ml.x - ref);
            l = fmaf(ml.y, e1, l);
#pragma unroll
            for (int e = 0; e < 8; e++) x[e] = fmaf(s_x[w][e][lane], e1, x[e]);
        }
    }
    if (!live) return;
    const float inv = l > 0.f ? 1.0f / l : 0.f;
    const int64_t tok = span.x + token;
    const int head = kvh * a.G + (r & 127) - r_token * a.G;
    *(uint4*)(a.out + tok * a.out_stride + (int64_t)head * D + col * 8) =
        make_uint4(pack_bf16x2(x[0] * inv, x[1] * inv), pack_bf16x2(x[2] * inv, x[3] * inv), pack_bf16x2(x[4] * inv, x[5] * inv), pack_bf16x2(x[6] * inv, x[7] * inv));
    if (a.lse && col == 0) a.lse[tok * a.Hq + head] = (m + log2f(l)) * 0.6931471805599453f;
}

struct PrefillPlan { int tiles, levels, chunks, chunk_tiles; size_t part, ml, desc, total; };
// Cutting the keys of a tile. With no more (row tile, kv head) pairs than SMs they are cut as far as all chunks still run at once, into 256
// keys at least: below, the partial outputs and the join cost what they save (1024 tokens of 8 heads of 256, 64 pairs: 26.9 us in 96 chunks of
// up to 512 keys, 24.8 in 120 of up to 384, 28.9 in 160 of up to 256, which do not all run at once). `chunk_tiles` is what that comes to for
// sequences of max_ctx; a call whose lengths are others finds its own from them, for which there is room for twice the chunks
// (8 tokens behind 4096 keys, max_ctx 131072: 27.6 us with chunks made for max_ctx, 14.4 with its own). With more pairs than SMs a
// tile is cut whose keys are a good deal more than half of an SM's share of the work, so that the longest does not decide the time, but not
// below 512 keys.
static PrefillPlan prefill_plan(int D, int kv_heads, int seqs, int total_q, int q_heads, int max_ctx, int window, bool has_prefix) {
    PrefillPlan p;
    const int rows = D == 256 ? 128 : 256, bn = D == 256 ? 64 : 128, tokens = rows / 128 * (128 / (q_heads / kv_heads)), sms = paged_sm_count();
    p.tiles = (int)std::min<int64_t>((int64_t)total_q / tokens + std::min(seqs, total_q), total_q);   // each sequence may end in one of its own
    p.levels = (max_ctx + bn - 1) / bn;
    const int64_t pairs = (int64_t)p.tiles * kv_heads;
    // key tiles of the longest row tile, and of an average one: the mean over a sequence's new rows is half of them less
    double keys = max_ctx, mean = std::max(0.5 * max_ctx, max_ctx - 0.5 * total_q / std::max(1, seqs));
    if (window > 0 && !has_prefix) {
        keys = std::min(keys, (double)window + tokens + bn);
        mean = std::min(mean, keys);
    }
    const double longest = keys / bn, each = std::max(1.0, mean / bn), half = 0.5 * each * pairs / sms;
    p.chunks = (int)std::max(1.0, std::min(longest / std::max((pairs <= sms ? 256.0 : 512.0) / bn, half), 1024.0));
    p.chunk_tiles = std::max(1, (int)((longest + p.chunks - 1) / p.chunks));
    // The other roles wait 0.2 s for the next item at the most. A look-up reads the sequences before the item's, 12 ns each, and of the up to
    // 4 * 148 chunks one CTA may come upon all that are not there, one after another; without chunks each look-up finds an item.
    if (seqs > 1 << 15) p.chunks = 1;
    if (pairs <= sms) p.chunk_tiles = std::max(p.chunk_tiles, (int)std::ceil(each / ((double)sms / pairs - 0.5)));   // a tile's last chunk is half full
    auto up = [](size_t b) { return (b + 255) & ~(size_t)255; };
    const size_t parts = p.chunks > 1 ? (size_t)pairs * p.chunks : 0;
    p.part = up(parts * rows * D * 4);
    p.ml = up(parts * rows * 8);
    p.desc = p.chunks > 1 ? up((size_t)p.tiles * 16) : 0;
    p.total = std::max<size_t>(16, p.part + p.ml + p.desc);
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

LTHN_HIDDEN int g_paged_give_up = 0;  // PrefillArgs::give_up: zero in the product library (setter: test_hooks.cu)

template <int D, int FEAT>
static int32_t launch_prefill(cudaStream_t s, PrefillArgs a) {
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
    paged_prefill_kernel<D, FEAT><<<a.tiles * a.c.kv_heads * a.chunks, C::THREADS, C::TOTAL, s>>>(qm, km, vm, a);
    LTHN_CUDA_TRY(cudaGetLastError());
    if (a.chunks > 1) {
        const int64_t ctas = (int64_t)a.tiles * a.c.kv_heads * (C::ROWS / 32 * (D / 8));    // of CG = 8; an SM runs 8
        const bool few = a.chunks <= 8 || ctas > 16 * a.sms;
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(a.tiles, a.c.kv_heads, C::ROWS / 32 * (few ? D / 64 : D / 8)); cfg.blockDim = dim3(256); cfg.stream = s;
        cudaLaunchAttribute at[1];
        at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        at[0].val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = at; cfg.numAttrs = 1;
        LTHN_CUDA_TRY(few ? cudaLaunchKernelEx(&cfg, paged_prefill_join_kernel<D, 1>, a) : cudaLaunchKernelEx(&cfg, paged_prefill_join_kernel<D, 8>, a));
    }
    return LTHN_OK;
}
template <int D>
static int32_t launch_prefill_feat(cudaStream_t s, const PrefillArgs& a) {
    // 8192 tokens of 32 heads of 128 under a cap of 100: 917 us in the form of the small caps, 720 in that of the large ones, 1154 there where
    // scores pass CAP_NEAR. Small caps stay with theirs: 1024 tokens of 8 heads of 256 take 25.0 us in it, 25.9 in the other, more code to fetch.
    switch ((a.o.softcap > CAP_SMALL ? 4 : a.o.softcap > 0.f ? 1 : 0) | (a.o.slopes ? 2 : 0)) {
        case 0: return launch_prefill<D, 0>(s, a);
        case 1: return launch_prefill<D, 1>(s, a);
        case 2: return launch_prefill<D, 2>(s, a);
        case 3: return launch_prefill<D, 3>(s, a);
        case 4: return launch_prefill<D, 4>(s, a);
        default: return launch_prefill<D, 6>(s, a);
    }
}

}  // namespace lthn

using namespace lthn;

static int32_t prefill_check(const lthn_paged_kv* cache, int32_t seqs, int32_t total_q, int32_t q_heads, int32_t max_ctx, PagedCache* c) {
    int32_t rc;
    if ((rc = paged_check_cache("paged_prefill_attention", cache, c))) return rc;
    LTHN_REQUIRE(seqs >= 0 && total_q >= 0 && max_ctx >= 0, "paged_prefill_attention: negative size");
    LTHN_REQUIRE(seqs <= cache->seqs, "paged_prefill_attention: more sequences than the page table has");
    LTHN_REQUIRE(seqs <= 1 << 20, "paged_prefill_attention: at most 2^20 sequences");   // 12 ms a look-up
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
    // without options: a window only makes the longest and the average tile shorter and more alike, so there are fewer pieces
    *bytes = prefill_plan(cache->head_dim, cache->kv_heads, seqs, total_q, q_heads, max_ctx ? std::min(max_ctx, c.capacity) : c.capacity, 0, false).total;
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
    const PrefillPlan p = prefill_plan(D, cache->kv_heads, seqs, total_q, q_heads, max_ctx ? std::min(max_ctx, a.c.capacity) : a.c.capacity, a.o.window,
                                       a.o.prefix != nullptr);
    // more than the queries of a whole device's memory come to; items that are not there take a CTA 1 us each, 0.1 s in all
    LTHN_REQUIRE((int64_t)p.tiles * cache->kv_heads * p.chunks < 1 << 24, "paged_prefill_attention: too many query rows or sequences");
    LTHN_REQUIRE(workspace_bytes >= p.total, "paged_prefill_attention: workspace too small");
    if ((rc = paged_check_pointers(me, {{"the cache's k", cache->k, 16, false}, {"the cache's v", cache->v, 16, false},
                                        {"page_table", cache->page_table, 4, true}, {"q", q, 16, false}, {"q_start", q_start, 4, true},
                                        {"kv_lens", kv_lens, 4, true}, {"out", out, 16, true}, {"lse", lse, 4, true}, {"workspace", workspace, 16, false},
                                        {"slopes", a.o.slopes, 4, true}, {"prefix_lens", a.o.prefix, 4, true}})))
        return rc;
    a.out_sectors = (((uintptr_t)out | (uintptr_t)(a.out_stride * 2)) & 31) == 0;
    a.q = q; a.out = out; a.q_start = q_start; a.lens = kv_lens; a.lse = lse;
    a.seqs = seqs; a.total_q = total_q; a.Hq = q_heads; a.G = q_heads / cache->kv_heads;
    a.tokens = 128 / a.G;
    a.tiles = p.tiles; a.chunks = p.chunks; a.chunk_tiles = p.chunk_tiles; a.levels = p.levels; a.sms = paged_sm_count();
    a.give_up = g_paged_give_up;
    a.part = (float4*)workspace;
    a.ml = (float2*)((char*)workspace + p.part);
    a.desc = (int4*)((char*)workspace + p.part + p.ml);
    a.wait_status = device_status_word();
    a.c.status = device_paged_status_word();
    if (!a.c.status) return fail(LTHN_ERR_CUDA, "paged_prefill_attention: no device status word");
    if (D == 64) return launch_prefill_feat<64>((cudaStream_t)stream, a);
    if (D == 128) return launch_prefill_feat<128>((cudaStream_t)stream, a);
    return launch_prefill_feat<256>((cudaStream_t)stream, a);
}

}  // extern "C"
