// paged_decode.cu — attention of one new token per sequence over the paged KV cache, split over the length and joined.
//
//   out = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m),   s_j = cap(q.k_j scale) - slope |i - j|,   m = max_j s_j
//
// Every visible K and V row has to be read once: 4*D bytes per key and kv head against 4*D*G flops (G query heads share a
// kv head), so HBM is the bound as long as the arithmetic of a group of query heads stays below it. With 8 or more query
// heads per kv head it does not on the FMA pipe (G/2 multiply-adds per byte), so the products run on mma.sync with the query heads
// as the M rows, where up to 16 heads cost what one costs.
//
// Work. The pieces (64 keys) of all (row, kv head, bundle of query heads) triples form one list, row by row, in which a triple begins with
// two units for its start; CTA c of C takes units [U c / C, U (c+1) / C) of the U, so every CTA has the same work whatever the
// lengths are, and no host knowledge of them is needed. (Without the units of the start the CTAs with many short
// triples came last: 32 rows of 257 to 4608 keys, first CTA done after 66 us, last after 99.) A triple that lies within one CTA
// is finished there; otherwise each CTA that holds part of it leaves (max, sum, unnormalised output) in its slot of the workspace
// - a CTA has at most two such parts, its first and its last - and a second kernel joins them. A few short triples would wait for the
// second launch longer than for their keys; each of those goes to a cluster of 8 or 16 CTAs, whose parts meet in distributed shared memory.
//
// A warp owns 16 keys of each piece and runs on its own: its own ring of shared-memory stages filled by its own cp.async (16 bytes,
// rows padded by 16 bytes so that ldmatrix is free of bank conflicts), its own running maximum, sum and output; the
// four warps meet at the end of a triple only, in the one stage of their rings that the next triple's first keys, already
// on their way then, leave free. Rows outside the visible range are filled with zeros instead of
// read: they may hold NaN, which a weight of zero would not silence.
//
// Types. K and V are exact in bf16. Bundles of up to 8 heads leave half of the 16 MMA rows free, and the free rows carry
// what rounding to bf16 cuts off:
//   bf16, <= 8 heads   rows 0-7 the weights rounded to bf16, rows 8-15 the remainders: the weights are good to 2^-16
//   bf16, > 8 heads    16 heads, weights rounded to bf16 (2^-8 each, no more than the rounding of the output)
//   f32                q and the weights as three bf16 parts (24 bits), two MMAs: rows 0-7 high, 8-15 middle; rows 0-7 low
#include "paged.cuh"

#include <algorithm>
#include <mutex>

namespace lthn {

enum { DEC_BF16_16 = 0, DEC_BF16_8 = 1, DEC_F32_8 = 2 };

struct DecodeArgs {
    PagedCache c;
    AttnOpts o;
    const void* q;
    void* out;
    int64_t q_stride, out_stride;
    const int32_t* lens;
    float* lse;
    int rows, Hq, G;      // G: query heads per kv head
    int nb;               // bundles per kv head
    int ctas;
    float* part;          // [2*ctas][HB][D] unnormalised outputs
    float2* ml;           // [2*ctas][HB] maximum (log2 units) and sum
    int64_t* base;        // [rows + 1] units before each row, and of all (written where there are more rows than the join scans)
};

constexpr int DEC_WARPS = 4;
constexpr int DEC_THREADS = DEC_WARPS * 32;
constexpr int DEC_WK = 16;                       // keys of a warp's tile
constexpr int DEC_TILE = DEC_WARPS * DEC_WK;

template <int D, int MODE>
struct DecCfg {
    static constexpr int HB = MODE == DEC_BF16_16 ? 16 : 8;
    static constexpr int NST = D == 64 ? 4 : 3;
    static constexpr int PITCH = D * 2 + 16;                    // bytes of a shared-memory row
    static constexpr int STAGE = 2 * DEC_WK * PITCH;            // K rows, then V rows
    static constexpr int QROWS = MODE == DEC_F32_8 ? 24 : MODE == DEC_BF16_16 ? 16 : 8;
    static constexpr int Q_BYTES = QROWS * PITCH;
    static constexpr int RING = DEC_WARPS * NST * STAGE;
    static constexpr size_t SMEM = (size_t)RING + Q_BYTES;
    static constexpr int CTAS_PER_SM = D == 256 ? 1 : 2;
    static_assert((SMEM + 2048) * CTAS_PER_SM <= 233472, "shared memory of an SM");
    static_assert(HB * D * 4 <= STAGE, "a stage holds a warp's output");
};

__device__ __forceinline__ KeyTiles decode_tiles(const DecodeArgs& a, int row) {
    const int len = paged_length(a.c, a.lens[row]);
    return key_tiles<DEC_TILE>(len - 1, len - 1, len, a.o.prefix ? a.o.prefix[row] : 0, a.o.window);
}

// Units of a triple of n pieces: its start and end cost about what two pieces cost (32 rows of 257 to 4608 keys: 97.8 us with 1, 96.6 with 2, 96.9 with 3).
constexpr int DEC_START = 2;
__device__ __forceinline__ int decode_units(int n) { return n > 0 ? n + DEC_START : 0; }
// n / d for n >= 0, d > 0: in 32 bits where they fit (a 64-bit division is a long call, and it stands before a CTA's first load)
__device__ __forceinline__ int64_t decode_div(int64_t n, int64_t d) {
    return ((n | d) >> 32) == 0 ? (int64_t)((uint32_t)n / (uint32_t)d) : n / d;
}
// the CTA that holds unit x
__device__ __forceinline__ int decode_cta_of(int64_t x, int64_t U, int ctas) { return (int)decode_div((x + 1) * ctas - 1, U); }

// capped, biased score in log2 units. x: the raw product; in: scale / cap or scale * log2 e; cap, slope: times log2 e
__device__ __forceinline__ float decode_score(float x, float in, float cap, float slope, int gap) {
    x *= in;
    if (cap > 0.f) x = cap * tanhf(x);
    return fmaf(-slope, (float)abs(gap), x);
}

// part of a triple
struct DecSeg {
    int row, kvh, bundle;
    int len, prefix, lo;  // visible: key < prefix, or lo <= key < len
    KeyTiles kt;
    int i0, i1;           // pieces
};

__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}
// address of a CTA's copy of a shared-memory variable
__device__ __forceinline__ uint32_t cluster_map(uint32_t addr, int cta) {
    uint32_t d;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(d) : "r"(addr), "r"(cta));
    return d;
}
__device__ __forceinline__ float4 cluster_ld4(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ float2 cluster_ld2(uint32_t addr) {
    float2 v;
    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
    return v;
}

// CLUSTER > 0: a triple belongs to a cluster of that many CTAs, an even share of its pieces each, and their parts meet in shared memory.
template <int D, int MODE, int CLUSTER>
__global__ void __launch_bounds__(DEC_THREADS, DecCfg<D, MODE>::CTAS_PER_SM) paged_decode_kernel(const DecodeArgs a) {
    using C = DecCfg<D, MODE>;
    constexpr int HB = C::HB, NST = C::NST, PITCH = C::PITCH;
    constexpr int KS = D / 16;                    // k-steps of q.k
    constexpr int ND = D / 8;                     // output n-tiles
    constexpr int NR = MODE == DEC_BF16_16 ? 2 : 1;   // head rows of a thread
    constexpr float LOG2E = 1.4426950408889634f;
    extern __shared__ __align__(128) unsigned char dec_smem[];
    __shared__ float s_m[DEC_WARPS][16], s_l[DEC_WARPS][16];
    __shared__ int s_scan[DEC_WARPS];
    __shared__ int s_row, s_base;
    __shared__ __align__(8) float2 s_part[HB];    // CLUSTER: maximum and sum of this CTA's part

    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int g = lane >> 2, t = lane & 3;
    unsigned char* q_sm = dec_smem + C::RING;
    const uint32_t q_addr = smem_u32(q_sm);
    const uint32_t ring = smem_u32(dec_smem) + warp * NST * C::STAGE;
    const int triples = a.c.kv_heads * a.nb;      // per row

    if (!CLUSTER) pdl_trigger();
    // ---- this CTA's units ------------------------------------------------------------------------------
    int64_t u = 0, u1 = 0, base = 0;
    int row = 0;
    if (!CLUSTER) {
        auto units_of = [&](int r) { return r < a.rows ? decode_units(decode_tiles(a, r).n) : 0; };
        int incl, mine = units_of(tid);
        int total = paged_block_scan<DEC_WARPS>(mine, incl, s_scan);
        int64_t U = total;                            // per triple of a row first
        const bool note = a.rows > DEC_THREADS && blockIdx.x == 0;   // the join looks them up
        if (note) a.base[tid] = incl - mine;
        for (int r0 = DEC_THREADS; r0 < a.rows; r0 += DEC_THREADS) {
            int x;
            const int n = units_of(r0 + tid), more = paged_block_scan<DEC_WARPS>(n, x, s_scan);
            if (note && r0 + tid < a.rows) a.base[r0 + tid] = U + x - n;
            U += more;
        }
        if (note && tid == 0) a.base[a.rows] = U;
        U *= triples;
        const int ctas = (int)min((int64_t)a.ctas, U);   // none of them without a unit
        if ((int)blockIdx.x >= ctas) return;
        const int64_t u0 = decode_div(U * blockIdx.x, ctas);
        u = u0;
        u1 = decode_div(U * (blockIdx.x + 1), ctas);
        // the row that holds unit u0
        for (int r0 = 0;;) {
            if ((base + total) * triples > u0) {
                if (mine > 0 && (base + incl) * triples > u0 && (base + incl - mine) * triples <= u0) { s_row = r0 + tid; s_base = incl - mine; }
                __syncthreads();
                row = s_row;
                base = (base + s_base) * triples;     // first unit of the row
                break;
            }
            base += total;
            r0 += DEC_THREADS;
            mine = units_of(r0 + tid);
            total = paged_block_scan<DEC_WARPS>(mine, incl, s_scan);
        }
    }
    const float s_in = a.o.softcap > 0.f ? paged_cap_in(a.o) : a.o.scale * LOG2E, s_cap = a.o.softcap * LOG2E;

    constexpr int CC = CLUSTER > 0 ? CLUSTER : 1;
    const int rank = blockIdx.x % CC, my_triple = blockIdx.x / CC;   // of a cluster
    bool begun = false;
    auto next_seg = [&](DecSeg& d) {              // the next part of a triple; false: there is none
        auto fill = [&](int at, int triple, const KeyTiles& kt) {
            d.row = at;
            d.kvh = triple / a.nb;
            d.bundle = triple - d.kvh * a.nb;
            d.len = paged_length(a.c, a.lens[at]);
            d.prefix = a.o.prefix ? min(max(a.o.prefix[at], 0), d.len) : 0;
            d.lo = a.o.window > 0 ? max(0, d.len - a.o.window) : 0;
            d.kt = kt;
        };
        if constexpr (CLUSTER > 0) {
            if (begun) return false;
            begun = true;
            const int at = my_triple / triples;
            fill(at, my_triple - at * triples, decode_tiles(a, at));
            d.i0 = d.kt.n * rank / CC;            // (at most 2^20 pieces)
            d.i1 = d.kt.n * (rank + 1) / CC;
            return true;                          // also where its share is empty: it then adds nothing
        } else {
            while (u < u1 && row < a.rows) {
                const KeyTiles kt = decode_tiles(a, row);
                const int w = decode_units(kt.n);
                if (w == 0) { row++; continue; }
                const int64_t in_row = u - base;
                const int triple = (int)decode_div(in_row, w), v = (int)(in_row - (int64_t)triple * w), take = (int)min((int64_t)(w - v), u1 - u);
                u += take;
                const int at = row;
                if (u - base >= (int64_t)w * triples) { base += (int64_t)w * triples; row++; }
                d.i0 = max(v - DEC_START, 0);
                d.i1 = max(v + take - DEC_START, 0);
                if (d.i0 >= d.i1) continue;           // its start alone: the next CTA begins it
                fill(at, triple, kt);
                return true;
            }
            return false;
        }
    };

    // ---- loads: piece i of a part goes to stage (sb + i - i0) % NST of this warp's ring, where sb counts the pieces before ------
    // lanes 0-15 keep the page of their key of the next piece to be loaded, fetched one piece ahead
    DecSeg S, N;                                  // the part at work, and the one after
    int sb = 0;
    auto my_key = [&](const DecSeg& d, int i) {   // -1: not visible (its row is zeros)
        const int key = d.kt.tile(i) * DEC_TILE + warp * DEC_WK + lane;
        return i < d.i1 && lane < DEC_WK && key < d.len && (key < d.prefix || key >= d.lo) ? key : -1;
    };
    auto page_of = [&](const DecSeg& d, int i) {
        const int key = my_key(d, i);
        return key >= 0 ? a.c.table[(int64_t)d.row * a.c.table_stride + paged_entry(a.c, key)] : 0;
    };
    auto issue = [&](const DecSeg& d, int first, int i, int page) {
        if (i < d.i1) {
            const int key = my_key(d, i);
            const int64_t off = key >= 0 ? paged_offset(a.c, page, paged_row(a.c, key)) : -1;
            const uint16_t* kbase = a.c.k + d.kvh * a.c.head_stride;
            const uint16_t* vbase = a.c.v + d.kvh * a.c.head_stride;
            constexpr int CPR = D / 8;            // 16-byte chunks per row
            constexpr int RPI = 32 / CPR > 0 ? 32 / CPR : 1;   // rows per instruction
            const uint32_t st = ring + ((first + i - d.i0) % NST) * C::STAGE;
            const int c = lane % CPR;
#pragma unroll
            for (int r0 = 0; r0 < DEC_WK; r0 += RPI) {
                const int r = r0 + (RPI > 1 ? lane / CPR : 0);
                const int64_t o = __shfl_sync(0xffffffffu, off, r);
                const int64_t e = (o < 0 ? 0 : o) + c * 8;
                const int n = o < 0 ? 0 : 16;
                cp_async16_zfill(st + r * PITCH + c * 16, kbase + e, n);
                cp_async16_zfill(st + (DEC_WK + r) * PITCH + c * 16, vbase + e, n);
            }
        }
        paged_cp_commit();
    };
    int page = 0;
    auto begin = [&](const DecSeg& d, int first) {   // the first NST - 1 pieces
        page = page_of(d, d.i0);
#pragma unroll 1
        for (int s = 0; s < NST - 1; s++) {
            const int next = page_of(d, d.i0 + s + 1);
            issue(d, first, d.i0 + s, page);
            page = next;
        }
    };
    // queries of a part: this thread's chunks of 8 elements; f32 ones as three bf16 parts
    constexpr int NQ = (HB * (D / 8) + DEC_THREADS - 1) / DEC_THREADS;
    constexpr int QW = MODE == DEC_F32_8 ? 8 : 4; // words of a chunk
    auto load_queries = [&](const DecSeg& d, uint32_t (&x)[NQ][QW]) {
        const int h0 = d.kvh * a.G + d.bundle * HB, nh = min(HB, a.G - d.bundle * HB);
#pragma unroll
        for (int n = 0; n < NQ; n++) {
            const int i = tid + n * DEC_THREADS, h = i / (D / 8), c = i - h * (D / 8);
            const int64_t at = d.row * a.q_stride + (int64_t)(h0 + h) * D + c * 8;
#pragma unroll
            for (int v = 0; v < QW / 4; v++) {
                uint4 y = make_uint4(0, 0, 0, 0);
                if (h < nh) y = MODE == DEC_F32_8 ? *(const uint4*)((const float*)a.q + at + 4 * v) : *(const uint4*)((const uint16_t*)a.q + at);
                x[n][4 * v] = y.x; x[n][4 * v + 1] = y.y; x[n][4 * v + 2] = y.z; x[n][4 * v + 3] = y.w;
            }
        }
    };
    auto store_queries = [&](uint32_t (&x)[NQ][QW]) {
#pragma unroll
        for (int n = 0; n < NQ; n++) {
            const int i = tid + n * DEC_THREADS, h = i / (D / 8), c = i - h * (D / 8);
            if (h >= HB) break;
            unsigned char* dst = q_sm + h * PITCH + c * 16;
            if (MODE == DEC_F32_8) {
                float f[8];
#pragma unroll
                for (int e = 0; e < 8; e++) f[e] = __uint_as_float(x[n][e % QW]);
#pragma unroll
                for (int part = 0; part < 3; part++) {
                    uint32_t w[4];
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        w[e] = pack_bf16x2(f[2 * e], f[2 * e + 1]);
                        f[2 * e] -= __uint_as_float(w[e] << 16);
                        f[2 * e + 1] -= __uint_as_float(w[e] & 0xffff0000u);
                    }
                    *(uint4*)(dst + part * 8 * PITCH) = make_uint4(w[0], w[1], w[2], w[3]);
                }
            } else {
                *(uint4*)dst = make_uint4(x[n][0], x[n][1], x[n][2], x[n][3]);
            }
        }
    };

    // four columns from d of a finished query head
    auto store_out = [&](int at_row, int head, int d, float m, float l, const float (&x)[4]) {
        const float inv = l > 0.f ? 1.0f / l : 0.f;
        const int64_t at = at_row * a.out_stride + (int64_t)head * D + d;
        if (MODE == DEC_F32_8) *(float4*)((float*)a.out + at) = make_float4(x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv);
        else *(uint2*)((uint16_t*)a.out + at) = make_uint2(pack_bf16x2(x[0] * inv, x[1] * inv), pack_bf16x2(x[2] * inv, x[3] * inv));
        if (a.lse && d == 0) a.lse[(int64_t)at_row * a.Hq + head] = (m + log2f(l)) * 0.6931471805599453f;
    };

    // One round: the next part's first keys set out, the last part's warps meet in the stage they leave free and store it, then the next part
    // is worked through. (One copy of this code: it is long, and a short call waits for its instructions too.)
    float acc[ND][4], mrun[2], lrun[2];
    bool have = false;
    for (int sn = 0;; sn = (sb + S.i1 - S.i0) % NST, have = true) {
        const bool more = next_seg(N);
        if (more) begin(N, sn);
        const int red_at = (CLUSTER ? NST - 1 : (sn + NST - 1) % NST) * C::STAGE;   // (nothing comes after a cluster's part)
        if (have) {
            float* red = (float*)(dec_smem + warp * NST * C::STAGE + red_at);   // [HB][D]
#pragma unroll
            for (int r = 0; r < NR; r++) {
                float l = lrun[r];
                l += __shfl_xor_sync(0xffffffffu, l, 1);
                l += __shfl_xor_sync(0xffffffffu, l, 2);
                if (t == 0) { s_m[warp][g + 8 * r] = mrun[r]; s_l[warp][g + 8 * r] = l; }
            }
#pragma unroll
            for (int n = 0; n < ND; n++) {
                if (MODE == DEC_BF16_16) {
                    *(float2*)(red + g * D + n * 8 + 2 * t) = make_float2(acc[n][0], acc[n][1]);
                    *(float2*)(red + (g + 8) * D + n * 8 + 2 * t) = make_float2(acc[n][2], acc[n][3]);
                } else {
                    *(float2*)(red + g * D + n * 8 + 2 * t) = make_float2(acc[n][0] + acc[n][2], acc[n][1] + acc[n][3]);
                }
            }
            __syncthreads();
        }
        uint32_t qx[NQ][QW];
        if (more) load_queries(N, qx);
        if (have) {
            const int h0 = S.kvh * a.G + S.bundle * HB, nh = min(HB, a.G - S.bundle * HB);   // first query head, heads
            const bool whole = !CLUSTER && S.i1 - S.i0 == S.kt.n;
            float* mine = (float*)dec_smem;                   // CLUSTER: this CTA's part, in a stage nobody uses any more
            const int slot = 2 * blockIdx.x + (S.i0 > 0 ? 0 : 1);
            for (int idx = tid; idx < nh * (D / 4); idx += DEC_THREADS) {
                const int h = idx / (D / 4), d = (idx - h * (D / 4)) * 4;
                const float m = fmaxf(fmaxf(s_m[0][h], s_m[1][h]), fmaxf(s_m[2][h], s_m[3][h]));
                const float ref = m == -INFINITY ? 0.f : m;
                float l = 0.f, x[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int w = 0; w < DEC_WARPS; w++) {
                    const float e = ex2(s_m[w][h] - ref);
                    const float4 y = *(const float4*)((const float*)(dec_smem + w * NST * C::STAGE + red_at) + h * D + d);
                    l = fmaf(s_l[w][h], e, l);
                    x[0] = fmaf(y.x, e, x[0]); x[1] = fmaf(y.y, e, x[1]); x[2] = fmaf(y.z, e, x[2]); x[3] = fmaf(y.w, e, x[3]);
                }
                if (whole) {
                    store_out(S.row, h0 + h, d, m, l, x);
                } else if (CLUSTER) {
                    *(float4*)(mine + h * D + d) = make_float4(x[0], x[1], x[2], x[3]);
                    if (d == 0) s_part[h] = make_float2(m, l);
                } else {
                    *(float4*)(a.part + ((int64_t)slot * HB + h) * D + d) = make_float4(x[0], x[1], x[2], x[3]);
                    if (d == 0) a.ml[slot * HB + h] = make_float2(m, l);
                }
            }
        }
        if constexpr (CLUSTER > 0) if (have) {
            cluster_sync();                                   // all parts of the triple are there
            const int h0 = S.kvh * a.G + S.bundle * HB, nh = min(HB, a.G - S.bundle * HB);
            const uint32_t x_at = smem_u32(dec_smem), ml_at = smem_u32(s_part);
            for (int idx = rank * DEC_THREADS + tid; idx < nh * (D / 4); idx += CC * DEC_THREADS) {
                const int h = idx / (D / 4), d = (idx - h * (D / 4)) * 4;
                float2 ml[CC];
                float4 y[CC];
                float m = -INFINITY;
#pragma unroll
                for (int c = 0; c < CC; c++) {
                    ml[c] = cluster_ld2(cluster_map(ml_at + h * 8, c));
                    y[c] = cluster_ld4(cluster_map(x_at + (h * D + d) * 4, c));
                }
#pragma unroll
                for (int c = 0; c < CC; c++) m = fmaxf(m, ml[c].x);
                const float ref = m == -INFINITY ? 0.f : m;
                float l = 0.f, x[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int c = 0; c < CC; c++) {
                    const float e = ex2(ml[c].x - ref);
                    l = fmaf(ml[c].y, e, l);
                    x[0] = fmaf(y[c].x, e, x[0]); x[1] = fmaf(y[c].y, e, x[1]); x[2] = fmaf(y[c].z, e, x[2]); x[3] = fmaf(y[c].w, e, x[3]);
                }
                store_out(S.row, h0 + h, d, m, l, x);
            }
            cluster_sync();                                   // nobody reads this CTA's memory any more
        }
        if (!more) break;
        store_queries(qx);                                    // (all warps are through with the last part's)
        S = N;
        sb = sn;
        __syncthreads();                                      // the queries are there, the stage is free
        const int h0 = S.kvh * a.G + S.bundle * HB, nh = min(HB, a.G - S.bundle * HB);
        float slope[2] = {0.f, 0.f};
        if (a.o.slopes) {
            if (g < nh) slope[0] = a.o.slopes[h0 + g] * LOG2E;
            if (HB == 16 && g + 8 < nh) slope[1] = a.o.slopes[h0 + g + 8] * LOG2E;
        }
#pragma unroll
        for (int n = 0; n < ND; n++) acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.f;
        mrun[0] = mrun[1] = -INFINITY;
        lrun[0] = lrun[1] = 0.f;
        for (int i = S.i0; i < S.i1; i++) {
            const int next = page_of(S, i + NST);
            paged_cp_wait<NST - 2>();
            __syncwarp();                         // piece i has landed for every lane; nobody still reads the stage that is filled next
            issue(S, sb, i + NST - 1, page);
            page = next;
            const uint32_t kst = ring + ((sb + i - S.i0) % NST) * C::STAGE, vst = kst + DEC_WK * PITCH;
            const int mi = lane >> 3;
            // ---- scores: c[n][e], n-tile n = keys 8n.., e: row g (e < 2) or g + 8, key 2t + (e & 1) ----
            float c[2][4] = {}, c2[2][4] = {};
#pragma unroll
            for (int kk = 0; kk < KS; kk++) {
                uint32_t kb[4];
                ldmatrix_x4(kb, kst + ((mi >> 1) * 8 + (lane & 7)) * PITCH + kk * 32 + (mi & 1) * 16);
                uint32_t qa[4];
                if (MODE == DEC_BF16_8) {
                    // rows 0-7 only: the address lanes of the two upper matrices repeat the lower ones
                    ldmatrix_x4(qa, q_addr + (lane & 7) * PITCH + kk * 32 + (lane >> 4) * 16);
                    mma_bf16_16816(c[0], qa[0], 0u, qa[2], 0u, kb[0], kb[1]);
                    mma_bf16_16816(c[1], qa[0], 0u, qa[2], 0u, kb[2], kb[3]);
                } else {
                    ldmatrix_x4(qa, q_addr + (lane & 15) * PITCH + kk * 32 + (lane >> 4) * 16);
                    mma_bf16_16816(c[0], qa[0], qa[1], qa[2], qa[3], kb[0], kb[1]);
                    mma_bf16_16816(c[1], qa[0], qa[1], qa[2], qa[3], kb[2], kb[3]);
                }
                if (MODE == DEC_F32_8) {
                    ldmatrix_x4(qa, q_addr + (16 + (lane & 7)) * PITCH + kk * 32 + (lane >> 4) * 16);
                    mma_bf16_16816(c2[0], qa[0], 0u, qa[2], 0u, kb[0], kb[1]);
                    mma_bf16_16816(c2[1], qa[0], 0u, qa[2], 0u, kb[2], kb[3]);
                }
            }
            const int key0 = S.kt.tile(i) * DEC_TILE + warp * DEC_WK;
            constexpr int NR = MODE == DEC_BF16_16 ? 2 : 1;   // head rows of this thread
            float p[NR][4];                                   // [row][n-tile*2 + key]
            float mx[NR];
#pragma unroll
            for (int r = 0; r < NR; r++) {
                mx[r] = -INFINITY;
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int n = e >> 1, x = e & 1, key = key0 + n * 8 + 2 * t + x;
                    float s = c[n][2 * r + x];
                    if (MODE == DEC_F32_8) s += c[n][2 + x] + c2[n][x];
                    s = decode_score(s, s_in, s_cap, slope[r], S.len - 1 - key);
                    p[r][e] = key < S.len && (key < S.prefix || key >= S.lo) ? s : -INFINITY;
                    mx[r] = fmaxf(mx[r], p[r][e]);
                }
                mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 1));
                mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 2));
            }
            bool grew = false;
            float alpha[NR];
#pragma unroll
            for (int r = 0; r < NR; r++) {
                const float m = fmaxf(mrun[r], mx[r]);
                const float ref = m == -INFINITY ? 0.f : m;   // no visible key yet: keep ex2 finite
                alpha[r] = ex2(mrun[r] - ref);                // -inf -> 0
                grew |= m != mrun[r];
                mrun[r] = m;
                float sum = 0.f;
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    p[r][e] = ex2(p[r][e] - ref);
                    sum += p[r][e];
                }
                lrun[r] = lrun[r] * alpha[r] + sum;
            }
            if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
                for (int n = 0; n < ND; n++) {
                    acc[n][0] *= alpha[0]; acc[n][1] *= alpha[0];
                    acc[n][2] *= alpha[NR - 1]; acc[n][3] *= alpha[NR - 1];
                }
            }
            // ---- weights as MMA rows ----------------------------------------------------------------------
            uint32_t w0[2], w1[2], w2[2];                     // [n-tile]: rows 0-7, rows 8-15, the second MMA's rows 0-7
#pragma unroll
            for (int n = 0; n < 2; n++) {
                w0[n] = pack_bf16x2(p[0][2 * n], p[0][2 * n + 1]);
                w2[n] = 0u;
                if (MODE == DEC_BF16_16) {
                    w1[n] = pack_bf16x2(p[NR - 1][2 * n], p[NR - 1][2 * n + 1]);
                } else {
                    const float r0 = p[0][2 * n] - __uint_as_float(w0[n] << 16), r1 = p[0][2 * n + 1] - __uint_as_float(w0[n] & 0xffff0000u);
                    w1[n] = pack_bf16x2(r0, r1);
                    if (MODE == DEC_F32_8) w2[n] = pack_bf16x2(r0 - __uint_as_float(w1[n] << 16), r1 - __uint_as_float(w1[n] & 0xffff0000u));
                }
            }
#pragma unroll
            for (int d2 = 0; d2 < D / 16; d2++) {
                uint32_t vb[4];
                ldmatrix_x4_trans(vb, vst + ((mi & 1) * 8 + (lane & 7)) * PITCH + d2 * 32 + (mi >> 1) * 16);
                mma_bf16_16816(acc[2 * d2], w0[0], w1[0], w0[1], w1[1], vb[0], vb[1]);
                mma_bf16_16816(acc[2 * d2 + 1], w0[0], w1[0], w0[1], w1[1], vb[2], vb[3]);
                if (MODE == DEC_F32_8) {
                    mma_bf16_16816(acc[2 * d2], w2[0], 0u, w2[1], 0u, vb[0], vb[1]);
                    mma_bf16_16816(acc[2 * d2 + 1], w2[0], 0u, w2[1], 0u, vb[2], vb[3]);
                }
            }
            __syncwarp();                                     // the stage may be refilled
        }
    }
    paged_cp_wait<0>();
}

// Joins the parts of triples that several CTAs hold, and writes the rows that see nothing. One CTA per (row, query head); warp w
// takes parts w, w+4, ... with a running maximum, four loads in flight. Which CTAs those are follows from the lengths, which
// do not have to be waited for.
template <int D>
__global__ void __launch_bounds__(128) paged_decode_join_kernel(const DecodeArgs a, int HB, int out_f32) {
    constexpr int DL = D / 32;
    __shared__ float sm[4], sl[4];
    __shared__ float so[4][D];
    __shared__ int s_scan[4];
    __shared__ int s_base;
    const int row = blockIdx.y, qh = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    float* of = (float*)a.out + row * a.out_stride + (int64_t)qh * D;
    uint16_t* ob = (uint16_t*)a.out + row * a.out_stride + (int64_t)qh * D;
    const int n = decode_tiles(a, row).n;
    int64_t base = 0, U = 0;
    if (a.rows <= 128) {
        int incl;
        const int mine = tid < a.rows ? decode_units(decode_tiles(a, tid).n) : 0;
        U = paged_block_scan<4>(mine, incl, s_scan);
        if (tid == row) s_base = incl - mine;
        __syncthreads();
        base = s_base;
        pdl_wait();
    } else {
        pdl_wait();
        base = a.base[row];
        U = a.base[a.rows];
    }
    if (n == 0) {
        for (int d = tid; d < D; d += 128) {
            if (out_f32) of[d] = 0.f;
            else ob[d] = 0;
        }
        if (a.lse && tid == 0) a.lse[(int64_t)row * a.Hq + qh] = -INFINITY;
        return;
    }
    const int triples = a.c.kv_heads * a.nb;
    U *= triples;
    const int ctas = (int)min((int64_t)a.ctas, U);
    const int kvh = qh / a.G, in = qh - kvh * a.G, bundle = in / HB, h = in - bundle * HB;
    base = base * triples + (int64_t)(kvh * a.nb + bundle) * decode_units(n) + DEC_START;   // the first piece
    const int first = decode_cta_of(base, U, ctas), last = decode_cta_of(base + n - 1, U, ctas);
    if (first == last) return;
    float m = -INFINITY, l = 0.f, acc[DL];
#pragma unroll
    for (int i = 0; i < DL; i++) acc[i] = 0.f;
    constexpr int B = 4;
    for (int c0 = first + warp; c0 <= last; c0 += 4 * B) {
        float2 ml[B];
        float2 x[B][DL / 2];
#pragma unroll
        for (int b = 0; b < B; b++) {
            const int c = c0 + 4 * b;
            const bool live = c <= last;
            const int64_t at = (int64_t)(2 * (live ? c : c0) + ((live ? c : c0) == first ? 1 : 0)) * HB + h;
            ml[b] = live ? a.ml[at] : make_float2(-INFINITY, 0.f);
#pragma unroll
            for (int i = 0; i < DL / 2; i++) x[b][i] = ((const float2*)(a.part + at * D))[lane + 32 * i];
        }
        float nm = m;
#pragma unroll
        for (int b = 0; b < B; b++) nm = fmaxf(nm, ml[b].x);
        if (nm == -INFINITY) continue;
        const float e0 = ex2(m - nm);
        l *= e0;
#pragma unroll
        for (int i = 0; i < DL; i++) acc[i] *= e0;
#pragma unroll
        for (int b = 0; b < B; b++) {
            const float e = ex2(ml[b].x - nm);
            l = fmaf(ml[b].y, e, l);
#pragma unroll
            for (int i = 0; i < DL / 2; i++) {
                acc[2 * i] = fmaf(x[b][i].x, e, acc[2 * i]);
                acc[2 * i + 1] = fmaf(x[b][i].y, e, acc[2 * i + 1]);
            }
        }
        m = nm;
    }
    if (lane == 0) { sm[warp] = m; sl[warp] = l; }
#pragma unroll
    for (int i = 0; i < DL / 2; i++) *(float2*)&so[warp][2 * (lane + 32 * i)] = make_float2(acc[2 * i], acc[2 * i + 1]);
    __syncthreads();
    const float gm = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
    const float ref = gm == -INFINITY ? 0.f : gm;
    float e[4], den = 0.f;
#pragma unroll
    for (int w = 0; w < 4; w++) { e[w] = ex2(sm[w] - ref); den = fmaf(sl[w], e[w], den); }
    const float inv = den > 0.f ? 1.0f / den : 0.f;
    for (int d = tid; d < D; d += 128) {
        const float o = (so[0][d] * e[0] + so[1][d] * e[1] + so[2][d] * e[2] + so[3][d] * e[3]) * inv;
        if (out_f32) of[d] = o;
        else ob[d] = f32_to_bf16_bits(o);
    }
    if (a.lse && tid == 0) a.lse[(int64_t)row * a.Hq + qh] = (gm + log2f(den)) * 0.6931471805599453f;
}

// Bundles of heads: f32 always 8 (three bf16 parts of q and of the weights fill the MMA rows), bf16 8 where that
// holds the whole group and 16 otherwise (twice the heads per pass over the keys).
static int decode_mode(int dtype, int G) { return dtype == LTHN_DTYPE_F32 ? DEC_F32_8 : G <= 8 ? DEC_BF16_8 : DEC_BF16_16; }
static int decode_bundle(int mode) { return mode == DEC_BF16_16 ? 16 : 8; }

struct DecodePlan { int mode, HB, nb, ctas; size_t part, ml, base, total; };
// capacity: the most keys a row can have
static DecodePlan decode_plan(int D, int kv_heads, int rows, int q_heads, int dtype, int capacity) {
    DecodePlan p;
    const int G = q_heads / kv_heads;
    p.mode = decode_mode(dtype, G);
    p.HB = decode_bundle(p.mode);
    p.nb = (G + p.HB - 1) / p.HB;
    // as many as run at once; a short table has fewer units than that
    const int64_t most = (int64_t)rows * kv_heads * p.nb * (((int64_t)capacity + DEC_TILE - 1) / DEC_TILE + DEC_START);
    p.ctas = (int)std::max<int64_t>(1, std::min<int64_t>(paged_sm_count() * (D == 256 ? 1 : 2), most));
    auto up = [](size_t b) { return (b + 255) & ~(size_t)255; };
    p.part = up((size_t)2 * p.ctas * p.HB * D * 4);
    p.ml = up((size_t)2 * p.ctas * p.HB * 8);
    p.base = up((size_t)(rows + 1) * 8);
    p.total = p.part + p.ml + p.base;
    return p;
}

// How many clusters of such CTAs (CLUSTER = 0: unknown) a device runs at once; the kernel is made ready on the way.
template <int D, int MODE, int CLUSTER>
static int32_t decode_ready(int* at_once) {
    using C = DecCfg<D, MODE>;
    static uint32_t known_devs = 0;
    static int known[32];
    static std::mutex mu;
    int dev = 0;
    LTHN_CUDA_TRY(cudaGetDevice(&dev));
    dev &= 31;
    std::lock_guard<std::mutex> lk(mu);
    if (known_devs >> dev & 1) {
        *at_once = known[dev];
        return LTHN_OK;
    }
    LTHN_CUDA_TRY(cudaFuncSetAttribute(paged_decode_kernel<D, MODE, CLUSTER>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)C::SMEM));
    int n = 0;
    if (CLUSTER > 0) {
        if (CLUSTER > 8) LTHN_CUDA_TRY(cudaFuncSetAttribute(paged_decode_kernel<D, MODE, CLUSTER>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
        cudaLaunchConfig_t cfg = {};
        cudaLaunchAttribute at[1];
        at[0].id = cudaLaunchAttributeClusterDimension;
        at[0].val.clusterDim = {CLUSTER, 1, 1};
        cfg.gridDim = dim3(CLUSTER); cfg.blockDim = dim3(DEC_THREADS); cfg.dynamicSmemBytes = C::SMEM; cfg.attrs = at; cfg.numAttrs = 1;
        LTHN_CUDA_TRY(cudaOccupancyMaxActiveClusters(&n, paged_decode_kernel<D, MODE, CLUSTER>, &cfg));
    }
    known_devs |= 1u << dev;
    *at_once = known[dev] = n;
    return LTHN_OK;
}

template <int D, int MODE, int CLUSTER>
static int32_t launch_decode_kernel(cudaStream_t s, const DecodeArgs& a) {
    using C = DecCfg<D, MODE>;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute at[1];
    cfg.attrs = at; cfg.numAttrs = 1; cfg.stream = s;
    if (CLUSTER > 0) {
        cfg.gridDim = dim3(a.rows * a.c.kv_heads * a.nb * CLUSTER); cfg.blockDim = dim3(DEC_THREADS); cfg.dynamicSmemBytes = C::SMEM;
        at[0].id = cudaLaunchAttributeClusterDimension;
        at[0].val.clusterDim = {CLUSTER, 1, 1};
        LTHN_CUDA_TRY(cudaLaunchKernelEx(&cfg, paged_decode_kernel<D, MODE, CLUSTER>, a));
        return LTHN_OK;
    }
    paged_decode_kernel<D, MODE, CLUSTER><<<a.ctas, DEC_THREADS, C::SMEM, s>>>(a);
    LTHN_CUDA_TRY(cudaGetLastError());
    cfg.gridDim = dim3(a.Hq, a.rows); cfg.blockDim = dim3(128);
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    LTHN_CUDA_TRY(cudaLaunchKernelEx(&cfg, paged_decode_join_kernel<D>, a, C::HB, MODE == DEC_F32_8 ? 1 : 0));
    return LTHN_OK;
}
// The size of the clusters that a call's triples go to, 0: the list. A cluster per triple, in one launch, where all clusters run at once and
// the longest row that a call can have gives a CTA no more than 512 / D pieces more than an even share over the whole GPU would: that
// many take as long as the join (8 triples, head_dim 128, bf16: 512 keys 7.0 us in even shares, 4.6 in clusters of 8; 2048 keys 8.6, 7.9; 4096
// keys 10.9, 11.5). For up to 4 triples with more than a piece for each of 8 CTAs the clusters have 16 (4 triples, head_dim 256, f32: 512
// keys 8.9 us, of 8 6.5, of 16 7.1; 1280 keys 10.8, 10.3, 8.9; 2048 keys 10.7, 12.3, 8.8; 8 triples, head_dim 128, 1280 keys: 8.7, 6.7, 7.4).
// "Can have" is by the table and the window, not by the lengths, which the host does not know: 4 triples of head_dim 256 take the list under tables of
// more than about 3600 rows, 8 of head_dim 128 from about 2600 on, however short their sequences are.
template <int D>
static int decode_cluster(const DecodeArgs& a) {
    const int64_t triples = (int64_t)a.rows * a.c.kv_heads * a.nb;
    if (triples > 16) return 0;
    int64_t pieces = ((int64_t)a.c.capacity + DEC_TILE - 1) / DEC_TILE;
    if (a.o.window > 0 && !a.o.prefix) pieces = std::min<int64_t>(pieces, a.o.window / DEC_TILE + 2);
    const int size = triples <= 4 && pieces > 8 ? 16 : 8;
    return pieces * (1.0 / size - (double)triples / a.ctas) * D <= 512.0 ? size : 0;
}
template <int D, int MODE>
static int32_t launch_decode_form(cudaStream_t s, const DecodeArgs& a) {
    const int triples = (int)std::min<int64_t>((int64_t)a.rows * a.c.kv_heads * a.nb, 1 << 30), size = decode_cluster<D>(a);
    int32_t rc;
    int at_once = 0;
    if (size == 16) {
        if ((rc = decode_ready<D, MODE, 16>(&at_once))) return rc;
        if (at_once >= triples) return launch_decode_kernel<D, MODE, 16>(s, a);
    } else if (size == 8) {
        if ((rc = decode_ready<D, MODE, 8>(&at_once))) return rc;
        if (at_once >= triples) return launch_decode_kernel<D, MODE, 8>(s, a);
    }
    if ((rc = decode_ready<D, MODE, 0>(&at_once))) return rc;
    return launch_decode_kernel<D, MODE, 0>(s, a);
}
template <int D>
static int32_t launch_decode_mode(cudaStream_t s, const DecodeArgs& a, int mode) {
    if (mode == DEC_BF16_16) return launch_decode_form<D, DEC_BF16_16>(s, a);
    if (mode == DEC_BF16_8) return launch_decode_form<D, DEC_BF16_8>(s, a);
    return launch_decode_form<D, DEC_F32_8>(s, a);
}

}  // namespace lthn

using namespace lthn;

static int32_t decode_check(const lthn_paged_kv* cache, int32_t rows, int32_t q_heads, int32_t dtype, PagedCache* c) {
    int32_t rc;
    if ((rc = paged_check_cache("paged_sdpa_decode", cache, c))) return rc;
    LTHN_REQUIRE(dtype == LTHN_DTYPE_F32 || dtype == LTHN_DTYPE_BF16, "paged_sdpa_decode: dtype must be f32 or bf16");
    LTHN_REQUIRE(rows >= 0 && rows <= 65535, "paged_sdpa_decode: rows must be in [0, 65535]");
    LTHN_REQUIRE(rows <= cache->seqs, "paged_sdpa_decode: more rows than the page table has sequences");
    LTHN_REQUIRE(q_heads > 0 && q_heads <= 65535 && q_heads % cache->kv_heads == 0, "paged_sdpa_decode: q_heads must be a positive multiple of kv_heads");
    return LTHN_OK;
}

extern "C" {

int32_t lthn_paged_sdpa_decode_workspace(const lthn_paged_kv* cache, int32_t rows, int32_t q_heads, int32_t dtype, size_t* bytes) {
    clear_error();
    LTHN_REQUIRE(bytes != nullptr, "paged_sdpa_decode_workspace: bytes is NULL");
    PagedCache c;
    int32_t rc;
    if ((rc = decode_check(cache, rows, q_heads, dtype, &c))) return rc;
    *bytes = decode_plan(cache->head_dim, cache->kv_heads, rows, q_heads, dtype, c.capacity).total;
    return LTHN_OK;
}

int32_t lthn_paged_sdpa_decode(void* stream, const lthn_paged_kv* cache, const lthn_attn_options* options, const void* q, int32_t dtype,
                               int64_t q_stride, const int32_t* kv_lens, int32_t rows, int32_t q_heads, void* out, int64_t out_stride,
                               float* lse, void* workspace, size_t workspace_bytes) {
    clear_error();
    const char* me = "paged_sdpa_decode";
    DecodeArgs a = {};
    int32_t rc;
    if ((rc = decode_check(cache, rows, q_heads, dtype, &a.c))) return rc;
    const int D = cache->head_dim;
    if ((rc = paged_check_options(me, options, D, &a.o))) return rc;
    if (rows == 0) return LTHN_OK;
    LTHN_REQUIRE(q && out && kv_lens && workspace, "paged_sdpa_decode: NULL pointer");
    a.q_stride = q_stride ? q_stride : (int64_t)q_heads * D;
    a.out_stride = out_stride ? out_stride : (int64_t)q_heads * D;
    LTHN_REQUIRE(((a.q_stride | a.out_stride) & 7) == 0, "paged_sdpa_decode: strides must be multiples of 8 elements");
    LTHN_REQUIRE(a.out_stride >= (int64_t)q_heads * D, "paged_sdpa_decode: rows of out would overlap");
    LTHN_REQUIRE((((uintptr_t)q | (uintptr_t)out | (uintptr_t)workspace) & 15) == 0, "paged_sdpa_decode: q, out and workspace must be 16-byte aligned");
    const DecodePlan p = decode_plan(D, cache->kv_heads, rows, q_heads, dtype, a.c.capacity);
    LTHN_REQUIRE(workspace_bytes >= p.total, "paged_sdpa_decode: workspace too small");
    if ((rc = paged_check_pointers(me, {{"the cache's k", cache->k, 16, false}, {"the cache's v", cache->v, 16, false},
                                        {"page_table", cache->page_table, 4, true}, {"q", q, 16, true}, {"kv_lens", kv_lens, 4, true}, {"out", out, 16, true},
                                        {"lse", lse, 4, true}, {"workspace", workspace, 16, false}, {"slopes", a.o.slopes, 4, true},
                                        {"prefix_lens", a.o.prefix, 4, true}})))
        return rc;
    a.q = q; a.out = out; a.lens = kv_lens; a.lse = lse; a.rows = rows; a.Hq = q_heads; a.G = q_heads / cache->kv_heads;
    a.nb = p.nb; a.ctas = p.ctas;
    a.part = (float*)workspace;
    a.ml = (float2*)((char*)workspace + p.part);
    a.base = (int64_t*)((char*)workspace + p.part + p.ml);
    a.c.status = device_paged_status_word();
    if (!a.c.status) return fail(LTHN_ERR_CUDA, "paged_sdpa_decode: no device status word");
    if (D == 64) return launch_decode_mode<64>((cudaStream_t)stream, a, p.mode);
    if (D == 128) return launch_decode_mode<128>((cudaStream_t)stream, a, p.mode);
    return launch_decode_mode<256>((cudaStream_t)stream, a, p.mode);
}

}  // extern "C"
