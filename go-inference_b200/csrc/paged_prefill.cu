// paged_prefill.cu — attention of packed prompt chunks over the paged KV cache.
//
//   out = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m),   s_j = cap(q.k_j scale) - slope |i - j|,   m = max_j s_j
//
// The query rows of a tile are the (token, query head) pairs of one kv head, token by token, so the heads that share
// K and V share their loads, and a chunk of a few tokens still fills a tile. One CTA = 64 rows, four warps of 16; K and V
// tiles by cp.async, double buffered; both products on mma.sync with a running softmax.
#include "paged.cuh"

#include <algorithm>
#include <mutex>

namespace lthn {

struct PrefillArgs {
    PagedCache c;
    AttnOpts o;
    const uint16_t* q;
    uint16_t* out;
    int64_t q_stride, out_stride;
    const int32_t *q_start, *lens;
    float* lse;
    int seqs, total_q, Hq, G;
};

// The rows of sequence s, made safe: within [0, total_q), never overlapping the next one's.
__device__ __forceinline__ int2 prefill_span(const PrefillArgs& a, int s) {
    const int b = a.q_start[s], e = a.q_start[s + 1];
    if (b < 0 || e < b || e > a.total_q) {
        atomicOr(a.c.status, LTHN_STATUS_PAGED);
        return make_int2(0, 0);
    }
    return make_int2(b, e - b);
}

// Tile blockIdx.x counts through the tiles (of ROWS rows of token * G + head) of all sequences. Returns false past the last.
template <int WARPS, int ROWS>
__device__ __forceinline__ bool prefill_tile(const PrefillArgs& a, int* sh, int& seq, int& tile) {
    int base = 0;
    for (int s0 = 0; s0 < a.seqs; s0 += WARPS * 32) {
        const int s = s0 + threadIdx.x;
        const int n = s < a.seqs ? (prefill_span(a, s).y * a.G + ROWS - 1) / ROWS : 0;
        int incl;
        const int total = paged_block_scan<WARPS>(n, incl, sh);
        const int want = (int)blockIdx.x - base;
        if (want < total) {
            if (incl > want && incl - n <= want) { sh[WARPS] = s; sh[WARPS + 1] = want - (incl - n); }
            __syncthreads();
            seq = sh[WARPS];
            tile = sh[WARPS + 1];
            return true;
        }
        base += total;
    }
    return false;
}

constexpr int PP_BM = 64;
constexpr int PP_WARPS = 4;
constexpr int PP_THREADS = PP_WARPS * 32;

template <int D>
struct PpCfg {
    static constexpr int BN = D >= 256 ? 32 : 64;
    static constexpr int PITCH = D * 2 + 16;
    static constexpr size_t SMEM = (size_t)(PP_BM + 4 * BN) * PITCH;
};

template <int D>
__global__ void __launch_bounds__(PP_THREADS) paged_prefill_kernel(const PrefillArgs a) {
    using C = PpCfg<D>;
    constexpr int BN = C::BN, PITCH = C::PITCH, NS = BN / 8, ND = D / 8, CPR = D / 8;
    constexpr float LOG2E = 1.4426950408889634f;
    extern __shared__ __align__(16) unsigned char pp_smem[];
    __shared__ int sh[PP_WARPS + 2];
    int seq, tile;
    if (!prefill_tile<PP_WARPS, PP_BM>(a, sh, seq, tile)) return;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3, mi = lane >> 3;
    const int kvh = blockIdx.y;
    const int2 span = prefill_span(a, seq);
    const int len = paged_length(a.c, a.lens[seq]);
    const int nrows = span.y * a.G, row0 = tile * PP_BM;
    const int pos0 = len - span.y;                                   // position of the sequence's first query
    const int prefix = a.o.prefix ? min(max(a.o.prefix[seq], 0), len) : 0;
    const int qlo = pos0 + row0 / a.G, qhi = pos0 + (min(row0 + PP_BM, nrows) - 1) / a.G;
    const KeyTiles kt = key_tiles<BN>(qlo, qhi, len, prefix, a.o.window);
    const int lo = a.o.window > 0 ? max(0, qlo - a.o.window + 1) : 0;
    const uint16_t* kbase = a.c.k + kvh * a.c.head_stride;
    const uint16_t* vbase = a.c.v + kvh * a.c.head_stride;
    const int32_t* trow = a.c.table + (int64_t)seq * a.c.table_stride;
    const uint32_t qs = smem_u32(pp_smem), ks = qs + PP_BM * PITCH, vs = ks + 2 * BN * PITCH;

    auto load_kv = [&](int i) {
        const int k0 = kt.tile(i) * BN, buf = i & 1;
        for (int x = tid; x < BN * CPR; x += PP_THREADS) {
            const int r = x / CPR, c = x - r * CPR, key = k0 + r;
            int64_t off = -1;
            if (key < len && (key < prefix || key >= lo)) off = paged_offset(a.c, trow[key / a.c.page_size], key % a.c.page_size);
            const int64_t e = (off < 0 ? 0 : off) + c * 8;
            const int n = off < 0 ? 0 : 16;
            cp_async16_zfill(ks + (buf * BN + r) * PITCH + c * 16, kbase + e, n);
            cp_async16_zfill(vs + (buf * BN + r) * PITCH + c * 16, vbase + e, n);
        }
        paged_cp_commit();
    };
    for (int x = tid; x < PP_BM * CPR; x += PP_THREADS) {
        const int r = x / CPR, c = x - r * CPR, row = row0 + r;
        uint4 v = make_uint4(0, 0, 0, 0);
        if (row < nrows) v = *(const uint4*)(a.q + (span.x + row / a.G) * a.q_stride + (int64_t)(kvh * a.G + row % a.G) * D + c * 8);
        *(uint4*)(pp_smem + r * PITCH + c * 16) = v;
    }
    if (kt.n > 0) load_kv(0);
    float o[ND][4];
#pragma unroll
    for (int n = 0; n < ND; n++) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
    float mrow[2] = {-INFINITY, -INFINITY}, lrow[2] = {0.f, 0.f}, slope[2] = {0.f, 0.f};
    int qpos[2];
#pragma unroll
    for (int h = 0; h < 2; h++) {
        const int row = row0 + warp * 16 + g + 8 * h;
        qpos[h] = pos0 + row / a.G;
        if (a.o.slopes && row < nrows) slope[h] = a.o.slopes[kvh * a.G + row % a.G];
    }
    for (int i = 0; i < kt.n; i++) {
        const int buf = i & 1, k0 = kt.tile(i) * BN;
        paged_cp_wait<0>();
        __syncthreads();
        if (i + 1 < kt.n) load_kv(i + 1);
        float s[NS][4];
#pragma unroll
        for (int n = 0; n < NS; n++) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
#pragma unroll
        for (int kk = 0; kk < D / 16; kk++) {
            uint32_t qa[4];
            ldmatrix_x4(qa, qs + (warp * 16 + (lane & 15)) * PITCH + kk * 32 + (lane >> 4) * 16);
#pragma unroll
            for (int n2 = 0; n2 < BN / 16; n2++) {
                uint32_t kb[4];
                ldmatrix_x4(kb, ks + (buf * BN + n2 * 16 + (mi >> 1) * 8 + (lane & 7)) * PITCH + kk * 32 + (mi & 1) * 16);
                mma_bf16_16816(s[2 * n2], qa[0], qa[1], qa[2], qa[3], kb[0], kb[1]);
                mma_bf16_16816(s[2 * n2 + 1], qa[0], qa[1], qa[2], qa[3], kb[2], kb[3]);
            }
        }
        float mx[2] = {mrow[0], mrow[1]};
#pragma unroll
        for (int n = 0; n < NS; n++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int key = k0 + n * 8 + 2 * t + (e & 1), gap = qpos[e >> 1] - key;
                float v = s[n][e] * a.o.scale;
                if (a.o.softcap > 0.f) v = a.o.softcap * tanhf(v / a.o.softcap);
                if (a.o.slopes) v -= slope[e >> 1] * (float)abs(gap);
                const bool seen = key < len && (key < prefix || (gap >= 0 && (a.o.window == 0 || gap < a.o.window)));
                s[n][e] = seen ? v * LOG2E : -INFINITY;
                mx[e >> 1] = fmaxf(mx[e >> 1], s[n][e]);
            }
        float alpha[2];
#pragma unroll
        for (int h = 0; h < 2; h++) {
            mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 1));
            mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 2));
            const float ref = mx[h] == -INFINITY ? 0.f : mx[h];
            alpha[h] = ex2(mrow[h] - ref);
            mrow[h] = mx[h];
            mx[h] = ref;
            lrow[h] *= alpha[h];
        }
        uint32_t p[NS][2];
#pragma unroll
        for (int n = 0; n < NS; n++) {
            const float p0 = ex2(s[n][0] - mx[0]), p1 = ex2(s[n][1] - mx[0]), p2 = ex2(s[n][2] - mx[1]), p3 = ex2(s[n][3] - mx[1]);
            lrow[0] += p0 + p1;
            lrow[1] += p2 + p3;
            p[n][0] = pack_bf16x2(p0, p1);
            p[n][1] = pack_bf16x2(p2, p3);
        }
#pragma unroll
        for (int n = 0; n < ND; n++) { o[n][0] *= alpha[0]; o[n][1] *= alpha[0]; o[n][2] *= alpha[1]; o[n][3] *= alpha[1]; }
#pragma unroll
        for (int k16 = 0; k16 < BN / 16; k16++)
#pragma unroll
            for (int d2 = 0; d2 < D / 16; d2++) {
                uint32_t vb[4];
                ldmatrix_x4_trans(vb, vs + (buf * BN + k16 * 16 + (mi & 1) * 8 + (lane & 7)) * PITCH + d2 * 32 + (mi >> 1) * 16);
                mma_bf16_16816(o[2 * d2], p[2 * k16][0], p[2 * k16][1], p[2 * k16 + 1][0], p[2 * k16 + 1][1], vb[0], vb[1]);
                mma_bf16_16816(o[2 * d2 + 1], p[2 * k16][0], p[2 * k16][1], p[2 * k16 + 1][0], p[2 * k16 + 1][1], vb[2], vb[3]);
            }
    }
#pragma unroll
    for (int h = 0; h < 2; h++) {
        float l = lrow[h];
        l += __shfl_xor_sync(0xffffffffu, l, 1);
        l += __shfl_xor_sync(0xffffffffu, l, 2);
        const int row = row0 + warp * 16 + g + 8 * h;
        if (row >= nrows) continue;
        const float inv = l > 0.f ? 1.0f / l : 0.f;
        const int64_t token = span.x + row / a.G;
        const int head = kvh * a.G + row % a.G;
        uint16_t* dst = a.out + token * a.out_stride + (int64_t)head * D + 2 * t;
#pragma unroll
        for (int n = 0; n < ND; n++) *(uint32_t*)(dst + n * 8) = pack_bf16x2(o[n][2 * h] * inv, o[n][2 * h + 1] * inv);
        if (a.lse && t == 0) a.lse[token * a.Hq + head] = (mrow[h] + log2f(l)) * 0.6931471805599453f;
    }
}

template <int D>
static int32_t launch_prefill(cudaStream_t s, const PrefillArgs& a) {
    static uint32_t attr_devs = 0;
    static std::mutex mu;
    int dev = 0;
    LTHN_CUDA_TRY(cudaGetDevice(&dev));
    {
        std::lock_guard<std::mutex> lk(mu);
        if (!(attr_devs >> (dev & 31) & 1)) {
            LTHN_CUDA_TRY(cudaFuncSetAttribute(paged_prefill_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)PpCfg<D>::SMEM));
            attr_devs |= 1u << (dev & 31);
        }
    }
    // at most this many tiles: each sequence may end in a tile of its own
    const int64_t tiles = (int64_t)a.total_q * a.G / PP_BM + a.seqs;
    paged_prefill_kernel<D><<<dim3((unsigned)tiles, a.c.kv_heads), PP_THREADS, PpCfg<D>::SMEM, s>>>(a);
    LTHN_CUDA_TRY(cudaGetLastError());
    return LTHN_OK;
}

}  // namespace lthn

using namespace lthn;

static int32_t prefill_check(const lthn_paged_kv* cache, int32_t seqs, int32_t total_q, int32_t q_heads, int32_t max_ctx, PagedCache* c) {
    int32_t rc;
    if ((rc = paged_check_cache("paged_prefill_attention", cache, c))) return rc;
    LTHN_REQUIRE(seqs >= 0 && total_q >= 0 && max_ctx >= 0, "paged_prefill_attention: negative size");
    LTHN_REQUIRE(seqs <= cache->seqs, "paged_prefill_attention: more sequences than the page table has");
    LTHN_REQUIRE(q_heads > 0 && q_heads <= 65535 && q_heads % cache->kv_heads == 0, "paged_prefill_attention: q_heads must be a positive multiple of kv_heads");
    LTHN_REQUIRE((int64_t)total_q * (q_heads / cache->kv_heads) + (int64_t)seqs * 256 < (int64_t)1 << 31, "paged_prefill_attention: too many query rows");
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
    *bytes = 16;
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
    LTHN_REQUIRE(a.out_stride >= (int64_t)q_heads * D, "paged_prefill_attention: rows of out would overlap");
    LTHN_REQUIRE((((uintptr_t)q | (uintptr_t)out | (uintptr_t)workspace) & 15) == 0, "paged_prefill_attention: q, out and workspace must be 16-byte aligned");
    LTHN_REQUIRE(workspace_bytes >= 16, "paged_prefill_attention: workspace too small");
    if ((rc = paged_check_device(me, "the cache", cache->k))) return rc;
    if ((rc = paged_check_device(me, "q", q))) return rc;
    a.q = q; a.out = out; a.q_start = q_start; a.lens = kv_lens; a.lse = lse;
    a.seqs = seqs; a.total_q = total_q; a.Hq = q_heads; a.G = q_heads / cache->kv_heads;
    a.c.status = device_paged_status_word();
    if (!a.c.status) return fail(LTHN_ERR_CUDA, "paged_prefill_attention: no device status word");
    if (D == 64) return launch_prefill<64>((cudaStream_t)stream, a);
    if (D == 128) return launch_prefill<128>((cudaStream_t)stream, a);
    return launch_prefill<256>((cudaStream_t)stream, a);
}

}  // extern "C"
