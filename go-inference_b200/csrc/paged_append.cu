// paged_append.cu — appending rows to the paged KV cache with the per-head norm and the rotation on the way, and the
// argument checks the paged entry points share.
//
//   q, k head x of position pos:  x <- x / sqrt(mean(x^2) + eps) * w            (optional)
//                                 (a, b) <- (a cos t - b sin t, a sin t + b cos t), t = pos * inv_freq[i]
//   k, v -> bf16 row of the page, q -> q_out
//
// Every element is read once and written once, so the kernel is bound by memory. A head is D/8 threads: thread j holds
// elements 4j..4j+3 of either half of the head, which makes both kinds of pairs, (i, i + D/2) and (2i, 2i+1), meet in one
// thread; the norm needs one shuffle reduction over the head's threads and nothing else crosses threads. One CTA is
// one token row: its D/2 angles are formed once, by one thread each, and read by all of the row's heads. Position, page,
// angles and norm are a chain of latencies, so what counts is how many rows an SM has at work: the first heads are loaded before
// position and page are known, and CTAs are small (8190 rows of 64 heads of 128, bf16, 268 MB: 64 us with 4 CTAs of 256 threads per SM,
// 53.5 us = 5.0 TB/s with 10 of 128, which leaves 48 registers and spills 8 bytes, 24 to 32 with f32 queries out; fetching the next row under this one instead: 67 us; 8 elements a
// thread and half the threads: 60 us). For a few rows the chain is all
// there is, and a row's heads are shared between CTAs (1 row of 16 heads of 256, f32: 3.9 us, shared 3.4; 64 rows of 48 heads
// of 128, bf16: 3.3, 2.6). The angle is the only place
// where 32 bits are not enough (position 200000 leaves an f32 angle 0.01 off), so it is formed in f64, in turns, reduced
// there to [-1/2, 1/2], and handed to sincospif.
#include "paged.cuh"

#include <cuda.h>

#include <algorithm>

namespace lthn {

static std::string named(const char* name, const char* what) { return std::string(name) + ": " + what; }

int paged_sm_count() {
    int dev = 0, sms = 148;
    if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    return sms;
}

typedef CUresult (*PointerAttributes)(unsigned, CUpointer_attribute*, void**, CUdeviceptr);
static PointerAttributes pointer_attributes() {
    static PointerAttributes fn = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        return cudaGetDriverEntryPoint("cuPointerGetAttributes", &p, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess
                   ? (PointerAttributes)p : nullptr;
    }();
    return fn;
}

int32_t paged_check_pointers(const char* name, std::initializer_list<PagedPtr> list) {
    for (const PagedPtr& x : list)
        if ((uintptr_t)x.p & (x.align - 1)) return fail(LTHN_ERR_INVALID, named(name, x.what) + " must be " + std::to_string(x.align) + "-byte aligned");
    int dev = 0;
    LTHN_CUDA_TRY(cudaGetDevice(&dev));
    if (!pointer_attributes()) return fail(LTHN_ERR_CUDA, named(name, "the driver has no pointer queries"));
    // A query takes about 45 ns of the host; arguments within an allocation that has been looked up are not asked for again.
    uintptr_t begin[4] = {}, end[4] = {};
    int known = 0;
    for (const PagedPtr& x : list) {
        const uintptr_t p = (uintptr_t)x.p;
        bool done = !p;
        for (int i = 0; i < std::min(known, 4); i++) done |= p >= begin[i] && p < end[i];
        if (done) continue;
        unsigned type = 0, managed = 0;
        int at = -1;
        CUdeviceptr device_ptr = 0, start = 0;
        size_t bytes = 0;
        CUpointer_attribute what[6] = {CU_POINTER_ATTRIBUTE_MEMORY_TYPE, CU_POINTER_ATTRIBUTE_IS_MANAGED, CU_POINTER_ATTRIBUTE_DEVICE_ORDINAL,
                                       CU_POINTER_ATTRIBUTE_DEVICE_POINTER, CU_POINTER_ATTRIBUTE_RANGE_START_ADDR, CU_POINTER_ATTRIBUTE_RANGE_SIZE};
        void* into[6] = {&type, &managed, &at, &device_ptr, &start, &bytes};
        if (pointer_attributes()(6, what, into, (CUdeviceptr)p) != CUDA_SUCCESS) type = managed = 0;
        const bool here = managed || (type == CU_MEMORYTYPE_DEVICE && at == dev);
        if (!here && !(x.pinned && type == CU_MEMORYTYPE_HOST && (uintptr_t)device_ptr == p))
            return fail(LTHN_ERR_INVALID, named(name, x.what) + " is not memory of the current device");
        if (here && bytes) {
            begin[known % 4] = (uintptr_t)start;
            end[known++ % 4] = (uintptr_t)start + bytes;
        }
    }
    return LTHN_OK;
}

int32_t paged_check_cache(const char* name, const lthn_paged_kv* c, PagedCache* out) {
    LTHN_REQUIRE(c != nullptr, named(name, "cache is NULL"));
    LTHN_REQUIRE(c->k && c->v && c->page_table, named(name, "NULL pointer in the cache description"));
    LTHN_REQUIRE(c->kv_heads > 0 && c->kv_heads <= 65535, named(name, "kv_heads must be in [1, 65535]"));
    LTHN_REQUIRE(c->head_dim == 64 || c->head_dim == 128 || c->head_dim == 256, named(name, "head_dim must be 64, 128 or 256"));
    LTHN_REQUIRE(c->page_size >= 1, named(name, "page_size must be at least 1"));
    LTHN_REQUIRE(c->pages >= 0 && c->table_stride >= 0 && c->seqs >= 0, named(name, "negative size in the cache description"));
    const int64_t kr = (int64_t)c->kv_heads * c->head_dim;
    LTHN_REQUIRE((int64_t)c->page_size <= INT64_MAX / kr / 2, named(name, "page_size too large"));
    PagedCache o;
    o.k = c->k; o.v = c->v; o.table = c->page_table;
    o.row_stride = c->row_stride ? c->row_stride : kr;
    o.head_stride = c->head_stride ? c->head_stride : c->head_dim;
    o.page_stride = c->page_stride ? c->page_stride : c->page_size * kr;
    LTHN_REQUIRE(o.row_stride > 0 && o.head_stride > 0 && o.page_stride > 0, named(name, "negative stride in the cache description"));
    LTHN_REQUIRE(((o.row_stride | o.head_stride | o.page_stride) & 7) == 0, named(name, "cache strides must be multiples of 8 elements"));
    LTHN_REQUIRE((((uintptr_t)c->k | (uintptr_t)c->v) & 15) == 0, named(name, "k and v must be 16-byte aligned"));
    o.pages = c->pages; o.page_size = c->page_size; o.table_stride = c->table_stride; o.seqs = c->seqs; o.kv_heads = c->kv_heads;
    o.capacity = (int)std::min<int64_t>((int64_t)c->table_stride * c->page_size, 1 << 26);
    o.status = nullptr;
    o.div_shift = 27;
    while (((int64_t)1 << (o.div_shift - 27)) < c->page_size) o.div_shift++;
    o.div_mul = (uint32_t)((((uint64_t)1 << o.div_shift) + c->page_size - 1) / (uint32_t)c->page_size);
    *out = o;
    return LTHN_OK;
}

int32_t paged_check_options(const char* name, const lthn_attn_options* o, int head_dim, AttnOpts* out) {
    AttnOpts a{0.f, 0.f, nullptr, 0, nullptr};
    if (o) {
        LTHN_REQUIRE(o->softcap >= 0.f && o->softcap < INFINITY, named(name, "softcap must be finite and not negative"));
        LTHN_REQUIRE(o->scale == o->scale && o->scale < INFINITY, named(name, "scale must be finite"));
        LTHN_REQUIRE(o->window >= 0, named(name, "window must not be negative"));
        a.scale = o->scale; a.softcap = o->softcap; a.slopes = o->slopes; a.window = std::min(o->window, 1 << 30); a.prefix = o->prefix_lens;
    }
    if (a.scale <= 0.f) a.scale = 1.0f / sqrtf((float)head_dim);
    // Larger caps leave f32 in the units of the kernels; they differ from this one in scores next to the largest f32 alone.
    a.softcap = std::min(a.softcap, 0x1p126f * std::min(a.scale, 1.0f));
    *out = a;
    return LTHN_OK;
}

struct AppendArgs {
    PagedCache c;
    const void *q, *k, *v;
    void* q_out;
    int64_t q_stride, k_stride, v_stride, q_out_stride;
    const int32_t *row_seq, *row_pos;
    const double* inv_freq;
    const float *q_norm, *k_norm;
    float eps;
    int Hq, half_rot, interleaved;
};

// four elements as they lie in memory, and as f32
template <typename T> struct Four;
template <> struct Four<float> {
    typedef float4 raw;
    static __device__ __forceinline__ void widen(const raw& v, float (&x)[4]) { x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w; }
};
template <> struct Four<uint16_t> {
    typedef uint2 raw;
    static __device__ __forceinline__ void widen(const raw& v, float (&x)[4]) {
        x[0] = __uint_as_float(v.x << 16); x[1] = __uint_as_float(v.x & 0xffff0000u);
        x[2] = __uint_as_float(v.y << 16); x[3] = __uint_as_float(v.y & 0xffff0000u);
    }
};
__device__ __forceinline__ void store4(float* p, const float (&x)[4]) { *(float4*)p = make_float4(x[0], x[1], x[2], x[3]); }
__device__ __forceinline__ void store4(uint16_t* p, const float (&x)[4]) {
    *(uint2*)p = make_uint2(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]));
}

constexpr int AP_THREADS = 128;
constexpr int AP_BATCH = 4;    // heads of a thread whose loads go out together

template <int D, typename TI, typename TQ>
__global__ void __launch_bounds__(AP_THREADS, sizeof(TI) == 2 ? 10 : 6) paged_append_kernel(const AppendArgs a) {
    constexpr int TPH = D / 8;                 // threads per head: 8, 16 or 32
    constexpr int HPP = AP_THREADS / TPH;      // heads per pass
    typedef typename Four<TI>::raw raw;
    __shared__ __align__(16) float2 turn[D / 2];   // (cos, sin) of each rotated pair
    const int row = blockIdx.x, tid = threadIdx.x, j = tid % TPH, heads = a.Hq + 2 * a.c.kv_heads;
    const int seq = a.row_seq[row];
    const int pos = a.row_pos[row];
    const TI* q_row = (const TI*)a.q + row * a.q_stride + 4 * j;
    const TI* k_row = (const TI*)a.k + row * a.k_stride + 4 * j - (int64_t)a.Hq * D;   // so that head h of q, k, v lies at h * D
    const TI* v_row = (const TI*)a.v + row * a.v_stride + 4 * j - (int64_t)(a.Hq + a.c.kv_heads) * D;
    raw lo[AP_BATCH], hi[AP_BATCH];            // elements 4j.. of the first and of the second half of this thread's heads
    auto load = [&](int h0) {
#pragma unroll
        for (int b = 0; b < AP_BATCH; b++) {
            const int h = h0 + b * HPP + tid / TPH;
            lo[b] = raw{};
            hi[b] = raw{};
            if (h < heads) {
                const TI* src = (h < a.Hq ? q_row : h < a.Hq + a.c.kv_heads ? k_row : v_row) + h * D;
                lo[b] = *(const raw*)src;
                hi[b] = *(const raw*)(src + D / 2);
            }
        }
    };
    load(HPP * AP_BATCH * blockIdx.y);                                   // needs neither position nor page: under way while those are looked up
    if (seq < 0) return;                       // padding row
    if (seq >= a.c.seqs || pos < 0 || pos >= a.c.capacity) {
        if (tid == 0) atomicOr(a.c.status, LTHN_STATUS_PAGED);
        return;
    }
    const int entry = paged_entry(a.c, pos);
    const int page = a.c.table[(int64_t)seq * a.c.table_stride + entry];
    for (int i = tid; i < a.half_rot; i += AP_THREADS) {
        const double turns = (double)pos * a.inv_freq[i] * 0.15915494309189535;  // of a full circle
        float s, c;
        sincospif(2.0f * (float)(turns - rint(turns)), &s, &c);
        turn[i] = make_float2(c, s);
    }
    const int64_t off = paged_offset(a.c, page, pos - entry * a.c.page_size);
    if (off < 0) return;                       // (the same for all threads)
    __syncthreads();
    // What this thread's pairs are multiplied with is the same for all its heads. Pair e: (x[e], y[e]), or of neighbours (x0 x1) (x2 x3)
    // (y0 y1) (y2 y3).
    const bool norms = a.q_norm || a.k_norm;
    float2 rot[4];
    bool turned[4];
#pragma unroll
    for (int e = 0; e < 4; e++) {
        const int i = a.interleaved ? 2 * j + (e & 1) + (e >> 1) * (D / 4) : 4 * j + e;
        turned[e] = i < a.half_rot;
        rot[e] = turned[e] ? turn[i] : make_float2(1.f, 0.f);
    }
    auto rotate = [](float& p, float& q, float2 t) {
        const float u = p, v = q;
        p = u * t.x - v * t.y;
        q = u * t.y + v * t.x;
    };
    TQ* q_dst = (TQ*)a.q_out + row * a.q_out_stride + 4 * j;
    uint16_t* k_dst = a.c.k + off + 4 * j;
    uint16_t* v_dst = a.c.v + off + 4 * j;
    for (int h0 = HPP * AP_BATCH * blockIdx.y;;) {                       // the same trip count for all: the reduction takes every thread
#pragma unroll
        for (int b = 0; b < AP_BATCH; b++) {
            const int h = h0 + b * HPP + tid / TPH;
            const bool live = h < heads, is_q = h < a.Hq, is_v = h >= a.Hq + a.c.kv_heads;
            float x[4], y[4];
            Four<TI>::widen(lo[b], x);
            Four<TI>::widen(hi[b], y);
            if (norms) {
                float ss = 0.f;
#pragma unroll
                for (int e = 0; e < 4; e++) ss = fmaf(x[e], x[e], fmaf(y[e], y[e], ss));
#pragma unroll
                for (int o = TPH / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o, TPH);
                const float* w = is_q ? a.q_norm : a.k_norm;
                if (w && live && !is_v) {
                    const float r = rsqrtf(fmaf(ss, 1.0f / D, a.eps));   // two units in the last place
                    const float4 wl = *(const float4*)(w + 4 * j), wh = *(const float4*)(w + 4 * j + D / 2);
                    x[0] *= r * wl.x; x[1] *= r * wl.y; x[2] *= r * wl.z; x[3] *= r * wl.w;
                    y[0] *= r * wh.x; y[1] *= r * wh.y; y[2] *= r * wh.z; y[3] *= r * wh.w;
                }
            }
            if (!live) continue;
            if (!is_v) {
                if (a.interleaved) {
                    if (turned[0]) rotate(x[0], x[1], rot[0]);
                    if (turned[1]) rotate(x[2], x[3], rot[1]);
                    if (turned[2]) rotate(y[0], y[1], rot[2]);
                    if (turned[3]) rotate(y[2], y[3], rot[3]);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        if (turned[e]) rotate(x[e], y[e], rot[e]);
                }
            }
            if (is_q) {
                TQ* dst = q_dst + h * D;
                store4(dst, x);
                store4(dst + D / 2, y);
            } else {
                uint16_t* dst = is_v ? v_dst + (h - a.Hq - a.c.kv_heads) * a.c.head_stride : k_dst + (h - a.Hq) * a.c.head_stride;
                store4(dst, x);
                store4(dst + D / 2, y);
            }
        }
        h0 += HPP * AP_BATCH * gridDim.y;
        if (h0 >= heads) break;
        load(h0);
    }
}

template <int D>
static void launch_append(cudaStream_t s, const AppendArgs& a, int rows, int dtype, int q_dtype) {
    const bool fi = dtype == LTHN_DTYPE_F32, fq = q_dtype == LTHN_DTYPE_F32;
    // Rows that leave SMs idle are shared between CTAs, AP_BATCH heads of a thread each; each forms the row's angles anew.
    constexpr int share = AP_THREADS / (D / 8) * AP_BATCH;
    const int shares = (a.Hq + 2 * a.c.kv_heads + share - 1) / share;
    const dim3 grid(rows, (int64_t)rows * shares <= 4 * 148 ? shares : 1);
    if (fi && fq) paged_append_kernel<D, float, float><<<grid, AP_THREADS, 0, s>>>(a);
    else if (fi) paged_append_kernel<D, float, uint16_t><<<grid, AP_THREADS, 0, s>>>(a);
    else if (fq) paged_append_kernel<D, uint16_t, float><<<grid, AP_THREADS, 0, s>>>(a);
    else paged_append_kernel<D, uint16_t, uint16_t><<<grid, AP_THREADS, 0, s>>>(a);
}

}  // namespace lthn

using namespace lthn;

extern "C" int32_t lthn_paged_kv_append(void* stream, const lthn_paged_kv* cache, const lthn_rope_params* rope, const void* q,
                                        const void* k, const void* v, int32_t dtype, int64_t q_stride, int64_t k_stride, int64_t v_stride,
                                        const int32_t* row_seq, const int32_t* row_pos, int32_t rows, int32_t q_heads, void* q_out,
                                        int32_t q_dtype, int64_t q_out_stride) {
    clear_error();
    const char* me = "paged_kv_append";
    AppendArgs a = {};
    int32_t rc;
    if ((rc = paged_check_cache(me, cache, &a.c))) return rc;
    LTHN_REQUIRE(rows >= 0, "paged_kv_append: negative row count");
    LTHN_REQUIRE(dtype == LTHN_DTYPE_F32 || dtype == LTHN_DTYPE_BF16, "paged_kv_append: dtype must be f32 or bf16");
    LTHN_REQUIRE(q_dtype == LTHN_DTYPE_F32 || q_dtype == LTHN_DTYPE_BF16, "paged_kv_append: q_dtype must be f32 or bf16");
    const int D = cache->head_dim;
    if (!q) q_heads = 0;
    LTHN_REQUIRE(q_heads >= 0 && q_heads <= 65535, "paged_kv_append: q_heads must be in [0, 65535]");
    if (rope) {
        LTHN_REQUIRE(rope->rotary_dim >= 0 && rope->rotary_dim % 2 == 0 && rope->rotary_dim <= D, "paged_kv_append: rotary_dim must be even and at most head_dim");
        LTHN_REQUIRE(rope->interleaved == 0 || rope->interleaved == 1, "paged_kv_append: interleaved must be 0 or 1");
        LTHN_REQUIRE((((uintptr_t)rope->q_norm | (uintptr_t)rope->k_norm) & 15) == 0, "paged_kv_append: norm weights must be 16-byte aligned");
        LTHN_REQUIRE(rope->eps >= 0.f && rope->eps < INFINITY, "paged_kv_append: eps must be finite and not negative");
        a.inv_freq = rope->inv_freq;
        a.half_rot = rope->inv_freq ? rope->rotary_dim / 2 : 0;
        a.interleaved = rope->interleaved;
        a.q_norm = rope->q_norm; a.k_norm = rope->k_norm; a.eps = rope->eps;
    }
    if (rows == 0) return LTHN_OK;
    LTHN_REQUIRE(k && v && row_seq && row_pos, "paged_kv_append: NULL pointer");
    LTHN_REQUIRE(!q_heads || q_out, "paged_kv_append: q_out is NULL");
    a.q_stride = q_stride ? q_stride : (int64_t)q_heads * D;
    a.q_out_stride = q_out_stride ? q_out_stride : (int64_t)q_heads * D;
    a.k_stride = k_stride ? k_stride : (int64_t)cache->kv_heads * D;
    a.v_stride = v_stride ? v_stride : (int64_t)cache->kv_heads * D;
    LTHN_REQUIRE(((a.q_stride | a.k_stride | a.v_stride | a.q_out_stride) & 7) == 0, "paged_kv_append: strides must be multiples of 8 elements");
    LTHN_REQUIRE(!q_heads || a.q_out_stride >= (int64_t)q_heads * D, "paged_kv_append: rows of q_out would overlap");
    LTHN_REQUIRE((((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)(q_heads ? q_out : nullptr)) & 15) == 0,
                 "paged_kv_append: q, k, v and q_out must be 16-byte aligned");
    LTHN_REQUIRE(!q_heads || q_out != q || (q_dtype == dtype && a.q_out_stride == a.q_stride),
                 "paged_kv_append: q_out may be q itself only with the same type and stride");
    if ((rc = paged_check_pointers(me, {{"the cache's k", cache->k, 16, false}, {"the cache's v", cache->v, 16, false},
                                        {"page_table", cache->page_table, 4, true}, {"k", k, 16, false}, {"v", v, 16, true}, {"q", q_heads ? q : nullptr, 16, true},
                                        {"q_out", q_heads ? q_out : nullptr, 16, true}, {"row_seq", row_seq, 4, true}, {"row_pos", row_pos, 4, true},
                                        {"inv_freq", a.half_rot ? a.inv_freq : nullptr, 8, true}, {"q_norm", q_heads ? a.q_norm : nullptr, 16, true},
                                        {"k_norm", a.k_norm, 16, true}})))
        return rc;
    a.q = q; a.k = k; a.v = v; a.q_out = q_out; a.Hq = q_heads;
    a.row_seq = row_seq; a.row_pos = row_pos;
    a.c.status = device_paged_status_word();
    if (!a.c.status) return fail(LTHN_ERR_CUDA, "paged_kv_append: no device status word");
    if (D == 64) launch_append<64>((cudaStream_t)stream, a, rows, dtype, q_dtype);
    else if (D == 128) launch_append<128>((cudaStream_t)stream, a, rows, dtype, q_dtype);
    else launch_append<256>((cudaStream_t)stream, a, rows, dtype, q_dtype);
    LTHN_CUDA_TRY(cudaGetLastError());
    return LTHN_OK;
}
