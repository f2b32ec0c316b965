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
// one token row: its D/2 angles are formed once, by one thread each, and read by all of the row's heads. The angle is the
// only place where 32 bits are not enough (position 200000 leaves an f32 angle 0.01 off), so it is formed in f64, in
// turns, reduced there to [-1/2, 1/2], and handed to sincospif.
#include "paged.cuh"

#include <algorithm>

namespace lthn {

static std::string named(const char* name, const char* what) { return std::string(name) + ": " + what; }

int paged_sm_count() {
    int dev = 0, sms = 148;
    if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    return sms;
}

int32_t paged_check_device(const char* name, const char* what, const void* p) {
    cudaPointerAttributes at;
    int dev = 0;
    LTHN_CUDA_TRY(cudaGetDevice(&dev));
    if (cudaPointerGetAttributes(&at, p) != cudaSuccess) {
        cudaGetLastError();
        return fail(LTHN_ERR_INVALID, named(name, what) + " is not a pointer CUDA knows");
    }
    if (at.type != cudaMemoryTypeManaged && (at.type != cudaMemoryTypeDevice || at.device != dev))
        return fail(LTHN_ERR_INVALID, named(name, what) + " is not memory of the current device");
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

__device__ __forceinline__ void load4(const float* p, float (&x)[4]) {
    const float4 v = *(const float4*)p;
    x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
}
__device__ __forceinline__ void load4(const uint16_t* p, float (&x)[4]) {
    const uint2 v = *(const uint2*)p;
    x[0] = __uint_as_float(v.x << 16); x[1] = __uint_as_float(v.x & 0xffff0000u);
    x[2] = __uint_as_float(v.y << 16); x[3] = __uint_as_float(v.y & 0xffff0000u);
}
__device__ __forceinline__ void store4(float* p, const float (&x)[4]) { *(float4*)p = make_float4(x[0], x[1], x[2], x[3]); }
__device__ __forceinline__ void store4(uint16_t* p, const float (&x)[4]) {
    *(uint2*)p = make_uint2(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]));
}

constexpr int AP_THREADS = 256;

template <int D, typename TI, typename TQ>
__global__ void __launch_bounds__(AP_THREADS) paged_append_kernel(const AppendArgs a) {
    constexpr int TPH = D / 8;                 // threads per head: 8, 16 or 32
    constexpr int HPP = AP_THREADS / TPH;      // heads per pass
    __shared__ float2 turn[D / 2];             // (cos, sin) of each rotated pair
    const int row = blockIdx.x, tid = threadIdx.x;
    const int seq = a.row_seq[row];
    if (seq < 0) return;                       // padding row
    const int pos = a.row_pos[row];
    if (seq >= a.c.seqs || pos < 0 || pos >= a.c.capacity) {
        if (tid == 0) atomicOr(a.c.status, LTHN_STATUS_PAGED);
        return;
    }
    const int entry = paged_entry(a.c, pos);
    const int64_t off = paged_offset(a.c, a.c.table[(int64_t)seq * a.c.table_stride + entry], pos - entry * a.c.page_size);
    if (off < 0) return;
    for (int i = tid; i < a.half_rot; i += AP_THREADS) {
        const double turns = (double)pos * a.inv_freq[i] * 0.15915494309189535;  // of a full circle
        float s, c;
        sincospif(2.0f * (float)(turns - rint(turns)), &s, &c);
        turn[i] = make_float2(c, s);
    }
    __syncthreads();
    const int j = tid % TPH, heads = a.Hq + 2 * a.c.kv_heads;
    const bool norms = a.q_norm || a.k_norm;
    for (int h0 = 0; h0 < heads; h0 += HPP) {  // the same trip count for all: the reduction below takes every thread
        const int h = h0 + tid / TPH;
        const bool live = h < heads, is_q = h < a.Hq, is_v = h >= a.Hq + a.c.kv_heads;
        const int kh = is_q ? h : is_v ? h - a.Hq - a.c.kv_heads : h - a.Hq;
        const TI* src = is_q ? (const TI*)a.q + row * a.q_stride : is_v ? (const TI*)a.v + row * a.v_stride : (const TI*)a.k + row * a.k_stride;
        src += (int64_t)kh * D + 4 * j;
        float lo[4] = {0.f, 0.f, 0.f, 0.f}, hi[4] = {0.f, 0.f, 0.f, 0.f};  // elements 4j.. of the first and of the second half
        if (live) {
            load4(src, lo);
            load4(src + D / 2, hi);
        }
        float ss = 0.f;
        if (norms) {
#pragma unroll
            for (int e = 0; e < 4; e++) ss += lo[e] * lo[e] + hi[e] * hi[e];
#pragma unroll
            for (int o = TPH / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o, TPH);
        }
        if (!live) continue;
        if (!is_v) {
            const float* w = is_q ? a.q_norm : a.k_norm;
            if (w) {
                const float r = 1.0f / sqrtf(ss * (1.0f / D) + a.eps);
                float wl[4], wh[4];
                load4(w + 4 * j, wl);
                load4(w + 4 * j + D / 2, wh);
#pragma unroll
                for (int e = 0; e < 4; e++) { lo[e] = lo[e] * r * wl[e]; hi[e] = hi[e] * r * wh[e]; }
            }
            if (a.interleaved) {
#pragma unroll
                for (int e = 0; e < 4; e += 2) {
                    const int p0 = 2 * j + e / 2, p1 = D / 4 + p0;
                    if (p0 < a.half_rot) {
                        const float2 t = turn[p0];
                        const float x = lo[e], y = lo[e + 1];
                        lo[e] = x * t.x - y * t.y;
                        lo[e + 1] = x * t.y + y * t.x;
                    }
                    if (p1 < a.half_rot) {
                        const float2 t = turn[p1];
                        const float x = hi[e], y = hi[e + 1];
                        hi[e] = x * t.x - y * t.y;
                        hi[e + 1] = x * t.y + y * t.x;
                    }
                }
            } else {
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    if (4 * j + e >= a.half_rot) continue;
                    const float2 t = turn[4 * j + e];
                    const float x = lo[e], y = hi[e];
                    lo[e] = x * t.x - y * t.y;
                    hi[e] = x * t.y + y * t.x;
                }
            }
        }
        if (is_q) {
            TQ* dst = (TQ*)a.q_out + row * a.q_out_stride + (int64_t)kh * D + 4 * j;
            store4(dst, lo);
            store4(dst + D / 2, hi);
        } else {
            uint16_t* dst = (is_v ? a.c.v : a.c.k) + off + kh * a.c.head_stride + 4 * j;
            store4(dst, lo);
            store4(dst + D / 2, hi);
        }
    }
}

template <int D>
static void launch_append(cudaStream_t s, const AppendArgs& a, int rows, int dtype, int q_dtype) {
    const bool fi = dtype == LTHN_DTYPE_F32, fq = q_dtype == LTHN_DTYPE_F32;
    if (fi && fq) paged_append_kernel<D, float, float><<<rows, AP_THREADS, 0, s>>>(a);
    else if (fi) paged_append_kernel<D, float, uint16_t><<<rows, AP_THREADS, 0, s>>>(a);
    else if (fq) paged_append_kernel<D, uint16_t, float><<<rows, AP_THREADS, 0, s>>>(a);
    else paged_append_kernel<D, uint16_t, uint16_t><<<rows, AP_THREADS, 0, s>>>(a);
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
    if ((rc = paged_check_device(me, "the cache", cache->k))) return rc;
    if ((rc = paged_check_device(me, "k", k))) return rc;
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
