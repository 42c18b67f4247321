// sc_paged.cu -- the paged KV cache: rotation and appending of new tokens, and causal attention of the
// new tokens over the pages.
#include <cudaTypedefs.h>

#include <atomic>
#include <mutex>
#include <string>

#include "saccade_qwen2.h"
#include "sc_device.cuh"
#include "sc_internal.h"
#include "sc_paged.cuh"

namespace sc {

template <typename T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// ---------------------------------------------------------------- rotation + append
// A thread has 8 rotated pairs (elements d..d+7 and d+hd/2..d+hd/2+7) of one token and takes the
// heads in turn, so that the token's angles are loaded once for all of its heads; q, k and v heads
// follow one another in the loop.  Bytes bound: q, k, v read, q' and the cache rows written, two
// table rows per token.  The loads of the first heads do not depend on the token's place: they are issued before
// it is looked up.  16-bit rows hold the angles in registers and take two heads at a time (43 us at 2 x 2048 tokens
// of 64 + 8 heads, bf16: 4.0 TB/s; from the L1 cache for each head 46 us); f32 rows, which need those registers,
// take the angles from the cache (4.2 us at 1,200 tokens of 14 + 2 heads; held 5.8 us).  CTAs that stay and
// fetch their next token beside the present one measured slower (50 us).
constexpr int kAppendThreads = 256;

struct AppendArgs {
    const void *q, *k, *v;
    int64_t q_stride, k_stride, v_stride;
    const float *cos_t, *sin_t;
    int64_t max_pos;
    void *kp, *vp, *q_out;
    PagedKv c;
    int vec_in;      // q, k, v rows start on 16-byte boundaries
    int vec_cache;   // the pages do
    int vec_table;   // the rotation tables do
    int vec_qout;
};

template <typename T>
struct Eight {  // 8 consecutive values as they are in memory
    __align__(16) T v[8];
    __device__ __forceinline__ void load(const T* p, bool vec) {
        if (vec) {
#pragma unroll
            for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i)
                reinterpret_cast<uint4*>(v)[i] = reinterpret_cast<const uint4*>(p)[i];
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = p[i];
        }
    }
};
template <typename T>
__device__ __forceinline__ void store8(T* p, bool vec, const float (&f)[8]) {
    __align__(16) T t[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) t[i] = from_f32<T>(f[i]);
    if (vec) {
#pragma unroll
        for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i)
            reinterpret_cast<uint4*>(p)[i] = reinterpret_cast<const uint4*>(t)[i];
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) p[i] = t[i];
    }
}

__device__ __forceinline__ float4 load4(const float* p, bool vec) {
    return vec ? __ldg(reinterpret_cast<const float4*>(p)) : make_float4(__ldg(p), __ldg(p + 1), __ldg(p + 2), __ldg(p + 3));
}
// (x, y) by the angle of (c0, s0) in x and (c1, s1) in y, products and sums each rounded.
__device__ __forceinline__ void rotate(float& x, float& y, float c0, float s0, float c1, float s1) {
    const float r = __fsub_rn(__fmul_rn(x, c0), __fmul_rn(y, s0));
    y = __fadd_rn(__fmul_rn(y, c1), __fmul_rn(x, s1));
    x = r;
}

template <typename In, typename Cache, int kHd>
__global__ void __launch_bounds__(kAppendThreads, sizeof(In) == 4 ? 4 : 3) k_paged_append(const AppendArgs a) {
    constexpr int kHalf = kHd / 2;
    constexpr int kChunks = kHalf / 8;                 // threads of one head
    constexpr int kHeads = kAppendThreads / kChunks;   // heads taken at a time
    constexpr bool kHeld = sizeof(In) == 2;            // the angles stay in registers
    constexpr int kBatch = kHeld ? 2 : 1;
    pdl_launch_dependents();
    const int64_t t = blockIdx.x;
    const int lane = threadIdx.x & 31;
    const int nh = a.c.nh, nkv = a.c.nkv, all = nh + 2 * nkv;
    const int d = (threadIdx.x % kChunks) * 8;
    const int step = kHeads * static_cast<int>(gridDim.y);
    int h0 = threadIdx.x / kChunks + static_cast<int>(blockIdx.y) * kHeads;
    Eight<In> x0[kBatch], x1[kBatch];
    auto load = [&]() {
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            const int h = h0 + i * step;
            if (h >= all) continue;
            const In* src = h < nh ? static_cast<const In*>(a.q) + t * a.q_stride + h * kHd
                            : h < nh + nkv ? static_cast<const In*>(a.k) + t * a.k_stride + (h - nh) * kHd
                                           : static_cast<const In*>(a.v) + t * a.v_stride + (h - nh - nkv) * kHd;
            x0[i].load(src + d, a.vec_in);
            x1[i].load(src + d + kHalf, a.vec_in);
        }
    };
    pdl_wait();
    load();
    // the token's sequence: the number of sequences that end at or before it
    int seq = 0;
    for (int b0 = 0; b0 < a.c.num_seqs; b0 += 32) {
        const bool before = b0 + lane < a.c.num_seqs && a.c.cu_q[b0 + lane + 1] <= t;
        seq += __popc(__ballot_sync(0xffffffffu, before));
    }
    if (seq >= a.c.num_seqs || t < a.c.cu_q[seq]) return;  // a row behind the last sequence
    const int64_t pos = static_cast<int64_t>(a.c.kv_len[seq]) - a.c.cu_q[seq + 1] + t;
    if (pos < 0 || pos >= a.max_pos) {
        if (threadIdx.x == 0) record_error(a.c.status, DEV_BAD_INDEX);
        return;
    }
    const float *ct = a.cos_t + pos * kHd + d, *st = a.sin_t + pos * kHd + d;
    float4 angle[kHeld ? 8 : 1];
    if constexpr (kHeld) {
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            angle[4 * q] = load4(ct + 4 * q, a.vec_table);
            angle[4 * q + 1] = load4(st + 4 * q, a.vec_table);
            angle[4 * q + 2] = load4(ct + kHalf + 4 * q, a.vec_table);
            angle[4 * q + 3] = load4(st + kHalf + 4 * q, a.vec_table);
        }
    }
    int64_t page = -1;
    const int64_t slot = pos >> a.c.page_shift;
    if (slot < a.c.max_pages) page = a.c.table[seq * a.c.max_pages + slot];
    const bool held = page >= 0 && page < a.c.num_pages;
    if (!held && threadIdx.x == 0) record_error(a.c.status, DEV_BAD_INDEX);
    const int64_t in_page = (pos & ((1ll << a.c.page_shift) - 1)) * kHd + d;
    for (; h0 < all; h0 += kBatch * step) {
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            const int h = h0 + i * step;
            if (h >= all || (h >= nh && !held)) continue;
            float lo[8], hi[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                lo[e] = to_f32(x0[i].v[e]);
                hi[e] = to_f32(x1[i].v[e]);
            }
            if (h < nh + nkv) {
#pragma unroll
                for (int q = 0; q < 8; q += 4) {
                    float4 c0, s0, c1, s1;
                    if constexpr (kHeld) {
                        c0 = angle[q], s0 = angle[q + 1], c1 = angle[q + 2], s1 = angle[q + 3];
                    } else {
                        c0 = load4(ct + q, a.vec_table), s0 = load4(st + q, a.vec_table);
                        c1 = load4(ct + kHalf + q, a.vec_table), s1 = load4(st + kHalf + q, a.vec_table);
                    }
                    rotate(lo[q], hi[q], c0.x, s0.x, c1.x, s1.x);
                    rotate(lo[q + 1], hi[q + 1], c0.y, s0.y, c1.y, s1.y);
                    rotate(lo[q + 2], hi[q + 2], c0.z, s0.z, c1.z, s1.z);
                    rotate(lo[q + 3], hi[q + 3], c0.w, s0.w, c1.w, s1.w);
                }
            }
            Cache* dst;
            bool vec = a.vec_cache;
            if (h < nh) {
                dst = static_cast<Cache*>(a.q_out) + (t * nh + h) * kHd + d;
                vec = a.vec_qout;
            } else {
                const int hk = h < nh + nkv ? h - nh : h - nh - nkv;
                dst = static_cast<Cache*>(h < nh + nkv ? a.kp : a.vp) + page * a.c.page_stride +
                      (static_cast<int64_t>(hk) << a.c.page_shift) * kHd + in_page;
            }
            store8(dst, vec, lo);
            store8(dst + kHalf, vec, hi);
        }
        if (h0 + kBatch * step < all) {
            const int keep = h0;
            h0 += kBatch * step;
            load();
            h0 = keep;
        }
    }
}

template <typename In, typename Cache>
static cudaError_t launch_append(const AppendArgs& a, int hd, cudaStream_t s) {
    const int heads_at_once = kAppendThreads / (hd / 16), heads = a.c.nh + 2 * a.c.nkv;
    // few tokens: the heads of one on several CTAs, down to one pass over them
    int split = 1;
    while (a.c.tokens * split < 296 && split * heads_at_once < heads) ++split;
    const dim3 grid(static_cast<unsigned>(a.c.tokens), static_cast<unsigned>(split));
    return hd == 128 ? launch_pdl(k_paged_append<In, Cache, 128>, grid, dim3(kAppendThreads), 0, s, a)
                     : launch_pdl(k_paged_append<In, Cache, 64>, grid, dim3(kAppendThreads), 0, s, a);
}

static PFN_cuTensorMapEncodeTiled_v12000 map_encoder() {
    static std::once_flag once;
    static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
    std::call_once(once, [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
    });
    return fn;
}

static cudaError_t encode_map(CUtensorMap* map, const void* base, int dtype, const cuuint64_t (&dims)[4],
                              const cuuint64_t (&strides)[3], const cuuint32_t (&box)[4], CUtensorMapL2promotion l2) {
    PFN_cuTensorMapEncodeTiled_v12000 encode = map_encoder();
    if (!encode) return cudaErrorNotSupported;
    const cuuint32_t es[4] = {1, 1, 1, 1};
    const CUresult r = encode(map, dtype == SC_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4,
                              const_cast<void*>(base), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
                              CU_TENSOR_MAP_SWIZZLE_128B, l2, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

cudaError_t paged_tensor_map(CUtensorMap* map, const PagedKv& c, const void* pages, int dtype, int hd, int box_rows) {
    const cuuint64_t page = 1ull << c.page_shift;
    const cuuint64_t dims[4] = {static_cast<cuuint64_t>(hd), page, static_cast<cuuint64_t>(c.nkv),
                                static_cast<cuuint64_t>(c.num_pages)};
    const cuuint64_t strides[3] = {static_cast<cuuint64_t>(hd) * 2, page * hd * 2,
                                   static_cast<cuuint64_t>(c.page_stride) * 2};
    const cuuint32_t box[4] = {64, static_cast<cuuint32_t>(box_rows), 1, 1};
    return encode_map(map, pages, dtype, dims, strides, box, CU_TENSOR_MAP_L2_PROMOTION_L2_256B);
}

cudaError_t paged_query_map(CUtensorMap* map, const PagedLaunch& a, int dtype, int hd, int box_tokens) {
    const int G = a.c.nh / a.c.nkv;
    const cuuint64_t dims[4] = {static_cast<cuuint64_t>(hd), static_cast<cuuint64_t>(G),
                                static_cast<cuuint64_t>(a.c.nkv), static_cast<cuuint64_t>(a.c.tokens)};
    // a single row's stride is never used, but must be a legal one
    const cuuint64_t row = a.c.tokens > 1 ? static_cast<cuuint64_t>(a.q_stride) * 2 : static_cast<cuuint64_t>(a.c.nh) * hd * 2;
    const cuuint64_t strides[3] = {static_cast<cuuint64_t>(hd) * 2, static_cast<cuuint64_t>(G) * hd * 2, row};
    const cuuint32_t box[4] = {64, static_cast<cuuint32_t>(G), 1, static_cast<cuuint32_t>(box_tokens)};
    return encode_map(map, a.q, dtype, dims, strides, box, CU_TENSOR_MAP_L2_PROMOTION_L2_128B);
}

int sm_count() {
    static std::atomic<int> cache[64];
    int dev = 0, n = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
    if ((n = cache[dev].load()) > 0) return n;
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) return 148;
    cache[dev].store(n);
    return n;
}

// The kernel of a call and its work division.
struct PagedPlan {
    enum Kind { kF32, kDecode, kChunk } kind;
    int64_t ctas;
    PagedTiling tl;
    int cluster;     // CTAs of an item's cluster; 0: the line of key tiles is cut, the pieces joined through the scratch
    size_t scratch;
};
static PagedPlan paged_plan(int dtype, int64_t num_seqs, int nh, int nkv, int hd, int64_t max_q, int64_t max_kv) {
    const int G = nh / nkv, sms = sm_count();
    const bool few = max_q <= 16 / G;
    PagedPlan p{};
    int64_t share = 0;  // positions of a clustered CTA at most
    if (dtype == SC_F32) {
        p.kind = PagedPlan::kF32;
        p.ctas = few || hd == 64 ? 2 * sms : sms;
        p.tl = few ? PagedTiling{16, 16, 16 / G, 64} : PagedTiling{64, 64, 64 / G, 64};
        share = few ? kClusterKeysF32 : 0;
    } else if (few) {
        p.kind = PagedPlan::kDecode;
        p.ctas = 2 * sms;
        p.tl = {16, 16, 16 / G, 64};
        share = kClusterKeys;
    } else {
        p.kind = PagedPlan::kChunk;
        p.ctas = sms;
        p.tl = {256, 128, 2 * (128 / G), 128};
    }
    if (share > 0) {  // few new tokens: a row tile per sequence and KV head
        const int64_t items = num_seqs * nkv;
        int cs = 1;
        while (cs < 8 && items * cs * 2 <= p.ctas && cs * 2 * p.tl.kt <= max_kv) cs *= 2;
        if (max_kv <= share * cs) {
            p.cluster = cs;
            p.ctas = items * cs;
        }
    }
    if (p.cluster == 0) p.scratch = paged_scratch_bytes(p.ctas, p.tl.rows, hd);
    return p;
}

static int64_t elem_size(int dtype) { return dtype == SC_F32 ? 4 : 2; }
static bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

static sc_status paged_bad(const char* who, const char* what) {
    set_error(std::string(who) + ": " + what);
    return SC_EINVAL;
}

// The arguments both entry points share.
static sc_status make_paged(const char* who, const void* k, const void* v, int dtype, int64_t num_pages, int64_t page_stride,
                            int page_size, const int32_t* table, int64_t max_pages, const int32_t* cu_q,
                            const int32_t* kv_len, int64_t num_seqs, int64_t tokens, int nh, int nkv, int hd,
                            uint32_t* status, PagedKv* c) {
    if (dtype != SC_F32 && dtype != SC_F16 && dtype != SC_BF16) return paged_bad(who, "the cache is f32, f16 or bf16");
    if (!k || !v || !table || !cu_q || !kv_len) return paged_bad(who, "null pages, block table or lengths");
    if (hd != 64 && hd != 128) return paged_bad(who, "head_dim is 64 or 128");
    if (nkv <= 0 || nh <= 0 || nh % nkv || nh / nkv > kPagedMaxGroup || nh > 65536)
        return paged_bad(who, "num_heads must be a multiple of num_kv_heads, at most 64 per KV head");
    if (page_size < kPagedMinPage || page_size > kPagedMaxPage || (page_size & (page_size - 1)))
        return paged_bad(who, "page_size must be a power of two in 8..256");
    if (num_pages <= 0 || num_pages > 0x7fffffff || page_stride < static_cast<int64_t>(nkv) * page_size * hd)
        return paged_bad(who, "pages overlap, or none");
    if (max_pages <= 0 || max_pages > 0x7fffffff / page_size) return paged_bad(who, "max_pages out of range");
    if (num_seqs <= 0 || num_seqs > (1 << 20) || tokens > 0x7fffffff / nh)
        return paged_bad(who, "too many sequences or tokens");
    const uintptr_t size = static_cast<uintptr_t>(elem_size(dtype));
    if ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) % size)
        return paged_bad(who, "pages must be aligned to their type");
    c->k = k;
    c->v = v;
    c->num_pages = num_pages;
    c->page_stride = page_stride;
    c->page_shift = 0;
    while ((1 << c->page_shift) < page_size) ++c->page_shift;
    c->table = table;
    c->max_pages = max_pages;
    c->cu_q = cu_q;
    c->kv_len = kv_len;
    c->num_seqs = static_cast<int>(num_seqs);
    c->tokens = tokens;
    c->nh = nh;
    c->nkv = nkv;
    c->status = status;
    return SC_OK;
}

}  // namespace sc

using namespace sc;

extern "C" {

sc_status sc_qwen2_paged_append(const void* q, const void* k, const void* v, int in_dtype, int64_t q_stride,
                                int64_t k_stride, int64_t v_stride, int64_t tokens, const float* cos_table,
                                const float* sin_table, int64_t max_pos, int num_heads, int num_kv_heads, int head_dim,
                                void* k_pages, void* v_pages, int cache_dtype, int64_t num_pages, int64_t page_stride,
                                int page_size, const int32_t* block_table, int64_t max_pages, const int32_t* cu_q,
                                const int32_t* kv_len, int64_t num_seqs, void* q_out, uint32_t* status, void* stream) {
    const char* who = "sc_qwen2_paged_append";
    if (tokens <= 0) return tokens == 0 ? SC_OK : paged_bad(who, "a negative number of tokens");
    AppendArgs a = {};
    const sc_status st = make_paged(who, k_pages, v_pages, cache_dtype, num_pages, page_stride, page_size, block_table,
                                    max_pages, cu_q, kv_len, num_seqs, tokens, num_heads, num_kv_heads, head_dim,
                                    status, &a.c);
    if (st != SC_OK) return st;
    if (!q || !k || !v || !q_out || !cos_table || !sin_table) return paged_bad(who, "null q, k, v, q_out or table");
    if (in_dtype != SC_F32 && in_dtype != cache_dtype) return paged_bad(who, "q, k and v are f32 or of the cache's type");
    if (max_pos <= 0) return paged_bad(who, "empty rotation tables");
    const int64_t qw = static_cast<int64_t>(num_heads) * head_dim, kw = static_cast<int64_t>(num_kv_heads) * head_dim;
    if (tokens > 1 && (q_stride < qw || k_stride < kw || v_stride < kw)) return paged_bad(who, "rows overlap");
    const int64_t is = elem_size(in_dtype), cs = elem_size(cache_dtype);
    if (q_out == q ? in_dtype != cache_dtype || (tokens > 1 && q_stride != qw)
                   : ranges_meet(q_out, tokens * qw * cs, q, ((tokens - 1) * q_stride + qw) * is))
        return paged_bad(who, "in place needs contiguous rows of the cache's type");
    if (ranges_meet(q_out, tokens * qw * cs, k, ((tokens - 1) * k_stride + kw) * is) ||
        ranges_meet(q_out, tokens * qw * cs, v, ((tokens - 1) * v_stride + kw) * is))
        return paged_bad(who, "q_out lies over k or v");
    if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) % is ||
        reinterpret_cast<uintptr_t>(q_out) % cs ||
        (reinterpret_cast<uintptr_t>(cos_table) | reinterpret_cast<uintptr_t>(sin_table)) % 4)
        return paged_bad(who, "tensors must be aligned to their type");
    a.q = q;
    a.k = k;
    a.v = v;
    a.q_stride = q_stride;
    a.k_stride = k_stride;
    a.v_stride = v_stride;
    a.cos_t = cos_table;
    a.sin_t = sin_table;
    a.max_pos = max_pos;
    a.kp = k_pages;
    a.vp = v_pages;
    a.q_out = q_out;
    a.vec_in = aligned16(q) && aligned16(k) && aligned16(v) && (q_stride * is | k_stride * is | v_stride * is) % 16 == 0;
    a.vec_cache = aligned16(k_pages) && aligned16(v_pages) && page_stride * cs % 16 == 0;
    a.vec_table = aligned16(cos_table) && aligned16(sin_table);
    a.vec_qout = aligned16(q_out);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const cudaError_t e =
        cache_dtype == SC_F32 ? launch_append<float, float>(a, head_dim, s)
        : cache_dtype == SC_F16
            ? (in_dtype == SC_F32 ? launch_append<float, __half>(a, head_dim, s) : launch_append<__half, __half>(a, head_dim, s))
            : (in_dtype == SC_F32 ? launch_append<float, __nv_bfloat16>(a, head_dim, s)
                                  : launch_append<__nv_bfloat16, __nv_bfloat16>(a, head_dim, s));
    return e == cudaSuccess ? SC_OK : cuda_fail(e, who);
}

size_t sc_qwen2_paged_attention_scratch(int64_t num_seqs, int num_heads, int num_kv_heads, int head_dim, int64_t max_q_len,
                                        int64_t max_kv_len, int cache_dtype) {
    if (num_seqs <= 0 || num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads ||
        num_heads / num_kv_heads > kPagedMaxGroup || max_q_len <= 0 || max_kv_len <= 0 || (head_dim != 64 && head_dim != 128))
        return 0;
    return paged_plan(cache_dtype, num_seqs, num_heads, num_kv_heads, head_dim, max_q_len, max_kv_len).scratch;
}

sc_status sc_qwen2_paged_attention(const void* q, int64_t q_stride, const void* k_pages, const void* v_pages,
                                   int cache_dtype, int64_t num_pages, int64_t page_stride, int page_size,
                                   const int32_t* block_table, int64_t max_pages, const int32_t* cu_q,
                                   const int32_t* kv_len, int64_t num_seqs, int64_t tokens, int num_heads,
                                   int num_kv_heads, int head_dim, int64_t max_q_len, int64_t max_kv_len, float scale,
                                   void* out, int out_dtype, float* lse, void* scratch, size_t scratch_bytes,
                                   uint32_t* status, void* stream) {
    const char* who = "sc_qwen2_paged_attention";
    if (tokens <= 0) return tokens == 0 ? SC_OK : paged_bad(who, "a negative number of tokens");
    PagedKv c;
    const sc_status st = make_paged(who, k_pages, v_pages, cache_dtype, num_pages, page_stride, page_size, block_table,
                                    max_pages, cu_q, kv_len, num_seqs, tokens, num_heads, num_kv_heads, head_dim,
                                    status, &c);
    if (st != SC_OK) return st;
    if (!q || !out) return paged_bad(who, "null q or out");
    if (out_dtype != cache_dtype && !(cache_dtype == SC_F32 && out_dtype == SC_F16))
        return paged_bad(who, "out is of the cache's type, or f16 from an f32 cache");
    if (max_q_len <= 0 || max_kv_len <= 0) return paged_bad(who, "max_q_len and max_kv_len must be positive");
    if (!(scale > 0.0f) || scale - scale != 0.0f) return paged_bad(who, "scale must be positive and finite");
    const int64_t cs = elem_size(cache_dtype);
    const int64_t qw = static_cast<int64_t>(num_heads) * head_dim;
    if (tokens > 1 && q_stride < qw) return paged_bad(who, "rows of q overlap");
    if (q == out ? out_dtype != cache_dtype || (tokens > 1 && q_stride != qw)
                 : ranges_meet(out, tokens * qw * elem_size(out_dtype), q, ((tokens - 1) * q_stride + qw) * cs))
        return paged_bad(who, "out over q needs contiguous rows of q's type");
    if (!aligned16(q) || (tokens > 1 && q_stride * cs % 16) || !aligned16(k_pages) || !aligned16(v_pages) ||
        page_stride * cs % 16 || !aligned16(out))
        return paged_bad(who, "q, the pages, their strides and out must be 16-byte aligned");
    const PagedPlan p = paged_plan(cache_dtype, num_seqs, num_heads, num_kv_heads, head_dim, max_q_len, max_kv_len);
    if (scratch_bytes < p.scratch) {
        set_error(std::string(who) + ": scratch too small");
        return SC_ENOMEM;
    }
    if (p.scratch > 0 && (!scratch || !aligned16(scratch))) return paged_bad(who, "scratch must be 16-byte aligned");
    if (p.ctas > 0x7fffffff) return paged_bad(who, "too many sequences");
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const int ctas = static_cast<int>(p.ctas);
    const PagedLaunch a{c, q, q_stride, max_q_len, {out, lse, scale * 1.4426950408889634f}, p.tl,
                        paged_scratch(scratch, p.cluster ? 0 : p.ctas, p.tl.rows, head_dim)};
    cudaError_t e = p.kind == PagedPlan::kF32      ? launch_paged_f32(a, out_dtype, head_dim, ctas, p.cluster, s)
                    : p.kind == PagedPlan::kDecode ? launch_paged_decode(a, cache_dtype, head_dim, ctas, p.cluster, s)
                                                   : launch_paged_chunk(a, cache_dtype, head_dim, ctas, s);
    if (e == cudaSuccess && p.cluster == 0) e = launch_paged_combine(a, out_dtype, head_dim, ctas, s);
    return e == cudaSuccess ? SC_OK : cuda_fail(e, who);
}

}  // extern "C"
