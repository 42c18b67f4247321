// sc_paged.cuh -- the paged KV cache as the kernels see it.
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include <atomic>
#include <type_traits>

#include "sc_device.cuh"
#include "sc_internal.h"

namespace sc {

constexpr int64_t kClusterKeys = 2048;     // positions of a clustered CTA's share at most (sc_paged_decode.cu)
constexpr int64_t kClusterKeysF32 = 128;  // (sc_paged_f32.cu)
constexpr int kPagedMaxGroup = 64;     // query heads per KV head
constexpr int kPagedMinPage = 8, kPagedMaxPage = 256;

struct PagedKv {
    const void *k, *v;            // [num_pages] pages of [nkv][page][hd], page_stride elements apart
    int64_t num_pages, page_stride;
    int page_shift;               // log2 of the page size
    const int32_t* table;         // [num_seqs][max_pages]
    int64_t max_pages;
    const int32_t* cu_q;          // [num_seqs + 1]
    const int32_t* kv_len;        // [num_seqs]
    int num_seqs;
    int64_t tokens;               // rows of q: no sequence reaches beyond them
    int nh, nkv;
    uint32_t* status;
};

// A sequence's token rows and cached positions, cut to what the tables and rows hold.
struct PagedSeq {
    int64_t row0;   // its first token row
    int q_len;      // its new tokens
    int kv_len;     // its cached positions
};

__device__ __forceinline__ PagedSeq paged_seq(const PagedKv& p, int b, int64_t max_q) {
    const int64_t c0 = p.cu_q[b], c1 = p.cu_q[b + 1];
    const int64_t kv = p.kv_len[b], cap = p.max_pages << p.page_shift;
    PagedSeq s{c0, 0, 0};
    if (c0 < 0 || c1 < c0 || c1 > p.tokens || c1 - c0 > max_q || kv < 0) {
        record_error(p.status, DEV_BAD_INDEX);
        s.row0 = 0;
        return s;
    }
    s.q_len = static_cast<int>(c1 - c0);
    s.kv_len = static_cast<int>(kv);
    if (kv > cap) {
        record_error(p.status, DEV_BAD_INDEX);
        s.q_len = 0;  // its newest positions have no pages: the sequence is skipped
        s.kv_len = 0;
    }
    return s;
}

// ---------------------------------------------------------------- work division
// An item is a (sequence, KV head, row tile): tt consecutive new tokens with all query heads of the
// KV head, over key tiles of kt positions 0 .. (the row tile's last position).  The key tiles of all
// items, sequences first, then KV heads, then row tiles, form one line that is cut into equal pieces,
// one per CTA: no CTA has more than one tile above the mean whatever the lengths are.  Before its tiles an item
// has one more unit on the line, for what it costs besides them (queries, output): without it the CTAs
// with many short items are the last (16 prompts of 129..512 tokens: 81 us, with it 71).  An item cut by a
// piece's border leaves partial results (unnormalised output, maximum, sum) in the scratch, one slot
// for the item that the CTA continues (0) and one for the item that it begins and does not finish (1);
// k_paged_combine joins them in order.
struct PagedCut {
    int64_t total, per;    // units in all, units per CTA
    int64_t first, left;   // this CTA's first unit and number of units
    int b, h, rt, unit;    // where the first one is: its item, and which of the item's units
    PagedSeq s;            // its sequence
};

__device__ __forceinline__ int paged_row_tiles(const PagedSeq& s, int tt) { return (s.q_len + tt - 1) / tt; }

// Key tiles of row tile rt: at least one, so that rows without a key get their zeros.
__device__ __forceinline__ int paged_key_tiles(const PagedSeq& s, int rt, int tt, int kt) {
    const int last = min((rt + 1) * tt, s.q_len);
    const int keys = s.kv_len - s.q_len + last;
    return keys <= kt ? 1 : (keys + kt - 1) / kt;
}

// Units of one KV head of a sequence.
__device__ __forceinline__ int64_t paged_seq_units(const PagedSeq& s, int tt, int kt) {
    const int rts = paged_row_tiles(s, tt);
    int64_t n = rts;
    for (int rt = 0; rt < rts; ++rt) n += paged_key_tiles(s, rt, tt, kt);
    return n;
}

// The piece of CTA blockIdx.x of gridDim.x; every thread of the block calls it.
template <int kThreads>
__device__ __forceinline__ void paged_cut(const PagedKv& p, int64_t max_q, int tt, int kt, PagedCut* cut) {
    __shared__ int64_t s_warp[kThreads / 32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    // inclusive prefix sums of the sequences' units, a block of sequences at a time
    auto scan = [&](int64_t v, int64_t* block) {
        int64_t x = v;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t y = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x += y;
        }
        __syncthreads();
        if (lane == 31) s_warp[warp] = x;
        __syncthreads();
        int64_t before = 0, all = 0;
#pragma unroll
        for (int i = 0; i < kThreads / 32; ++i) {
            if (i < warp) before += s_warp[i];
            all += s_warp[i];
        }
        *block = all;
        return x + before;
    };
    auto units = [&](int b) -> int64_t {
        return b < p.num_seqs ? p.nkv * paged_seq_units(paged_seq(p, b, max_q), tt, kt) : 0;
    };
    int64_t total = 0, block = 0, mine = 0, incl = 0;
    for (int b0 = 0; b0 < p.num_seqs; b0 += kThreads) {
        mine = units(b0 + tid);
        incl = scan(mine, &block);
        total += block;
    }
    // (32-bit divisions where they do: a 64-bit one costs a hundred instructions)
    const bool small = total <= 0x7fffffff;
    const int64_t per = total <= 0 ? 1
                        : small    ? static_cast<int64_t>((static_cast<uint32_t>(total) + gridDim.x - 1) / gridDim.x)
                                   : (total + gridDim.x - 1) / gridDim.x;
    const int64_t first = per * blockIdx.x;
    if (tid == 0) {
        cut->total = total;
        cut->per = per;
        cut->first = first;
        cut->left = first < total ? imin64(per, total - first) : 0;
    }
    int64_t base = 0;
    for (int b0 = 0; b0 < p.num_seqs && first < total; b0 += kThreads) {
        if (p.num_seqs > kThreads) {
            mine = units(b0 + tid);
            incl = scan(mine, &block);
        }
        const int64_t rel = first - base;
        if (rel >= incl - mine && rel < incl) {
            const int b = b0 + tid;
            const PagedSeq s = paged_seq(p, b, max_q);
            int64_t at = rel - (incl - mine);
            const int64_t per_head = small ? static_cast<uint32_t>(mine) / static_cast<uint32_t>(p.nkv) : mine / p.nkv;
            const int h = static_cast<int>(small ? static_cast<uint32_t>(at) / static_cast<uint32_t>(per_head) : at / per_head);
            at -= h * per_head;
            cut->s = s;
            cut->b = b;
            cut->h = h;
            int rt = 0;
            for (int n; at >= (n = 1 + paged_key_tiles(s, rt, tt, kt)); ++rt) at -= n;
            cut->rt = rt;
            cut->unit = static_cast<int>(at);
        }
        base += block;
    }
    __syncthreads();
}

// Walks the items of a piece; every role of a CTA walks them by itself.
struct PagedWalk {
    PagedSeq s;
    int b, h, rt;
    int rts;        // row tiles of the sequence
    int tiles;      // key tiles of the item
    int t0, t1;     // the piece's share of them
    int64_t at, left;
    int unit;       // the next item's first unit in this piece

    __device__ __forceinline__ void begin(const PagedCut& c, int tt) {
        s = c.s;
        rts = c.left > 0 ? paged_row_tiles(s, tt) : 0;
        b = c.b;
        h = c.h;
        rt = c.rt - 1;
        unit = c.unit;
        at = c.first;
        left = c.left;
        t0 = t1 = tiles = 0;
    }
    // The next item that has tiles in this piece, or false at the piece's end.
    __device__ __forceinline__ bool next(const PagedKv& p, int64_t max_q, int tt, int kt) {
        if (left <= (unit == 0 ? 1 : 0)) return false;  // nothing, or an item's first unit alone
        if (++rt >= rts) {
            rt = 0;
            if (++h >= p.nkv) {
                h = 0;
                do {
                    if (++b >= p.num_seqs) return false;
                    s = paged_seq(p, b, max_q);
                } while (s.q_len == 0);
                rts = paged_row_tiles(s, tt);
            }
        }
        tiles = paged_key_tiles(s, rt, tt, kt);
        if (unit == 0) {
            unit = 1;
            ++at;
            --left;
        }
        t0 = unit - 1;
        t1 = static_cast<int>(imin64(tiles, t0 + left));
        unit = 0;
        at += t1 - t0;
        left -= t1 - t0;
        return true;
    }
    __device__ __forceinline__ bool whole() const { return t0 == 0 && t1 == tiles; }
    __device__ __forceinline__ int slot() const { return t0 > 0 ? 0 : 1; }
    // The pieces of an item that this piece begins: to the CTA that has its last tile.
    __device__ __forceinline__ int pieces(const PagedCut& c) const {
        return static_cast<int>((at - (t1 - t0) + tiles - 1) / c.per) - static_cast<int>(blockIdx.x) + 1;
    }
};

// ---------------------------------------------------------------- values that are not finite
// A row must not see the values of positions behind its own, but the products give them the weight 0, and
// 0 * inf is NaN.  The positions that some rows of an item attend and others do not are the item's own new
// tokens.  The kernels look their values over where they are staged, replace what is not finite by 0, and, once
// a CTA has met such a value, add these tokens' to the rows that do attend them after the rows have been
// written (inf or NaN, as the formula has them).

// Adds the values that are not finite of positions first .. last to columns c0 + kStep i .. + 3 of a written row.
template <typename T, int kHd, int kStep, typename Out>
__device__ __forceinline__ void paged_add_not_finite(const PagedKv& p, int b, int h, int first, int last, int c0, Out* row) {
#pragma unroll 1
    for (int key = first; key <= last; ++key) {
        const int64_t page = p.table[b * p.max_pages + (key >> p.page_shift)];
        if (page < 0 || page >= p.num_pages) continue;
        const T* v = static_cast<const T*>(p.v) + page * p.page_stride +
                     ((static_cast<int64_t>(h) << p.page_shift) + (key & ((1 << p.page_shift) - 1))) * kHd;
#pragma unroll 1
        for (int i = c0; i < kHd; i += kStep)
#pragma unroll 1
            for (int c = i; c < i + 4; ++c) {
                const float x = static_cast<float>(v[c]);
                if (!(x - x == 0.0f)) row[c] = static_cast<Out>(static_cast<float>(row[c]) + x);
            }
    }
}

// 16 bytes of 16-bit values of which any is not finite: those become 0.
template <typename T>
__device__ __forceinline__ bool finite_only(uint4& v) {
    constexpr uint32_t kExp = sizeof(T) == 2 && std::is_same<T, __half>::value ? 0x7C00u : 0x7F80u;
    uint32_t w[4] = {v.x, v.y, v.z, v.w};
    bool bad = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const bool lo = (w[i] & kExp) == kExp, hi = (w[i] >> 16 & kExp) == kExp;
        if (lo) w[i] &= 0xFFFF0000u;
        if (hi) w[i] &= 0x0000FFFFu;
        bad = bad || lo || hi;
    }
    v = make_uint4(w[0], w[1], w[2], w[3]);
    return bad;
}

// What k_paged_combine joins: the item that CTA w begins and does not finish (pieces 0: none).
struct PagedJoin {
    int64_t row0;          // the sequence's first token row
    int q_len, h, rt, pieces;
};

// Scratch of a launch of `ctas` CTAs with row tiles of `rows` rows.
struct PagedScratch {
    PagedJoin* join;       // [ctas]
    float* ml;             // [ctas][2 slots][rows][maximum (log2 units), sum]
    float* o;              // [ctas][2 slots][rows][hd]
};
inline size_t paged_scratch_bytes(int64_t ctas, int rows, int hd) {
    return static_cast<size_t>(ctas) * (sizeof(PagedJoin) + 2ull * rows * (hd + 2) * 4);
}
inline PagedScratch paged_scratch(void* base, int64_t ctas, int rows, int hd) {
    PagedScratch s;
    s.o = static_cast<float*>(base);
    s.ml = s.o + ctas * 2 * rows * hd;
    s.join = reinterpret_cast<PagedJoin*>(s.ml + ctas * 2 * rows * 2);
    return s;
}

// How a launch divides its work.
struct PagedTiling {
    int rows;   // rows of a row tile as the kernel holds them (token-major, `group` query heads each)
    int sub;    // rows per independent half, of which floor(sub / group) * group are used
    int tt;     // tokens of a row tile
    int kt;     // positions of a key tile
};

struct PagedOut {
    void* out;
    float* lse;
    float sl2;             // scale * log2(e)
};

// Row r of a row tile is token `tok` of the tile (beyond every sequence: none) and query head `g` of the group,
// whatever the item: the divisions are done once.
struct PagedRow {
    int tok, g;
    __device__ __forceinline__ PagedRow(int r, int sub, int group) {
        const int per = sub / group, half = r / sub, x = r - half * sub;
        const int t = x / group;
        g = x - t * group;
        tok = t < per ? half * per + t : 1 << 30;
    }
    // The row's token in the sequence, or -1.
    __device__ __forceinline__ int token(int rt, int tt, int q_len) const {
        return tok < q_len - rt * tt ? rt * tt + tok : -1;
    }
};

// Two f32 as two 16-bit values of the cache's type, and back.
template <typename T>
struct Pack16;
template <>
struct Pack16<__half> {
    static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
        const __half2 h = __floats2half2_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    static __device__ __forceinline__ float2 unpack(uint32_t v) { return __half22float2(*reinterpret_cast<__half2*>(&v)); }
};
template <>
struct Pack16<__nv_bfloat16> {
    static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    static __device__ __forceinline__ float2 unpack(uint32_t v) {
        return __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&v));
    }
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(map)) : "memory");
}

__device__ __forceinline__ void tma_page(void* smem_dst, const CUtensorMap* map, int col, int row, int head, int page,
                                         uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], "
        "[%6];" ::"r"(smem_u32(smem_dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(col), "r"(row), "r"(head), "r"(page), "r"(smem_u32(bar))
        : "memory");
}

__device__ __forceinline__ float4 ld_dsmem_v4(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                 : "r"(addr)
                 : "memory");
    return v;
}

struct PagedLaunch {
    PagedKv c;
    const void* q;
    int64_t q_stride;
    int64_t max_q;
    PagedOut o;
    PagedTiling tl;
    PagedScratch sc;
};

// The pages as a tensor {head_dim, page, KV heads, pages} with boxes of 64 elements x box_rows positions, each
// box landing as rows of 128 bytes in the 128-byte swizzle (16-bit caches); the queries as {head_dim, query
// heads of a KV head, KV heads, tokens} with boxes of 64 elements x the group x box_tokens.
cudaError_t paged_query_map(CUtensorMap* map, const PagedLaunch& a, int dtype, int hd, int box_tokens);
cudaError_t paged_tensor_map(CUtensorMap* map, const PagedKv& c, const void* pages, int dtype, int hd, int box_rows);

// Raises a kernel's dynamic shared-memory limit once per device.
template <typename Kern>
cudaError_t paged_allow_smem(Kern kern, std::atomic<uint64_t>& flags, int bytes) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    const uint64_t bit = 1ull << (dev & 63);
    if (flags.load() & bit) return cudaSuccess;
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess) flags.fetch_or(bit);
    return e;
}

// A launch of `ctas` CTAs in clusters, with programmatic stream serialization.
template <typename Params>
cudaError_t paged_launch_clusters(void (*kernel)(Params), int ctas, int threads, int smem, int cluster, cudaStream_t s,
                                  const std::remove_const_t<Params>& p) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(ctas));
    cfg.blockDim = dim3(static_cast<unsigned>(threads));
    cfg.dynamicSmemBytes = static_cast<size_t>(smem);
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = static_cast<unsigned>(cluster);
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    g_launches.fetch_add(1, std::memory_order_relaxed);
    return cudaLaunchKernelEx(&cfg, kernel, p);
}

// cluster 0: the line cut into `ctas` pieces; otherwise ctas = items * cluster.
cudaError_t launch_paged_decode(const PagedLaunch& a, int dtype, int hd, int ctas, int cluster, cudaStream_t s);
cudaError_t launch_paged_chunk(const PagedLaunch& a, int dtype, int hd, int ctas, cudaStream_t s);
cudaError_t launch_paged_f32(const PagedLaunch& a, int out_dtype, int hd, int ctas, int cluster, cudaStream_t s);
cudaError_t launch_paged_combine(const PagedLaunch& a, int out_dtype, int hd, int ctas, cudaStream_t s);

}  // namespace sc
