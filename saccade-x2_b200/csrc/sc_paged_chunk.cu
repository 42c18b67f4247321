// sc_paged_chunk.cu -- attention of many new tokens per sequence over the paged cache (16-bit caches): the
// tensor cores' part, tcgen05 with everything between the loads and the output in tensor memory.
//
// A row tile is two halves of 128 rows (tokens x the query heads of one KV head), over key tiles of 128
// positions that both halves share.  Per half and key tile
//   S = Q K^T      tcgen05.mma, Q and K in shared memory (K-major, 128-byte swizzle), S f32 in tensor memory
//   P = 2^(S sl2 - m), m a running reference of the row, rows' sums in f32; P as 16-bit values over S
//   O += P V       tcgen05.mma, P from tensor memory, V in shared memory (its rows are the K dimension: the
//                  N-major operand), O f32 in tensor memory
// 4 * 128 * 128 * hd flops per half against 128 * 128 exponentials: at hd 128 the tensor pipe needs
// 1024 cycles and the special-function units (16 a cycle) 1024 as well, so the two halves run in
// turn: while one half's softmax runs, the tensor cores have the other's products.
//   warps 0-3, 4-7  softmax of half 0, 1: a thread per row (no shuffles)
//   warp 8          loads: Q boxes once per item, K and V boxes (min(page, 128) rows) through a ring
//   warp 9          (10 and 11 idle) issues every tcgen05.mma: PV(j) of a half, then S(j + 1) of it, which may overwrite P(j)
//                   because the tensor pipe keeps the order of one thread's instructions
// The reference m moves only when a row's maximum leaves it by more than a factor that P's type holds
// (2^14 in f16): O is then rescaled in tensor memory, which is rare after the first tiles.
// Pieces of the line of key tiles go to the CTAs evenly (sc_paged.cuh).
// Measured: 4 x 512 new tokens over 7001..8192 positions, bf16, 64 + 8 heads of 128: 464 us at a full clock (1010
// TFLOP/s), 528 to 556 under the power cap (990 W at 1.6 GHz; 840 to 887); 16 prompts of 129..512 tokens, f16, 28 + 4 heads: 71 us.
// What bounds it is each half's chain: softmax 1850 cycles, then P V and the next S 1420 with their hand-overs, 3600
// per pair of tiles where the tensor pipe alone needs 2048 (it is active 51 % of the time, the special-function units
// 51 %).  Its registers spill (472 bytes stored, 436 loaded at head_dim 128).  Tensor memory is full (S and O of two halves), so S cannot run ahead.  Tried on the first case: 16 softmax
// warps of 16 rows each 465 us, the same with S ahead in steps of 64 positions (N = 64 products) 570, a tensor-core warp
// per half and P handed over in two parts 543, the halves' exponentials strictly in turn 521, a quarter of them as
// polynomials on the FMA pipe 10 to 25 us more each time, row sums in place of maxima to tell when a reference
// must move 467.  Prompts spend half their time between items: queries' loads, the first S, the outputs.  Their loop
// unrolled with its loads ahead costs 6 us more; a kernel a third shorter (rolled loops, compact waits) the same or 20 us more
// on the first case.
#include <atomic>
#include <type_traits>

#include "sc_paged.cuh"

namespace sc {

__device__ __forceinline__ void tc_ld32(uint32_t taddr, uint32_t* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,"
        "%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tc_st32(uint32_t taddr, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
        "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
        "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
        "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
        : "memory");
}
// Waits for the loads of `r`, which no use of it may pass.
__device__ __forceinline__ void tc_wait_ld32(uint32_t* r) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]),
                   "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]),
                   "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]),
                   "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
                 :
                 : "memory");
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
__device__ __forceinline__ uint64_t pair(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
// 16 lanes x 32 columns: lane (g, c) = (lane / 4, lane % 4) gets, per 8 columns k, columns 8 k + 2 c and + 1 of TMEM lanes
// g (r[4 k], r[4 k + 1]) and g + 8 (r[4 k + 2], r[4 k + 3]).
__device__ __forceinline__ void tc_ld_16x32(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tc_wait_ld16x2(uint32_t (&a)[16], uint32_t (&b)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(a[0]), "+r"(a[1]), "+r"(a[2]), "+r"(a[3]), "+r"(a[4]), "+r"(a[5]), "+r"(a[6]), "+r"(a[7]), "+r"(a[8]),
                   "+r"(a[9]), "+r"(a[10]), "+r"(a[11]), "+r"(a[12]), "+r"(a[13]), "+r"(a[14]), "+r"(a[15]), "+r"(b[0]),
                   "+r"(b[1]), "+r"(b[2]), "+r"(b[3]), "+r"(b[4]), "+r"(b[5]), "+r"(b[6]), "+r"(b[7]), "+r"(b[8]),
                   "+r"(b[9]), "+r"(b[10]), "+r"(b[11]), "+r"(b[12]), "+r"(b[13]), "+r"(b[14]), "+r"(b[15])
                 :
                 : "memory");
}
// Lane c of each four gives p[k] to lane k and gets p[c] of lane k as p[k].
__device__ __forceinline__ void quad_transpose(uint32_t (&p)[4], int c) {
#pragma unroll
    for (int d = 1; d < 4; d <<= 1)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if (k & d) continue;
            const bool up = c & d;  // keeps p[k + d], gives p[k]
            const uint32_t got = __shfl_xor_sync(0xffffffffu, up ? p[k] : p[k + d], d);
            if (up) p[k] = got;
            else p[k + d] = got;
        }
}
// D[128 x N] (+)= A[128 x 16] * B[16 x N], both operands in shared memory.
__device__ __forceinline__ void tc_mma_ss(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                          uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}
// Descriptors of a [rows][128 bytes] tile in the 128-byte swizzle.  Rows as M or N, the bytes along K: 8-row
// groups 1024 bytes apart (the leading offset is unused).  Rows along K, the bytes as N: groups of 8 K
// rows 1024 bytes apart, blocks of 64 N elements `block` bytes apart.
// `low` is chunk_low() of the tile plus the offset in 16-byte units; the address field does not carry out.
__device__ __forceinline__ uint32_t chunk_low(uint32_t addr, uint32_t block) {
    return ((addr >> 4) & 0x3FFFu) | ((block >> 4) & 0x3FFFu) << 16;
}
__device__ __forceinline__ uint64_t chunk_desc(uint32_t low) {
    constexpr uint32_t kHigh = (1024u >> 4) | (1u << 14) | (2u << 29);  // 8-row stride, sm_100 version, swizzle
    uint64_t d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "r"(low), "r"(kHigh));
    return d;
}

template <int kHd>
struct ChunkCfg {
    static constexpr int kKeys = 128;
    static constexpr int kBlocks = kHd / 64;              // 64-element blocks of a row
    static constexpr int kBlock = 128 * 128;              // bytes of 128 rows of a block
    static constexpr int kTile = kBlocks * kBlock;        // a K or V tile, or a half's Q
    static constexpr int kSlots = kHd == 128 ? 5 : 8;     // ring of K and V tiles in turn
    static constexpr int kThreads = 384;                  // 64,512 registers at launch: 208 for each softmax thread, 88 for the others
    static constexpr int kSmem = 1024 + (2 + kSlots) * kTile;
    static constexpr uint32_t kS = 0, kO = 256;           // tensor memory columns: S of half 1 at 128, O at 384
};

struct alignas(64) ChunkParams {
    CUtensorMap kmap, vmap, qmap;
    PagedLaunch a;
    int box_shift;     // log2 of the rows of a K or V box
};

template <typename T, int kHd>
__global__ void __launch_bounds__(384, 1) k_paged_chunk(const __grid_constant__ ChunkParams P) {
    using C = ChunkCfg<kHd>;
    using M = Pack16<T>;
    constexpr bool kF16 = std::is_same<T, __half>::value;
    extern __shared__ unsigned char smem_raw[];
    __shared__ __align__(8) uint64_t q_full, q_empty, kv_full[C::kSlots], kv_empty[C::kSlots], s_full[2], p_full[2],
        o_full[2], done;
    __shared__ uint32_t tmem_slot;
    __shared__ PagedCut cut;
    __shared__ int s_not_finite;  // a new token's value that is not has been met
    unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    unsigned char* ring = smem + 2 * C::kTile;
    const PagedLaunch& A = P.a;
    const PagedKv& kv = A.c;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int G = kv.nh / kv.nkv, per = 128 / G, tt = 2 * per;
    if (tid == 0) {
        mbar_init(&q_full, 1);
        mbar_init(&q_empty, 1);
        for (int i = 0; i < C::kSlots; ++i) {
            mbar_init(&kv_full[i], 1);
            mbar_init(&kv_empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&s_full[i], 1);
            mbar_init(&p_full[i], 4);
            mbar_init(&o_full[i], 1);
        }
        mbar_init(&done, 1);
        fence_mbar_init();
        s_not_finite = 0;
    }
    if (tid == 32 * 8) {
        prefetch_map(&P.qmap);
        prefetch_map(&P.kmap);
        prefetch_map(&P.vmap);
    }
    if (warp == 9) {
        tmem_alloc(&tmem_slot, 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;
    pdl_launch_dependents();
    pdl_wait();
    paged_cut<C::kThreads>(kv, A.max_q, tt, C::kKeys, &cut);  // synchronises the block
    PagedWalk w;
    w.begin(cut, tt);

    if (warp < 8) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
        // ---------------- softmax: warps 0-3 half 0, 4-7 half 1; thread = row
        const int half = warp >> 2, row = tid & 127;
        const uint32_t lanes = static_cast<uint32_t>(32 * (warp & 3)) << 16;
        const uint32_t ts = tmem + lanes + C::kS + half * 128, to = tmem + lanes + C::kO + half * 128;
        // f16: a new reference makes the largest weight 2^6, so that its steps of 2^-24 are 2^-30 of the largest, and
        // weights may grow to 2^14 (bf16: 2^40) before it moves.  2^10 and 2^15, for steps of 2^-34, move more often: f16
        // 4 x 512 new tokens over 8192 positions 542 us against 463, 16 prompts 79 against 73.
        constexpr float kShift = kF16 ? 6.0f : 0.0f;
        constexpr float kMove = kF16 ? 14.0f : 40.0f;
        const float sl2 = A.o.sl2;
        int it = 0;              // ring tiles, as the loads count them
        uint32_t count = 0, items = 0;
        bool ok = true;
        const PagedRow mine(half * 128 + row, 128, G);
        PagedJoin join{0, 0, 0, 0, 0};
        PagedWalk wn = w;
        bool more = wn.next(kv, A.max_q, tt, C::kKeys);
        while (ok && more) {
            w = wn;
            const int n = w.t1 - w.t0;
            const bool two = w.rt * tt + per < w.s.q_len;
            if (!w.whole() && w.t0 == 0)
                join = PagedJoin{w.s.row0, w.s.q_len, w.h, w.rt, w.pieces(cut)};
            if (half == 1 && !two) {
                it += 2 * n;
                // a cut item's second half is empty: its rows are never joined
                more = wn.next(kv, A.max_q, tt, C::kKeys);
                continue;
            }
            const int tok = mine.token(w.rt, tt, w.s.q_len);
            const int start = w.s.kv_len - w.s.q_len;
            const int first_pos = start + w.rt * tt + half * per;  // the least position of the half's rows
            const int keys = start + min((w.rt + 1) * tt, w.s.q_len);
            const int pos = tok >= 0 ? start + tok : keys - 1;  // (a row of no token: as little masked as any)
            float m = -INFINITY, l = 0.0f;
            for (int j = 0; j < n; ++j, ++count) {
                const int k0 = (w.t0 + j) * C::kKeys;
                if (half == 0 && k0 + C::kKeys > first_pos + 1) {
                    // V rows behind the item's last position hold whatever was there: 0 * NaN must not be.  Nor must it
                    // for the new tokens that only some of the rows attend: their values are looked over.
                    const int vt = it + 2 * j + 1, none = max(0, keys - k0);
                    ok = ok && __all_sync(0xffffffffu, mbar_wait(&kv_full[vt % C::kSlots], (vt / C::kSlots) & 1, kv.status));
                    unsigned char* vb = ring + (vt % C::kSlots) * C::kTile;
                    for (int i = max(0, first_pos + 1 - k0) * 8 + row; i < 128 * 8; i += 128) {
                        // (a row of 128 bytes: eight lanes)
                        bool bad = false;
#pragma unroll
                        for (int b = 0; b < C::kBlocks; ++b) {
                            uint4* at = reinterpret_cast<uint4*>(vb + b * C::kBlock + i * 16);
                            if (i >= none * 8) {
                                *at = make_uint4(0, 0, 0, 0);
                            } else {
                                uint4 v = *at;
                                if (finite_only<T>(v)) {
                                    *at = v;
                                    bad = true;
                                }
                            }
                        }
                        if (bad) s_not_finite = 1;
                    }
                    fence_proxy_async_smem();
                }
                ok = ok && __all_sync(0xffffffffu, mbar_wait(&s_full[half], count & 1, kv.status));
                if (!ok) break;
                tc_fence_after();
                const bool edge = k0 + C::kKeys > first_pos + 1;
                const int lim = pos - k0;  // columns up to it are attended
                auto mask = [&](uint32_t* v, int c) {
                    if (edge && !__all_sync(0xffffffffu, lim >= 32 * c + 31)) {
                        const int x = lim - 32 * c;
                        const uint32_t live = x >= 31 ? 0xFFFFFFFFu : x < 0 ? 0u : (2u << x) - 1u;
#pragma unroll
                        for (int i = 0; i < 32; ++i)
                            if (!(live & (1u << i))) v[i] = 0xFF800000u;  // -inf
                    }
                };
                // P against the reference as it is, and the row's maximum beside it, 32 columns at a time while the
                // next 32 are loaded.  A row without a reference takes the first columns' maximum for one; a row that
                // has left its reference too far takes its own maximum, and P is computed once more.
                uint32_t pk[64];
                float part[2];
                for (;;) {
                    const uint64_t sl = pair(sl2, sl2);
                    uint64_t mm = 0, sum[2] = {0, 0};
                    float mx[2] = {-INFINITY, -INFINITY};
                    uint32_t v[2][32];
                    tc_ld32(ts, v[0]);
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        uint32_t* x = v[c & 1];
                        tc_wait_ld32(x);
                        if (c < 3) tc_ld32(ts + 32 * (c + 1), v[(c + 1) & 1]);
                        mask(x, c);
#pragma unroll
                        for (int i = 0; i < 16; ++i)
                            mx[i & 1] = max3(mx[i & 1], __uint_as_float(x[2 * i]), __uint_as_float(x[2 * i + 1]));
                        if (c == 0) {
                            if (m == -INFINITY) m = fmaxf(mx[0], mx[1]) * sl2 - kShift;
                            const float ms = m == -INFINITY ? 0.0f : m;
                            mm = pair(-ms, -ms);
                        }
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            uint64_t t;
                            asm("fma.rn.f32x2 %0, %1, %2, %3;"
                                : "=l"(t)
                                : "l"(pair(__uint_as_float(x[2 * i]), __uint_as_float(x[2 * i + 1]))), "l"(sl), "l"(mm));
                            float e0, e1;
                            asm("mov.b64 {%0, %1}, %2;" : "=f"(e0), "=f"(e1) : "l"(t));
                            e0 = ex2(e0);
                            e1 = ex2(e1);
                            asm("add.rn.f32x2 %0, %0, %1;" : "+l"(sum[i & 1]) : "l"(pair(e0, e1)));
                            pk[16 * c + i] = M::pack(e0, e1);
                        }
                    }
                    asm("add.rn.f32x2 %0, %0, %1;" : "+l"(sum[0]) : "l"(sum[1]));
                    asm("mov.b64 {%0, %1}, %2;" : "=f"(part[0]), "=f"(part[1]) : "l"(sum[0]));
                    const float top = fmaxf(mx[0], mx[1]) * sl2;
                    const bool move = top > m + kMove;
                    if (!__any_sync(0xffffffffu, move)) break;
                    const float mn = move ? top - kShift : m;  // each row by itself
                    const float f = mn == -INFINITY ? 1.0f : ex2(m - mn);
                    l *= f;
                    m = mn;
                    if (j > 0) {
#pragma unroll 1
                        for (int c = 0; c < kHd; c += 32) {
                            uint32_t o[32];
                            tc_ld32(to + c, o);
                            tc_wait_ld32(o);
#pragma unroll
                            for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
                            tc_st32(to + c, o);
                        }
                    }
                }
                l += part[0] + part[1];
                tc_st32(ts, pk);
                tc_st32(ts + 32, pk + 32);
                tc_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&p_full[half]);
            }
            it += 2 * n;
            more = wn.next(kv, A.max_q, tt, C::kKeys);  // while the last product ends
            ok = ok && __all_sync(0xffffffffu, mbar_wait(&o_full[half], items & 1, kv.status));
            if (!ok) break;
            tc_fence_after();
            const bool whole = w.whole();
            const int orow = tok < 0 ? -1 : static_cast<int>((w.s.row0 + tok) * kv.nh) + w.h * G + mine.g;
            const int64_t slot_row = (static_cast<int64_t>(blockIdx.x) * 2 + w.slot()) * 256 + half * 128 + 32 * (warp & 3);
            const float inv = l > 0.0f ? 1.0f / l : 0.0f;
            // 16 rows x 32 columns at a time, four lanes to a row (a lane per row would touch 32 lines with
            // every store): lane (g4, c4) has columns 8 k + 2 c4 .. + 1 of rows g4 and g4 + 8
            const int g4 = lane >> 2, c4 = lane & 3;
            int orows[4];
            float invs[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                orows[i] = __shfl_sync(0xffffffffu, orow, 8 * i + g4);
                invs[i] = __shfl_sync(0xffffffffu, inv, 8 * i + g4);
            }
            // (rolled: what runs once per item should not push the softmax out of the instruction cache)
#pragma unroll 1
            for (int c = 0; c < kHd; c += 32) {
                uint32_t o[2][16];
                tc_ld_16x32(to + c, o[0]);
                tc_ld_16x32(to + (16u << 16) + c, o[1]);
                tc_wait_ld16x2(o[0], o[1]);
                if (whole) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {  // rows g4 + 8 i
                        const uint32_t* x = o[i >> 1] + 2 * (i & 1);
                        uint32_t p[4];
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            p[k] = M::pack(__uint_as_float(x[4 * k]) * invs[i], __uint_as_float(x[4 * k + 1]) * invs[i]);
                        quad_transpose(p, c4);  // lane c4 now has columns 8 c4 .. + 7
                        if (orows[i] >= 0)
                            *reinterpret_cast<uint4*>(static_cast<T*>(A.o.out) + static_cast<int64_t>(orows[i]) * kHd + c +
                                                      8 * c4) = make_uint4(p[0], p[1], p[2], p[3]);
                    }
                } else {
                    float* dst = A.sc.o + (slot_row + g4) * kHd + c + 2 * c4;
#pragma unroll
                    for (int i = 0; i < 4; ++i)
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            if (orows[i] >= 0)
                                *reinterpret_cast<uint2*>(dst + 8 * i * kHd + 8 * k) =
                                    make_uint2(o[i >> 1][4 * k + 2 * (i & 1)], o[i >> 1][4 * k + 2 * (i & 1) + 1]);
                }
            }
            tc_fence_before();
            if (tok >= 0) {
                if (!whole) *reinterpret_cast<float2*>(A.sc.ml + (slot_row + lane) * 2) = make_float2(m, l);
                else if (A.o.lse) A.o.lse[orow] = l == 0.0f ? -INFINITY : (m + log2f(l)) * 0.69314718055994531f;
            }
            if (__any_sync(0xffffffffu, *const_cast<volatile int*>(&s_not_finite) != 0)) {  // rare
                __syncwarp();  // the row's stores by the other lanes
                const int from = max(start + w.rt * tt + 1, w.t0 * C::kKeys), to = min(pos, w.t1 * C::kKeys - 1);
                if (tok >= 0 && whole)
                    paged_add_not_finite<T, kHd, 4>(kv, w.b, w.h, from, to, 0, static_cast<T*>(A.o.out) + static_cast<int64_t>(orow) * kHd);
                else if (tok >= 0)
                    paged_add_not_finite<T, kHd, 4>(kv, w.b, w.h, from, to, 0, A.sc.o + (slot_row + lane) * kHd);
                __syncwarp();
            }
            ++items;
        }
        if (tid == 0) A.sc.join[blockIdx.x] = join;
        __syncwarp();
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
        if (warp == 8) {
            // ---------------- loads: the whole warp, a box per lane
            int it = 0, item = 0, issued = 0, queries = 0;  // ring tiles (K and V count), items, loads of each
            bool stop = false;
            while (!stop && w.next(kv, A.max_q, tt, C::kKeys)) {
                const int shift = kv.page_shift, bs = P.box_shift;
                const int keys = w.s.kv_len - w.s.q_len + min((w.rt + 1) * tt, w.s.q_len);
                const int32_t* table = kv.table + w.b * kv.max_pages;
                int have = -1, id = 0;  // pages have .. have + 31 of the sequence, one per lane
                auto load_q = [&]() {
                    const bool two = w.rt * tt + per < w.s.q_len;
                    const int parts = (two ? 2 : 1) * C::kBlocks;
                    if (lane == 0) mbar_arrive_expect_tx(&q_full, static_cast<uint32_t>(parts) * G * per * 128u);
                    __syncwarp();
                    if (lane < parts) {
                        const int half = lane / C::kBlocks, blk = lane % C::kBlocks;
                        tma_page(smem + half * C::kTile + blk * C::kBlock, &P.qmap, blk * 64, 0, w.h,
                                 static_cast<int>(w.s.row0) + w.rt * tt + half * per, &q_full);
                    }
                    ++queries;
                };
                if (item == 0) load_q();
                for (int t = w.t0; t < w.t1 && !stop; ++t) {
                    const int k0 = t * C::kKeys, n = max(0, min(C::kKeys, keys - k0));
                    const int boxes = (n + (1 << bs) - 1) >> bs;
                    const int p0 = k0 >> shift, p1 = n > 0 ? (k0 + n - 1) >> shift : p0;
                    if (n > 0 && (have < 0 || p0 < have || p1 >= have + 32)) {
                        have = p0;
                        id = static_cast<int>(kv.num_pages);
                        if (p0 + lane <= (keys - 1) >> shift) {
                            id = table[p0 + lane];
                            if (id < 0 || id >= kv.num_pages) {
                                record_error(kv.status, DEV_BAD_INDEX);
                                id = static_cast<int>(kv.num_pages);  // outside the map: zeros are loaded
                            }
                        }
                    }
                    for (int v = 0; v < 2; ++v, ++it) {  // K, then V
                        const int sl = it % C::kSlots;
                        if (it >= C::kSlots && !mbar_wait(&kv_empty[sl], ((it / C::kSlots) - 1) & 1, kv.status)) stop = true;
                        if (__any_sync(0xffffffffu, stop)) {
                            stop = true;
                            break;
                        }
                        if (lane == 0)
                            mbar_arrive_expect_tx(&kv_full[sl], static_cast<uint32_t>(boxes) * C::kBlocks * (128u << bs));
                        __syncwarp();
                        ++issued;
                        unsigned char* dst = ring + sl * C::kTile;
                        for (int i0 = 0; i0 < boxes * C::kBlocks; i0 += 32) {
                            const int i = i0 + lane, box = i / C::kBlocks, blk = i % C::kBlocks;
                            const int key = k0 + (box << bs);
                            const int page = __shfl_sync(0xffffffffu, id, ((key >> shift) - have) & 31);
                            if (i < boxes * C::kBlocks)
                                tma_page(dst + blk * C::kBlock + (box << bs) * 128, v ? &P.vmap : &P.kmap, blk * 64,
                                         key & ((1 << shift) - 1), w.h, page, &kv_full[sl]);
                        }
                    }
                    if (t == w.t0 && item > 0 && !stop) {
                        // the item's queries, after its first keys: the item before may still be read
                        if (!mbar_wait(&q_empty, (item - 1) & 1, kv.status)) stop = true;
                        stop = __any_sync(0xffffffffu, stop);
                        if (!stop) load_q();
                    }
                }
                ++item;
            }

            // copies in flight end before the block does
            if (lane == 0) {
                for (int i = issued > C::kSlots ? issued - C::kSlots : 0; i < issued; ++i)
                    mbar_wait(&kv_full[i % C::kSlots], (i / C::kSlots) & 1, nullptr, kDrainNs);
                if (queries > 0) mbar_wait(&q_full, (queries - 1) & 1, nullptr, kDrainNs);
            }
            __syncwarp();
        } else if (warp == 9) {
            // ---------------- tensor cores
            const uint32_t fmt = kF16 ? 0u : (1u << 7) | (1u << 10);  // bf16 operands
            const uint32_t idesc_s = idesc_f16_f32(128, 128) | fmt;
            const uint32_t idesc_o = idesc_f16_f32(128, kHd) | fmt | (1u << 16);  // V: N-major
            const uint32_t qa = smem_u32(smem), ra = smem_u32(ring);
            int it = 0, item = 0;
            uint32_t pcount[2] = {0, 0};  // P tiles taken, per half
            bool ok = true;
            auto wait = [&](uint64_t* bar, uint32_t parity) {
                ok = ok && __all_sync(0xffffffffu, mbar_wait(bar, parity, kv.status));
                return ok;
            };
            auto issue_s = [&](int half, int tile) {  // S of `half` from ring tile `tile`
                const uint32_t a = chunk_low(qa + half * C::kTile, 16), b = chunk_low(ra + (tile % C::kSlots) * C::kTile, 16);
    #pragma unroll 4
                for (int k = 0; k < kHd / 16; ++k) {
                    const uint32_t off = ((k >> 2) * C::kBlock + (k & 3) * 32) >> 4;
                    tc_mma_ss(tmem + C::kS + half * 128, chunk_desc(a + off), chunk_desc(b + off), idesc_s, k ? 1u : 0u);
                }
                tc_commit(&s_full[half]);
            };
            while (ok && w.next(kv, A.max_q, tt, C::kKeys)) {
                const int n = w.t1 - w.t0;
                const bool two = w.rt * tt + per < w.s.q_len;
                if (!wait(&kv_full[it % C::kSlots], (it / C::kSlots) & 1) || !wait(&q_full, item & 1)) break;
                tc_fence_after();
                if (elect_one()) {
                    issue_s(0, it);
                    if (two) issue_s(1, it);
                    tc_commit(&kv_empty[it % C::kSlots]);
                    if (n == 1) tc_commit(&q_empty);
                }
                __syncwarp();
                for (int j = 0; j < n && ok; ++j) {
                    const int vt = it + 2 * j + 1, kt = vt + 1;  // ring tiles of V(j) and K(j + 1)
                    if (!wait(&kv_full[vt % C::kSlots], (vt / C::kSlots) & 1)) break;
                    if (j + 1 < n && !wait(&kv_full[kt % C::kSlots], (kt / C::kSlots) & 1)) break;
                    for (int half = 0; half < (two ? 2 : 1); ++half) {
                        if (!wait(&p_full[half], pcount[half] & 1)) break;
                        ++pcount[half];
                            tc_fence_after();
                        const bool end = half == (two ? 1 : 0);
                        if (elect_one()) {
                            const uint32_t b = chunk_low(ra + (vt % C::kSlots) * C::kTile, C::kBlock);
    #pragma unroll 4
                            for (int k = 0; k < C::kKeys / 16; ++k)
                                tc_mma_ts(tmem + C::kO + half * 128, tmem + C::kS + half * 128 + k * 8,
                                          chunk_desc(b + k * (2048 >> 4)), idesc_o, (j | k) ? 1u : 0u);
                            if (end) tc_commit(&kv_empty[vt % C::kSlots]);
                            if (j + 1 < n) {
                                issue_s(half, kt);
                                if (end) {
                                    tc_commit(&kv_empty[kt % C::kSlots]);
                                    if (j + 2 == n) tc_commit(&q_empty);
                                }
                            } else {
                                tc_commit(&o_full[half]);
                            }
                        }
                        __syncwarp();
                    }
                }
                it += 2 * n;
                ++item;
            }
            if (elect_one()) tc_commit(&done);
            __syncwarp();
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 9) {
        mbar_wait(&done, 0, nullptr, kDrainNs);  // every product has ended (at once, but after a wait that ran out)
        tc_fence_after();
        __syncwarp();
        tmem_dealloc(tmem, 512);
    }
}

template <typename T, int kHd>
static cudaError_t launch_chunk_t(const ChunkParams& p, int ctas, cudaStream_t s) {
    using C = ChunkCfg<kHd>;
    static std::atomic<uint64_t> flags{0};
    cudaError_t e = paged_allow_smem(k_paged_chunk<T, kHd>, flags, C::kSmem);
    if (e != cudaSuccess) return e;
    return launch_pdl(k_paged_chunk<T, kHd>, dim3(static_cast<unsigned>(ctas)), dim3(C::kThreads), C::kSmem, s, p);
}

cudaError_t launch_paged_chunk(const PagedLaunch& a, int dtype, int hd, int ctas, cudaStream_t s) {
    ChunkParams p;
    p.a = a;
    p.box_shift = a.c.page_shift < 7 ? a.c.page_shift : 7;
    const int G = a.c.nh / a.c.nkv;
    cudaError_t e = paged_tensor_map(&p.kmap, a.c, a.c.k, dtype, hd, 1 << p.box_shift);
    if (e == cudaSuccess) e = paged_tensor_map(&p.vmap, a.c, a.c.v, dtype, hd, 1 << p.box_shift);
    if (e == cudaSuccess) e = paged_query_map(&p.qmap, a, dtype, hd, 128 / G);
    if (e != cudaSuccess) return e;
    if (dtype == SC_F16)
        return hd == 128 ? launch_chunk_t<__half, 128>(p, ctas, s) : launch_chunk_t<__half, 64>(p, ctas, s);
    return hd == 128 ? launch_chunk_t<__nv_bfloat16, 128>(p, ctas, s) : launch_chunk_t<__nv_bfloat16, 64>(p, ctas, s);
}

}  // namespace sc
