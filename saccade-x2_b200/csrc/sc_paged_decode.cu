// sc_paged_decode.cu -- attention of few new tokens per sequence over the paged cache (16-bit caches).
//
// Up to 16 rows (new tokens x query heads of one KV head) share each key and value that is loaded:
// 4 * 16 flops at most per 2 bytes, so the cache's bytes bound it and the tensor work (mma.sync
// m16n8k16, under a tenth of its rate) does not.  What counts is that the loads never stop:
//   producer warp   per key tile of 64 positions, boxes of K and V (min(page, 64) rows x 64 elements,
//                   128-byte swizzle) by TMA into a ring of stages, two CTAs per SM: ~190 KB in flight
//   4 warps         each takes 16 of the tile's 64 positions with a running maximum and sum of its own,
//                   so no warp waits for another until the item ends: S = Q K^T (registers), weights
//                   p = 2^(s scale log2 e - m) <= 1 in f32, split into a high and a low 16-bit part at no time that
//                   shows, O += P V.  bf16's parts have 16 bits of p.  f16's are those of 2^15 p, so that its short
//                   exponent range lies below the largest weight: 22 bits down to p = 2^-18, below that steps of
//                   2^-39 (unscaled, weights under 2^-25 were lost, and thousands of them add up); the factor is
//                   exact and leaves O again where the warps are joined
//   item end        the 4 warps' maxima, sums and outputs are joined through shared memory.
// Long sequences: the work is cut evenly over the CTAs along the positions (sc_paged.cuh) and the pieces are joined
// by a second kernel.  Where no CTA's share can pass kClusterKeys positions, finding the cut and that kernel
// cost more than they even out: each (sequence, KV head) then goes to a cluster of 1 to 8 CTAs, as many as keep the
// launch within one wave, which divide its tiles and join them through distributed shared memory.
// Measured, f16, 28 + 4 heads of 128: one sequence of 640 positions 10.0 us cut, 5.9 us in clusters of 8; 64 of
// 513..768 26.0 and 19.4 us (4.4 TB/s); one of 8192 18.7 and 14.3, of 16384 23.9 and 24.4, of 30000 29.4 and 41.2;
// 200 of 2048 139 and 126.  8 of 20001..32768, 64 + 8 heads, bf16, cut: 143 us (6.2 TB/s, 0.96 of a copy).
#include <atomic>
#include <type_traits>

#include "sc_paged.cuh"

namespace sc {

__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}

template <typename T>
__device__ __forceinline__ void mma_16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma_16<__half>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    mma_16816(d, a, b0, b1);
}
template <>
__device__ __forceinline__ void mma_16<__nv_bfloat16>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <int kHd>
struct DecCfg {
    static constexpr int kKeys = 64;                            // positions of a stage
    static constexpr int kTile = kKeys * kHd * 2;               // bytes of its K (or V)
    static constexpr int kStages = kHd == 128 ? 3 : 6;
    static constexpr int kWarps = 4;
    static constexpr int kThreads = (kWarps + 1) * 32;
    static constexpr int kJoinDims = 32;                        // output columns joined at a time
    static constexpr int kSmem = 1024 + kStages * 2 * kTile + kWarps * 16 * kJoinDims * 4;
};

struct alignas(64) DecodeParams {
    CUtensorMap kmap, vmap;
    PagedLaunch a;
    int box_shift;         // log2 of the rows of a box
    int cluster;           // CTAs of an item (the clustered kernel)
};

template <typename T, int kHd, bool kCluster>
__global__ void __launch_bounds__(DecCfg<kHd>::kThreads, 2) k_paged_decode(const __grid_constant__ DecodeParams P) {
    using C = DecCfg<kHd>;
    using M = Pack16<T>;
    constexpr int kSteps = kHd / 16, kBlocks = kHd / 64;
    constexpr float kScale = std::is_same<T, __half>::value ? 32768.0f : 1.0f;  // of the weights in O
    extern __shared__ unsigned char smem_raw[];
    __shared__ __align__(8) uint64_t full[C::kStages], empty[C::kStages];
    __shared__ float s_m[C::kWarps][16], s_l[C::kWarps][16];
    __shared__ float s_ml[16][2];
    __shared__ PagedCut cut;
    unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    float* s_o = reinterpret_cast<float*>(smem + C::kStages * 2 * C::kTile);  // [warp][16][kJoinDims]
    const PagedLaunch& A = P.a;
    const PagedKv& kv = A.c;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int G = kv.nh / kv.nkv, tt = A.tl.tt;
    if (tid == 32 * C::kWarps) {
        prefetch_map(&P.kmap);
        prefetch_map(&P.vmap);
    }
    if (tid == 0) {
        for (int i = 0; i < C::kStages; ++i) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], C::kWarps);
        }
        fence_mbar_init();
    }
    pdl_launch_dependents();
    pdl_wait();
    PagedWalk w;
    const int cs = kCluster ? P.cluster : 1, rank = kCluster ? static_cast<int>(blockIdx.x) % cs : 0;
    if constexpr (kCluster) {
        const int item = static_cast<int>(blockIdx.x) / cs;
        w.b = item / kv.nkv;
        w.h = item - w.b * kv.nkv;
        w.rt = 0;
        w.s = paged_seq(kv, w.b, A.max_q);
        if (w.s.q_len == 0) return;  // the whole cluster
        w.tiles = paged_key_tiles(w.s, 0, tt, C::kKeys);
        w.t0 = w.tiles * rank / cs;
        w.t1 = w.tiles * (rank + 1) / cs;
        __syncthreads();  // the barriers are there
    } else {
        paged_cut<C::kThreads>(kv, A.max_q, tt, C::kKeys, &cut);  // synchronises the block
        w.begin(cut, tt);
    }
    bool item_left = true;  // a cluster's CTA has one item
    auto next_item = [&]() {
        if constexpr (kCluster) {
            const bool r = item_left;
            item_left = false;
            return r;
        } else {
            return w.next(kv, A.max_q, tt, C::kKeys);
        }
    };

    if (warp == C::kWarps) {
        // ---- producer: the whole warp, a box per lane
        int it = 0, issued = 0;
        while (next_item()) {
            const int page_shift = kv.page_shift, bs = P.box_shift;
            const int last = min((w.rt + 1) * tt, w.s.q_len);
            const int keys = w.s.kv_len - w.s.q_len + last;  // positions the item's rows attend
            const int32_t* table = kv.table + w.b * kv.max_pages;
            int have = -1, id = 0;  // pages have .. have + 31 of the sequence, one per lane
            bool stop = false;
            for (int t = w.t0; t < w.t1; ++t, ++it) {
                const int st = it % C::kStages;
                const int k0 = t * C::kKeys, n = max(0, min(C::kKeys, keys - k0));
                const int boxes = (n + (1 << bs) - 1) >> bs;
                const int p0 = k0 >> page_shift, p1 = n > 0 ? (k0 + n - 1) >> page_shift : p0;
                if (n > 0 && (have < 0 || p0 < have || p1 >= have + 32)) {
                    have = p0;
                    id = -2;
                    if (p0 + lane <= (keys - 1) >> page_shift) {
                        id = table[p0 + lane];
                        if (id < 0 || id >= kv.num_pages) {
                            record_error(kv.status, DEV_BAD_INDEX);
                            id = static_cast<int>(kv.num_pages);  // outside the map: zeros are loaded
                        }
                    }
                }
                if (it >= C::kStages && !mbar_wait(&empty[st], ((it / C::kStages) - 1) & 1, kv.status)) stop = true;
                if (__any_sync(0xffffffffu, stop)) {
                    stop = true;
                    break;
                }
                const uint32_t box_bytes = 128u << bs;
                if (lane == 0)
                    mbar_arrive_expect_tx(&full[st], static_cast<uint32_t>(boxes) * kBlocks * 2u * box_bytes);
                __syncwarp();
                ++issued;
                unsigned char* kd = smem + st * 2 * C::kTile;
                for (int i0 = 0; i0 < boxes * kBlocks * 2; i0 += 32) {
                    const int i = i0 + lane;
                    const int box = i / (kBlocks * 2), part = i % (kBlocks * 2);  // part: K blocks, then V blocks
                    const int key = k0 + (box << bs);
                    const int page = __shfl_sync(0xffffffffu, id, ((key >> page_shift) - have) & 31);
                    if (i < boxes * kBlocks * 2) {
                        const int blk = part % kBlocks;
                        const bool v = part >= kBlocks;
                        tma_page(kd + (v ? C::kTile : 0) + blk * C::kKeys * 128 + (box << bs) * 128, v ? &P.vmap : &P.kmap,
                                 blk * 64, key & ((1 << page_shift) - 1), w.h, page, &full[st]);
                    }
                }
            }
            if (stop) break;
        }
        // copies in flight end before the block does
        if (lane == 0)
            for (int i = issued > C::kStages ? issued - C::kStages : 0; i < issued; ++i)
                mbar_wait(&full[i % C::kStages], (i / C::kStages) & 1, nullptr, kDrainNs);
        __syncwarp();
        if (kCluster && cs > 1) {  // with the consumers' two
            cluster_sync();
            cluster_sync();
        }
        return;
    }

    // ---- consumers
    const int g4 = lane >> 2, c4 = lane & 3;
    const uint32_t ring = smem_u32(smem);
    // ldmatrix rows: K matrices (keys 0-7, dims 0-7), (0-7, 8-15), (8-15, 0-7), (8-15, 8-15);
    // V matrices (keys 0-7, dims 0-7), (8-15, 0-7), (0-7, 8-15), (8-15, 8-15)
    const int kkey = 16 * warp + (lane >> 4) * 8 + (lane & 7), kchunk = (lane >> 3) & 1;
    const int vkey = 16 * warp + ((lane >> 3) & 1) * 8 + (lane & 7), vchunk = lane >> 4;
    const PagedRow rows[2] = {PagedRow(g4, 16, G), PagedRow(g4 + 8, 16, G)}, written(tid >> 3, 16, G);
    PagedJoin join{0, 0, 0, 0, 0};
    int it = 0;
    bool late = false;
    while (next_item()) {
        // this thread's two rows
        int tok[2];
        uint32_t qa[kSteps][4];
        int pos[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            tok[r] = rows[r].token(w.rt, tt, w.s.q_len);
            pos[r] = tok[r] >= 0 ? w.s.kv_len - w.s.q_len + tok[r] : -1;
            const T* src = static_cast<const T*>(A.q) + (w.s.row0 + (tok[r] < 0 ? 0 : tok[r])) * A.q_stride +
                           (w.h * G + rows[r].g) * kHd + 2 * c4;
#pragma unroll
            for (int k = 0; k < kSteps; ++k)
#pragma unroll
                for (int x = 0; x < 2; ++x)
                    qa[k][r + 2 * x] =
                        tok[r] >= 0 ? *reinterpret_cast<const uint32_t*>(src + 16 * k + 8 * x) : 0u;
        }
        const int first_pos = w.s.kv_len - w.s.q_len + w.rt * tt;  // the least position of the item's rows
        const int keys = w.s.kv_len - w.s.q_len + min((w.rt + 1) * tt, w.s.q_len);
        float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
        bool bad = false;  // has met a new token's value that is not finite
        float o[kHd / 8][4];
#pragma unroll
        for (int i = 0; i < kHd / 8; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) o[i][j] = 0.0f;
        for (int t = w.t0; t < w.t1; ++t, ++it) {
            const int st = it % C::kStages;
            // after a wait that ran out (recorded in the status) nothing is waited for any more
            if (!late && !mbar_wait(&full[st], (it / C::kStages) & 1, kv.status)) late = true;
            const uint32_t kb = ring + st * 2 * C::kTile, vb = kb + C::kTile;
            float s[2][4] = {};
#pragma unroll
            for (int k = 0; k < kSteps; ++k) {
                uint32_t b[4];
                const int ch = 2 * (k & 3) + kchunk;
                ldsm4(kb + (k >> 2) * (C::kKeys * 128) + kkey * 128 + ((ch ^ (kkey & 7)) << 4), b);
                mma_16<T>(s[0], qa[k], b[0], b[1]);
                mma_16<T>(s[1], qa[k], b[2], b[3]);
            }
            const int j0 = t * C::kKeys + 16 * warp + 2 * c4;  // this thread's keys: j0 + {0, 1, 8, 9}
            const bool edge = (t + 1) * C::kKeys > first_pos + 1;
            float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    float v = s[n][x] * A.o.sl2;
                    if (edge && j0 + 8 * n + (x & 1) > pos[x >> 1]) v = -INFINITY;
                    s[n][x] = v;
                    mx[x >> 1] = fmaxf(mx[x >> 1], v);
                }
            float f[2];
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 1));
                mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 2));
                const float mn = fmaxf(m[r], mx[r]);
                f[r] = mn == -INFINITY ? 1.0f : ex2(m[r] - mn);
                m[r] = mn;
            }
            uint32_t ph[4], pl[4];
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const float ms = m[r] == -INFINITY ? 0.0f : m[r];
                l[r] *= f[r];
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    const float p0 = ex2(s[n][2 * r] - ms), p1 = ex2(s[n][2 * r + 1] - ms);
                    l[r] += p0 + p1;
                    const uint32_t h = M::pack(p0 * kScale, p1 * kScale);
                    const float2 u = M::unpack(h);
                    ph[r + 2 * n] = h;
                    pl[r + 2 * n] = M::pack(p0 * kScale - u.x, p1 * kScale - u.y);
                }
            }
            if (__any_sync(0xffffffffu, f[0] != 1.0f || f[1] != 1.0f)) {
#pragma unroll
                for (int i = 0; i < kHd / 8; ++i) {
                    o[i][0] *= f[0];
                    o[i][1] *= f[0];
                    o[i][2] *= f[1];
                    o[i][3] *= f[1];
                }
            }
            if (w.s.q_len > 1 && edge) {
                // this warp's positions among the new tokens behind the first row's: only some rows attend them
                const int from = max(first_pos + 1, t * C::kKeys + 16 * warp), to = min(keys, t * C::kKeys + 16 * warp + 16);
                for (int i = from * 8 + lane; i < to * 8; i += 32) {
                    const int r = (i >> 3) - t * C::kKeys;
#pragma unroll
                    for (int blk = 0; blk < kBlocks; ++blk) {
                        uint4* at = reinterpret_cast<uint4*>(smem + st * 2 * C::kTile + C::kTile + blk * (C::kKeys * 128) + r * 128 +
                                                             (i & 7) * 16);
                        uint4 v = *at;
                        if (finite_only<T>(v)) {
                            *at = v;
                            bad = true;
                        }
                    }
                }
                fence_proxy_async_smem();  // before the stage is loaded again
                __syncwarp();
            }
            // positions behind the item's last key hold whatever the page or the ring held: no 0 * NaN
            uint32_t va = 0xFFFFFFFFu, vz = 0xFFFFFFFFu;
            const bool tail = (t + 1) * C::kKeys > keys;
            if (tail) {
                va = (j0 < keys ? 0xFFFFu : 0u) | (j0 + 1 < keys ? 0xFFFF0000u : 0u);
                vz = (j0 + 8 < keys ? 0xFFFFu : 0u) | (j0 + 9 < keys ? 0xFFFF0000u : 0u);
            }
#pragma unroll
            for (int d = 0; d < kHd / 16; ++d) {
                uint32_t b[4];
                const int ch = 2 * (d & 3) + vchunk;
                ldsm4t(vb + (d >> 2) * (C::kKeys * 128) + vkey * 128 + ((ch ^ (vkey & 7)) << 4), b);
                if (tail) {
                    b[0] &= va;
                    b[1] &= vz;
                    b[2] &= va;
                    b[3] &= vz;
                }
                mma_16<T>(o[2 * d], ph, b[0], b[1]);
                mma_16<T>(o[2 * d + 1], ph, b[2], b[3]);
                mma_16<T>(o[2 * d], pl, b[0], b[1]);
                mma_16<T>(o[2 * d + 1], pl, b[2], b[3]);
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&empty[st]);
        }
        // ---- the item's end: join the four warps
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
            if (c4 == 0) {
                s_m[warp][g4 + 8 * r] = m[r];
                s_l[warp][g4 + 8 * r] = l[r];
            }
        }
        int any_bad;
        asm volatile(
            "{\n.reg .pred p;\nsetp.ne.s32 p, %1, 0;\nbarrier.cta.red.or.pred p, 1, 128, p;\nselp.s32 %0, 1, 0, p;\n}"
            : "=r"(any_bad)
            : "r"(static_cast<int>(bad))
            : "memory");
        float wf[2];  // this warp's weights
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            float mm = -INFINITY;
#pragma unroll
            for (int i = 0; i < C::kWarps; ++i) mm = fmaxf(mm, s_m[i][g4 + 8 * r]);
            wf[r] = m[r] == -INFINITY ? 0.0f : ex2(m[r] - mm) * (1.0f / kScale);
        }
        // the rows as they are written: thread (row tid / 8, columns 4 (tid % 8) .. + 3)
        const int row = tid >> 3, cq = (tid & 7) * 4;
        float mm = -INFINITY, ll = 0.0f;
#pragma unroll
        for (int i = 0; i < C::kWarps; ++i) mm = fmaxf(mm, s_m[i][row]);
#pragma unroll
        for (int i = 0; i < C::kWarps; ++i) ll += s_l[i][row] == 0.0f ? 0.0f : s_l[i][row] * ex2(s_m[i][row] - mm);
        const int ot = written.token(w.rt, tt, w.s.q_len);
        const int64_t orow = (w.s.row0 + (ot < 0 ? 0 : ot)) * kv.nh + w.h * G + written.g;
        const bool whole = kCluster ? cs == 1 : w.whole();
        const int64_t slot = static_cast<int64_t>(blockIdx.x) * 2 + w.slot();
        float* s_part = reinterpret_cast<float*>(smem);  // a cluster CTA's rows, where the ring was: every tile has been read
        const float inv = ll > 0.0f ? 1.0f / ll : 0.0f;
#pragma unroll
        for (int d0 = 0; d0 < kHd; d0 += C::kJoinDims) {
#pragma unroll
            for (int i = 0; i < C::kJoinDims / 8; ++i)
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const int oi = d0 / 8 + i;
                    *reinterpret_cast<float2*>(s_o + (warp * 16 + g4 + 8 * r) * C::kJoinDims + 8 * i + 2 * c4) =
                        make_float2(o[oi][2 * r] * wf[r], o[oi][2 * r + 1] * wf[r]);
                }
            asm volatile("bar.sync 1, 128;" ::: "memory");
            float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int i = 0; i < C::kWarps; ++i) {
                const float4 u = *reinterpret_cast<const float4*>(s_o + (i * 16 + row) * C::kJoinDims + cq);
                v.x += u.x;
                v.y += u.y;
                v.z += u.z;
                v.w += u.w;
            }
            if (whole) {
                if (ot >= 0)
                    *reinterpret_cast<uint2*>(static_cast<T*>(A.o.out) + orow * kHd + d0 + cq) =
                        make_uint2(M::pack(v.x * inv, v.y * inv), M::pack(v.z * inv, v.w * inv));
            } else if constexpr (kCluster) {
                *reinterpret_cast<float4*>(s_part + row * kHd + d0 + cq) = v;
            } else {
                *reinterpret_cast<float4*>(A.sc.o + (slot * 16 + row) * kHd + d0 + cq) = v;
            }
            asm volatile("bar.sync 1, 128;" ::: "memory");
        }
        if (any_bad && ot >= 0) {  // rare
            const int from = max(first_pos + 1, w.t0 * C::kKeys), to = min(w.s.kv_len - w.s.q_len + ot, w.t1 * C::kKeys - 1);
            if (whole) paged_add_not_finite<T, kHd, 32>(kv, w.b, w.h, from, to, cq, static_cast<T*>(A.o.out) + orow * kHd);
            else if (kCluster) paged_add_not_finite<T, kHd, 32>(kv, w.b, w.h, from, to, cq, s_part + row * kHd);
            else paged_add_not_finite<T, kHd, 32>(kv, w.b, w.h, from, to, cq, A.sc.o + (slot * 16 + row) * kHd);
        }
        if ((tid & 7) == 0) {
            if (whole) {
                if (A.o.lse && ot >= 0) A.o.lse[orow] = ll == 0.0f ? -INFINITY : (mm + log2f(ll)) * 0.69314718055994531f;
            } else if constexpr (kCluster) {
                s_ml[row][0] = mm;
                s_ml[row][1] = ll;
            } else {
                *reinterpret_cast<float2*>(A.sc.ml + (slot * 16 + row) * 2) = make_float2(mm, ll);
            }
        }
        if constexpr (kCluster) {
            if (cs > 1) {
                __syncwarp();
                cluster_sync();
                // this CTA's share of the rows' 16-byte columns: the pieces in order, weighted by 2^(m_i - m)
                constexpr int kQuads = 16 * kHd / 4;
                for (int i = kQuads * rank / cs + tid; i < kQuads * (rank + 1) / cs; i += 128) {
                    const int r = i / (kHd / 4), c = i % (kHd / 4) * 4;
                    float mi[8], li[8];
                    float4 u[8];
#pragma unroll
                    for (int p = 0; p < 8; ++p) {
                        mi[p] = -INFINITY, li[p] = 0.0f;
                        if (p < cs) {
                            mi[p] = ld_dsmem_f32(dsmem_addr(&s_ml[r][0], p));
                            li[p] = ld_dsmem_f32(dsmem_addr(&s_ml[r][1], p));
                            u[p] = ld_dsmem_v4(dsmem_addr(s_part + r * kHd + c, p));
                        }
                    }
                    float m_all = -INFINITY, l_all = 0.0f;
#pragma unroll
                    for (int p = 0; p < 8; ++p) m_all = fmaxf(m_all, mi[p]);
                    float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                    for (int p = 0; p < 8; ++p)
                        if (li[p] != 0.0f) {
                            const float f = ex2(mi[p] - m_all);
                            l_all += f * li[p];
                            x.x += f * u[p].x;
                            x.y += f * u[p].y;
                            x.z += f * u[p].z;
                            x.w += f * u[p].w;
                        }
                    const PagedRow pr(r, 16, G);
                    const int t = pr.token(0, tt, w.s.q_len);
                    if (t < 0) continue;
                    const float f = l_all > 0.0f ? 1.0f / l_all : 0.0f;
                    const int64_t at = (w.s.row0 + t) * kv.nh + w.h * G + pr.g;
                    *reinterpret_cast<uint2*>(static_cast<T*>(A.o.out) + at * kHd + c) =
                        make_uint2(M::pack(x.x * f, x.y * f), M::pack(x.z * f, x.w * f));
                    if (A.o.lse && c == 0) A.o.lse[at] = l_all == 0.0f ? -INFINITY : (m_all + log2f(l_all)) * 0.69314718055994531f;
                }
                __syncwarp();
                cluster_sync();  // no CTA leaves while another reads from it
            }
        } else if (!whole && w.t0 == 0)
            join = PagedJoin{w.s.row0, w.s.q_len, w.h, w.rt, w.pieces(cut)};
    }
    if (!kCluster && tid == 0) A.sc.join[blockIdx.x] = join;
}

// ---------------------------------------------------------------- joining the pieces of cut items
// CTA (w, part): 16 rows of the item that CTA w began and others finished, 16 threads to a row: each thread loads
// the maxima and sums of every 16th piece, then all add the outputs weighted by 2^(m_i - m), in the pieces'
// order, four pieces' loads at a time (one after the other they took 11 us for 10 pieces, all of it latency).
constexpr int kCombineRows = 16;
template <typename Out, int kHd>
__global__ void __launch_bounds__(256) k_paged_combine(const PagedLaunch A) {
    constexpr int kCols = kHd / 16;  // columns of a thread
    const int sub = threadIdx.x & 15, row = blockIdx.y * kCombineRows + (threadIdx.x >> 4), c0 = sub * kCols;
    const int G = A.c.nh / A.c.nkv, rows = A.tl.rows;
    const PagedRow mine(row, A.tl.sub, G);
    const uint32_t half = 0xFFFFu << (threadIdx.x & 16);  // the row's threads
    pdl_launch_dependents();
    pdl_wait();
    const PagedJoin j = A.sc.join[blockIdx.x];
    if (j.pieces == 0) return;
    const int tok = mine.token(j.rt, A.tl.tt, j.q_len);
    if (tok < 0) return;
    // piece i: slot 1 of CTA w for the first, slot 0 of CTA w + i for the others
    auto at = [&](int i) { return (static_cast<int64_t>(blockIdx.x + i) * 2 + (i == 0 ? 1 : 0)) * rows + row; };
    float m = -INFINITY, l = 0.0f;
    float o[kCols] = {};
    for (int i0 = 0; i0 < j.pieces; i0 += 16) {  // pieces beyond 16: joined to what there is
        float2 ml = make_float2(-INFINITY, 0.0f);
        if (i0 + sub < j.pieces) ml = *reinterpret_cast<const float2*>(A.sc.ml + at(i0 + sub) * 2);
        float mx = ml.x;
#pragma unroll
        for (int x = 8; x > 0; x >>= 1) mx = fmaxf(mx, __shfl_xor_sync(half, mx, x));
        const float mn = fmaxf(m, mx);
        const float ms = mn == -INFINITY ? 0.0f : mn;
        const float f = ex2(ml.x - ms), keep = ex2(m - ms);
        float ls = f * ml.y;
#pragma unroll
        for (int x = 8; x > 0; x >>= 1) ls += __shfl_xor_sync(half, ls, x);
        l = l * keep + ls;
        m = mn;
#pragma unroll
        for (int c = 0; c < kCols; ++c) o[c] *= keep;
        const int n = min(16, j.pieces - i0);
        for (int i1 = 0; i1 < n; i1 += 4) {
            float4 v[4][kCols / 4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int c = 0; c < kCols / 4; ++c)
                    v[i][c] = i1 + i < n ? *reinterpret_cast<const float4*>(A.sc.o + at(i0 + i1 + i) * kHd + c0 + 4 * c)
                                         : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float w = __shfl_sync(half, f, (threadIdx.x & 16) + i1 + i);
#pragma unroll
                for (int c = 0; c < kCols / 4; ++c) {
                    o[4 * c] += w * v[i][c].x;
                    o[4 * c + 1] += w * v[i][c].y;
                    o[4 * c + 2] += w * v[i][c].z;
                    o[4 * c + 3] += w * v[i][c].w;
                }
            }
        }
    }
    const float inv = l > 0.0f ? 1.0f / l : 0.0f;
    const int64_t orow = (j.row0 + tok) * A.c.nh + j.h * G + mine.g;
    Out* dst = static_cast<Out*>(A.o.out) + orow * kHd + c0;
    if constexpr (sizeof(Out) == 4) {
#pragma unroll
        for (int c = 0; c < kCols; c += 4)
            *reinterpret_cast<float4*>(dst + c) = make_float4(o[c] * inv, o[c + 1] * inv, o[c + 2] * inv, o[c + 3] * inv);
    } else {
#pragma unroll
        for (int c = 0; c < kCols; c += 4)
            *reinterpret_cast<uint2*>(dst + c) = make_uint2(Pack16<Out>::pack(o[c] * inv, o[c + 1] * inv),
                                                            Pack16<Out>::pack(o[c + 2] * inv, o[c + 3] * inv));
    }
    if (A.o.lse && sub == 0) A.o.lse[orow] = l == 0.0f ? -INFINITY : (m + log2f(l)) * 0.69314718055994531f;
}

template <typename Out>
static cudaError_t launch_combine_t(const PagedLaunch& a, int hd, int ctas, cudaStream_t s) {
    const dim3 grid(static_cast<unsigned>(ctas), static_cast<unsigned>(a.tl.rows / kCombineRows));
    return hd == 128 ? launch_pdl(k_paged_combine<Out, 128>, grid, dim3(256), 0, s, a)
                     : launch_pdl(k_paged_combine<Out, 64>, grid, dim3(256), 0, s, a);
}
cudaError_t launch_paged_combine(const PagedLaunch& a, int out_dtype, int hd, int ctas, cudaStream_t s) {
    return out_dtype == SC_F16    ? launch_combine_t<__half>(a, hd, ctas, s)
           : out_dtype == SC_BF16 ? launch_combine_t<__nv_bfloat16>(a, hd, ctas, s)
                                  : launch_combine_t<float>(a, hd, ctas, s);
}

template <typename T, int kHd>
static cudaError_t launch_decode_t(const DecodeParams& p, int ctas, cudaStream_t s) {
    using C = DecCfg<kHd>;
    static std::atomic<uint64_t> flags{0}, flags_cluster{0};
    if (p.cluster == 0) {
        cudaError_t e = paged_allow_smem(k_paged_decode<T, kHd, false>, flags, C::kSmem);
        if (e != cudaSuccess) return e;
        return launch_pdl(k_paged_decode<T, kHd, false>, dim3(static_cast<unsigned>(ctas)), dim3(C::kThreads), C::kSmem, s, p);
    }
    cudaError_t e = paged_allow_smem(k_paged_decode<T, kHd, true>, flags_cluster, C::kSmem);
    if (e != cudaSuccess) return e;
    return paged_launch_clusters(k_paged_decode<T, kHd, true>, ctas, C::kThreads, C::kSmem, p.cluster, s, p);
}

cudaError_t launch_paged_decode(const PagedLaunch& a, int dtype, int hd, int ctas, int cluster, cudaStream_t s) {
    DecodeParams p;
    p.a = a;
    p.cluster = cluster;
    p.box_shift = a.c.page_shift < 6 ? a.c.page_shift : 6;
    cudaError_t e = paged_tensor_map(&p.kmap, a.c, a.c.k, dtype, hd, 1 << p.box_shift);
    if (e == cudaSuccess) e = paged_tensor_map(&p.vmap, a.c, a.c.v, dtype, hd, 1 << p.box_shift);
    if (e != cudaSuccess) return e;
    if (dtype == SC_F16)
        return hd == 128 ? launch_decode_t<__half, 128>(p, ctas, s) : launch_decode_t<__half, 64>(p, ctas, s);
    return hd == 128 ? launch_decode_t<__nv_bfloat16, 128>(p, ctas, s) : launch_decode_t<__nv_bfloat16, 64>(p, ctas, s);
}

}  // namespace sc
