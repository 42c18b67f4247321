// sc_paged_f32.cu -- attention over an f32 paged cache, in f32 on the CUDA cores.
//
// No tensor-core format holds 24 bits, so the products are f32 FMAs, two to an instruction
// (fma.rn.f32x2).  Their operands come from shared memory: a thread takes 4 rows x (1 or 4) keys of S and 4 rows x
// hd / 16 columns of O, 16-byte loads along head_dim and along the columns.  A row tile has 64 rows, or 16 for few
// new tokens; there the 16 positions of a quarter of the key tile go to a quarter of the threads
// with a running maximum and sum of its own, joined at the item's end, so that every thread keeps 4 rows.
// K and V tiles of 64 positions come by 16-byte asynchronous copies, the next K while O is updated, the
// next V while S is computed, with four barriers a tile: the kernel waits more than it issues (31 % of the cycles at 12
// sequences of 1..24 new tokens); rows padded by 16 bytes keep 8 of them on different banks.  Positions behind
// the last one are zero-filled.  Pieces of the line of key tiles go to the CTAs evenly (sc_paged.cuh); few new
// tokens whose CTAs would have at most kClusterKeysF32 positions each go to clusters as in sc_paged_decode.cu (one
// sequence of 1..256 positions, 28 + 4 heads of 128: 12.2 us cut, 8.4 us in clusters; 4 of 513..1024 16.2 and 18.5;
// row tiles of 64 rows, bound by their arithmetic, want the even cut: 12 sequences of 1..24 new tokens over up to
// 1500 positions 36 us cut, 56 us in clusters of 4).
#include <atomic>
#include <type_traits>

#include "sc_paged.cuh"

namespace sc {

__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool valid) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// d += a * b on two f32 at once.
__device__ __forceinline__ void fma2(uint64_t& d, uint64_t a, uint64_t b) {
    asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(d) : "l"(a), "l"(b));
}
__device__ __forceinline__ uint64_t two(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float2 both(uint64_t v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
struct alignas(16) Four {
    uint64_t a, b;
};

template <int kRows, int kHd>
struct F32Cfg {
    static constexpr int kKeys = 64, kThreads = 256, kLd = kHd + 4;
    static constexpr int kGroups = 64 / kRows;           // quarters of the key tile (16 rows), or the whole of it
    static constexpr int kKpt = 4 / kGroups;             // keys of a thread
    static constexpr int kPld = kKeys / kGroups + 4;     // row of a group's weights
    static constexpr int kQ = kRows * kLd, kKv = kKeys * kLd, kP = kGroups * kRows * kPld;
    static constexpr int kSmem = (kQ + 2 * kKv + kP) * 4;
};

// kCluster (few new tokens: one row tile): a (sequence, KV head) per cluster of P.cluster CTAs, which divide its key
// tiles and join them through distributed shared memory; otherwise a piece of the line per CTA.
struct F32Params {
    PagedLaunch a;
    int cluster;
};

template <typename Out, int kRows, int kHd, bool kCluster>
__global__ void __launch_bounds__(256, kRows == 16 || kHd == 64 ? 2 : 1) k_paged_f32(const F32Params P) {
    using C = F32Cfg<kRows, kHd>;
    const PagedLaunch& A = P.a;
    constexpr int kC8 = kHd / 16;  // columns of O of a thread: 4 at 4 tx + 64 i
    extern __shared__ __align__(16) float sm[];
    __shared__ PagedCut cut;
    __shared__ float s_m[C::kGroups][kRows], s_l[C::kGroups][kRows], s_ml[kRows][2];
    float *sq = sm, *sk = sm + C::kQ, *sv = sk + C::kKv, *sp = sv + C::kKv;
    const PagedKv& kv = A.c;
    const int tid = threadIdx.x, G = kv.nh / kv.nkv, tt = A.tl.tt;
    const int tx = tid & 15, ty = (tid >> 4) % (kRows / 4), grp = tid / (kRows * 4);
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
    } else {
        paged_cut<C::kThreads>(kv, A.max_q, tt, C::kKeys, &cut);
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
    const PagedRow mine[4] = {PagedRow(ty * 4, kRows, G), PagedRow(ty * 4 + 1, kRows, G), PagedRow(ty * 4 + 2, kRows, G),
                              PagedRow(ty * 4 + 3, kRows, G)};
    PagedJoin join{0, 0, 0, 0, 0};
    const float sl2 = A.o.sl2;
    while (next_item()) {
        const int start = w.s.kv_len - w.s.q_len;
        const int keys = start + min((w.rt + 1) * tt, w.s.q_len);
        const int some = start + w.rt * tt + 1;  // from here on only some of the rows attend
        bool bad = false;                        // has met a value there that is not finite
        const int32_t* table = kv.table + w.b * kv.max_pages;
        // this thread copies chunk `cc` of rows cr + kStep j: their places in the pages are found for a K tile and
        // kept for its V tile
        constexpr int kStep = C::kThreads / (kHd / 4), kCopies = C::kKeys / kStep;
        const int cr = tid / (kHd / 4), cc = tid % (kHd / 4) * 4;
        int64_t place[kCopies];
        int id[kCopies];
        auto look_up = [&](int t) {  // the rows' pages, a tile ahead
#pragma unroll
            for (int j = 0; j < kCopies; ++j) {
                const int key = t * C::kKeys + cr + kStep * j;
                id[j] = key < keys ? table[key >> kv.page_shift] : -1;
            }
        };
        auto find = [&](int t) {
#pragma unroll
            for (int j = 0; j < kCopies; ++j) {
                const int key = t * C::kKeys + cr + kStep * j;
                if (id[j] >= 0 && id[j] < kv.num_pages) {
                    place[j] = id[j] * kv.page_stride +
                               ((static_cast<int64_t>(w.h) << kv.page_shift) + (key & ((1 << kv.page_shift) - 1))) * kHd + cc;
                } else {
                    if (key < keys) record_error(kv.status, DEV_BAD_INDEX);
                    place[j] = -1;  // zeros
                }
            }
        };
        auto load = [&](const void* pages, float* dst) {  // a K or V tile, asynchronously
            const uint32_t d0 = smem_u32(dst + cr * C::kLd + cc);
#pragma unroll
            for (int j = 0; j < kCopies; ++j)
                cp16(d0 + j * kStep * C::kLd * 4, static_cast<const float*>(pages) + (place[j] < 0 ? 0 : place[j]), place[j] >= 0);
            cp_commit();
        };
        if (w.t0 < w.t1) look_up(w.t0);  // (a cluster's CTA may have none)
        constexpr int kQueries = kRows * (kHd / 4) / C::kThreads;
        float4 qv[kQueries];
#pragma unroll
        for (int j = 0; j < kQueries; ++j) {  // the query rows this thread stages
            const PagedRow row(cr + kStep * j, kRows, G);
            const int tok = row.token(w.rt, tt, w.s.q_len);
            qv[j] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (tok >= 0)
                qv[j] = *reinterpret_cast<const float4*>(static_cast<const float*>(A.q) + (w.s.row0 + tok) * A.q_stride +
                                                         (w.h * G + row.g) * kHd + cc);
        }
        __syncthreads();  // the item before has read its tiles
        if (w.t0 < w.t1) {
            find(w.t0);
            load(kv.k, sk);
            load(kv.v, sv);
        }
#pragma unroll
        for (int j = 0; j < kQueries; ++j) *reinterpret_cast<float4*>(sq + (cr + kStep * j) * C::kLd + cc) = qv[j];
        int pos[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int tok = mine[i].token(w.rt, tt, w.s.q_len);
            pos[i] = tok >= 0 ? start + tok : -1;
        }
        float m[4], l[4];
        uint64_t o[4][kC8 / 2];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            m[i] = -INFINITY;
            l[i] = 0.0f;
#pragma unroll
            for (int c = 0; c < kC8 / 2; ++c) o[i][c] = 0;
        }
        for (int t = w.t0; t < w.t1; ++t) {
            if (t + 1 < w.t1) look_up(t + 1);
            cp_wait<1>();
            __syncthreads();  // K(t) is there (and the queries)
            uint64_t s2[4][C::kKpt];
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < C::kKpt; ++j) s2[i][j] = 0;
            const float* q0 = sq + ty * 4 * C::kLd;
            const float* k0 = sk + (grp * 16 + tx) * C::kLd;
#pragma unroll 4
            for (int d = 0; d < kHd; d += 4) {
                Four q[4], k[C::kKpt];
#pragma unroll
                for (int i = 0; i < 4; ++i) q[i] = *reinterpret_cast<const Four*>(q0 + i * C::kLd + d);
#pragma unroll
                for (int j = 0; j < C::kKpt; ++j) k[j] = *reinterpret_cast<const Four*>(k0 + j * 16 * C::kLd + d);
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int j = 0; j < C::kKpt; ++j) {
                        fma2(s2[i][j], q[i].a, k[j].a);
                        fma2(s2[i][j], q[i].b, k[j].b);
                    }
            }
            __syncthreads();  // K(t) has been read
            if (t + 1 < w.t1) {
                find(t + 1);
                load(kv.k, sk);
            } else {
                cp_commit();
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float s[C::kKpt], mx = -INFINITY;
#pragma unroll
                for (int j = 0; j < C::kKpt; ++j) {
                    const float2 u = both(s2[i][j]);
                    s[j] = t * C::kKeys + grp * 16 + 16 * j + tx <= pos[i] ? u.x + u.y : -INFINITY;
                    mx = fmaxf(mx, s[j]);
                }
#pragma unroll
                for (int x = 8; x > 0; x >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
                const float mn = fmaxf(m[i], mx * sl2);
                const float ms = mn == -INFINITY ? 0.0f : mn;
                const float f = ex2(m[i] - ms);
                m[i] = mn;
                l[i] *= f;
                const uint64_t f2 = two(f, f);
#pragma unroll
                for (int c = 0; c < kC8 / 2; ++c) asm("mul.rn.f32x2 %0, %0, %1;" : "+l"(o[i][c]) : "l"(f2));
#pragma unroll
                for (int j = 0; j < C::kKpt; ++j) {
                    const float p = ex2(fmaf(s[j], sl2, -ms));
                    l[i] += p;
                    sp[(grp * kRows + ty * 4 + i) * C::kPld + 16 * j + tx] = p;
                }
            }
            cp_wait<1>();
            if ((t + 1) * C::kKeys > some) {  // the values that this thread copied
#pragma unroll
                for (int j = 0; j < kCopies; ++j) {
                    float* at = sv + (cr + kStep * j) * C::kLd + cc;
                    const float4 v = *reinterpret_cast<const float4*>(at);
                    // (finite values' differences are 0, and so is their sum)
                    if (!((v.x - v.x) + (v.y - v.y) + (v.z - v.z) + (v.w - v.w) == 0.0f) && t * C::kKeys + cr + kStep * j >= some) {
                        for (int c = 0; c < 4; ++c)
                            if (!(at[c] - at[c] == 0.0f)) at[c] = 0.0f;
                        bad = true;
                    }
                }
            }
            __syncthreads();  // V(t) is there, and the weights
            const float* p0 = sp + (grp * kRows + ty * 4) * C::kPld;
            const float* v0 = sv + grp * 16 * C::kLd + 4 * tx;
#pragma unroll 2
            for (int k = 0; k < C::kKeys / C::kGroups; k += 4) {
                float4 p[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) p[i] = *reinterpret_cast<const float4*>(p0 + i * C::kPld + k);
#pragma unroll
                for (int x = 0; x < 4; ++x) {
#pragma unroll
                    for (int c = 0; c < kC8 / 4; ++c) {
                        const Four v = *reinterpret_cast<const Four*>(v0 + (k + x) * C::kLd + 64 * c);
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const float pv = x == 0 ? p[i].x : x == 1 ? p[i].y : x == 2 ? p[i].z : p[i].w;
                            const uint64_t pp = two(pv, pv);
                            fma2(o[i][2 * c], pp, v.a);
                            fma2(o[i][2 * c + 1], pp, v.b);
                        }
                    }
                }
            }
            __syncthreads();  // V(t) and the weights have been read
            if (t + 1 < w.t1) load(kv.v, sv);
            else cp_commit();
        }
        cp_wait<0>();
        // ---- the item's end
#pragma unroll
        for (int i = 0; i < 4; ++i) {
#pragma unroll
            for (int x = 8; x > 0; x >>= 1) l[i] += __shfl_xor_sync(0xffffffffu, l[i], x);
            if (C::kGroups > 1 && tx == 0) {
                s_m[grp][ty * 4 + i] = m[i];
                s_l[grp][ty * 4 + i] = l[i];
            }
        }
        if (kCluster) __syncthreads();  // (K's and V's place is written again)
        const bool whole = kCluster ? cs == 1 : w.whole();
        const int64_t slot = static_cast<int64_t>(blockIdx.x) * 2 + w.slot();
        auto write = [&](int row, int col, float4 v, float mm, float ll) {  // 4 columns of a row, and its sums once
            if (kCluster && !whole) {  // where K was: every tile has been read
                *reinterpret_cast<float4*>(sk + row * kHd + col) = v;
                if (col == 0) s_ml[row][0] = mm, s_ml[row][1] = ll;
                return;
            }
            const PagedRow r(row, kRows, G);
            const int tok = r.token(w.rt, tt, w.s.q_len);
            if (tok < 0) return;
            const int64_t orow = (w.s.row0 + tok) * kv.nh + w.h * G + r.g;
            if (whole) {
                const float inv = ll > 0.0f ? 1.0f / ll : 0.0f;
                v.x *= inv, v.y *= inv, v.z *= inv, v.w *= inv;
                if constexpr (std::is_same<Out, __half>::value)
                    *reinterpret_cast<uint2*>(static_cast<__half*>(A.o.out) + orow * kHd + col) =
                        make_uint2(Pack16<__half>::pack(v.x, v.y), Pack16<__half>::pack(v.z, v.w));
                else
                    *reinterpret_cast<float4*>(static_cast<float*>(A.o.out) + orow * kHd + col) = v;
                if (col == 0 && A.o.lse) A.o.lse[orow] = ll == 0.0f ? -INFINITY : (mm + log2f(ll)) * 0.69314718055994531f;
            } else {
                *reinterpret_cast<float4*>(A.sc.o + (slot * kRows + row) * kHd + col) = v;
                if (col == 0) *reinterpret_cast<float2*>(A.sc.ml + (slot * kRows + row) * 2) = make_float2(mm, ll);
            }
        };
        if (C::kGroups == 1) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int c = 0; c < kC8 / 4; ++c) {
                    const float2 a = both(o[i][2 * c]), b = both(o[i][2 * c + 1]);
                    write(ty * 4 + i, 4 * tx + 64 * c, make_float4(a.x, a.y, b.x, b.y), m[i], l[i]);
                }
        } else {
            __syncthreads();  // the groups' maxima and sums are there, V has been read
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float mm = -INFINITY;
#pragma unroll
                for (int x = 0; x < C::kGroups; ++x) mm = fmaxf(mm, s_m[x][ty * 4 + i]);
                const float f = m[i] == -INFINITY ? 0.0f : ex2(m[i] - mm);
#pragma unroll
                for (int c = 0; c < kC8 / 4; ++c) {
                    const float2 a = both(o[i][2 * c]), b = both(o[i][2 * c + 1]);
                    *reinterpret_cast<float4*>(sv + (grp * kRows + ty * 4 + i) * C::kLd + 4 * tx + 64 * c) =
                        make_float4(a.x * f, a.y * f, b.x * f, b.y * f);
                }
            }
            __syncthreads();
            for (int i = tid; i < kRows * (kHd / 4); i += C::kThreads) {
                const int row = i / (kHd / 4), col = i % (kHd / 4) * 4;
                float mm = -INFINITY, ll = 0.0f;
#pragma unroll
                for (int x = 0; x < C::kGroups; ++x) mm = fmaxf(mm, s_m[x][row]);
                float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                for (int x = 0; x < C::kGroups; ++x) {
                    const float4 u = *reinterpret_cast<const float4*>(sv + (x * kRows + row) * C::kLd + col);
                    v.x += u.x, v.y += u.y, v.z += u.z, v.w += u.w;
                    ll += s_l[x][row] == 0.0f ? 0.0f : s_l[x][row] * ex2(s_m[x][row] - mm);
                }
                write(row, col, v, mm, ll);
            }
        }
        if (__syncthreads_or(bad)) {  // rare; the rows have been written
            const PagedRow r(tid, kRows, G);
            const int tok = tid < kRows ? r.token(w.rt, tt, w.s.q_len) : -1;
            const int from = max(some, w.t0 * C::kKeys), to = min(start + tok, w.t1 * C::kKeys - 1);
            const int64_t orow = (w.s.row0 + tok) * kv.nh + w.h * G + r.g;
            if (tok >= 0) {
                if (whole) paged_add_not_finite<float, kHd, 4>(kv, w.b, w.h, from, to, 0, static_cast<Out*>(A.o.out) + orow * kHd);
                else if (kCluster) paged_add_not_finite<float, kHd, 4>(kv, w.b, w.h, from, to, 0, sk + tid * kHd);
                else paged_add_not_finite<float, kHd, 4>(kv, w.b, w.h, from, to, 0, A.sc.o + (slot * kRows + tid) * kHd);
            }
            __syncthreads();
        }
        if constexpr (kCluster) {
            if (cs > 1) {
                __syncwarp();
                cluster_sync();
                // this CTA's share of the rows' 16-byte columns: the pieces in order, weighted by 2^(m_i - m)
                constexpr int kQuads = kRows * kHd / 4;
                for (int i = kQuads * rank / cs + tid; i < kQuads * (rank + 1) / cs; i += C::kThreads) {
                    const int row = i / (kHd / 4), col = i % (kHd / 4) * 4;
                    float mi[8], li[8];
                    float4 u[8];
#pragma unroll
                    for (int p = 0; p < 8; ++p) {
                        mi[p] = -INFINITY, li[p] = 0.0f;
                        if (p < cs) {
                            mi[p] = ld_dsmem_f32(dsmem_addr(&s_ml[row][0], p));
                            li[p] = ld_dsmem_f32(dsmem_addr(&s_ml[row][1], p));
                            u[p] = ld_dsmem_v4(dsmem_addr(sk + row * kHd + col, p));
                        }
                    }
                    float mm = -INFINITY, ll = 0.0f;
#pragma unroll
                    for (int p = 0; p < 8; ++p) mm = fmaxf(mm, mi[p]);
                    float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                    for (int p = 0; p < 8; ++p)
                        if (li[p] != 0.0f) {
                            const float f = ex2(mi[p] - mm);
                            ll += f * li[p];
                            x.x += f * u[p].x;
                            x.y += f * u[p].y;
                            x.z += f * u[p].z;
                            x.w += f * u[p].w;
                        }
                    const PagedRow r(row, kRows, G);
                    const int tok = r.token(w.rt, tt, w.s.q_len);
                    if (tok < 0) continue;
                    const float inv = ll > 0.0f ? 1.0f / ll : 0.0f;
                    const int64_t orow = (w.s.row0 + tok) * kv.nh + w.h * G + r.g;
                    x.x *= inv, x.y *= inv, x.z *= inv, x.w *= inv;
                    if constexpr (std::is_same<Out, __half>::value)
                        *reinterpret_cast<uint2*>(static_cast<__half*>(A.o.out) + orow * kHd + col) =
                            make_uint2(Pack16<__half>::pack(x.x, x.y), Pack16<__half>::pack(x.z, x.w));
                    else
                        *reinterpret_cast<float4*>(static_cast<float*>(A.o.out) + orow * kHd + col) = x;
                    if (col == 0 && A.o.lse) A.o.lse[orow] = ll == 0.0f ? -INFINITY : (mm + log2f(ll)) * 0.69314718055994531f;
                }
                __syncwarp();
                cluster_sync();  // no CTA leaves while another reads from it
            }
        } else if (!whole && w.t0 == 0)
            join = PagedJoin{w.s.row0, w.s.q_len, w.h, w.rt, w.pieces(cut)};
    }
    if (!kCluster && tid == 0) A.sc.join[blockIdx.x] = join;
}

template <typename Out, int kRows, int kHd>
static cudaError_t launch_f32_t(const F32Params& p, int ctas, cudaStream_t s) {
    using C = F32Cfg<kRows, kHd>;
    static std::atomic<uint64_t> flags{0}, flags_cluster{0};
    if constexpr (kRows == 16) {
        if (p.cluster > 0) {
            const cudaError_t e = paged_allow_smem(k_paged_f32<Out, kRows, kHd, true>, flags_cluster, C::kSmem);
            if (e != cudaSuccess) return e;
            return paged_launch_clusters(k_paged_f32<Out, kRows, kHd, true>, ctas, C::kThreads, C::kSmem, p.cluster, s, p);
        }
    }
    const cudaError_t e = paged_allow_smem(k_paged_f32<Out, kRows, kHd, false>, flags, C::kSmem);
    if (e != cudaSuccess) return e;
    return launch_pdl(k_paged_f32<Out, kRows, kHd, false>, dim3(static_cast<unsigned>(ctas)), dim3(C::kThreads), C::kSmem, s, p);
}

cudaError_t launch_paged_f32(const PagedLaunch& a, int out_dtype, int hd, int ctas, int cluster, cudaStream_t s) {
    const F32Params p{a, cluster};
    if (a.tl.rows == 16) {
        if (out_dtype == SC_F16)
            return hd == 128 ? launch_f32_t<__half, 16, 128>(p, ctas, s) : launch_f32_t<__half, 16, 64>(p, ctas, s);
        return hd == 128 ? launch_f32_t<float, 16, 128>(p, ctas, s) : launch_f32_t<float, 16, 64>(p, ctas, s);
    }
    if (out_dtype == SC_F16)
        return hd == 128 ? launch_f32_t<__half, 64, 128>(p, ctas, s) : launch_f32_t<__half, 64, 64>(p, ctas, s);
    return hd == 128 ? launch_f32_t<float, 64, 128>(p, ctas, s) : launch_f32_t<float, 64, 64>(p, ctas, s);
}

}  // namespace sc
