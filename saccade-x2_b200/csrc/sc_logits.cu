// sc_logits.cu -- penalties, biases and grammar masks on logits, with the best token of each row.
//
// Per token v of a row, in f32 and rounded once to the logits' type:
//   x1 = seen(v) ? (x > 0 ? x / r : x * r) : x          seen: v occurs in the row's history
//   x2 = x1 - f * n(v) - (n(v) > 0 ? p : 0)             n: times v occurs among the generated tokens
//   x3 = x2 + b(v)                                      b: the last bias entry of v
//   y  = allowed(v) ? x3 : -inf
// One pass: each logit is read once and written once; the floor is rows * vocab * 2 * size bytes.
//
// A CTA has a tile of a row's vocabulary.  The counts n(v) of its tokens live in its shared memory, one
// word per token, so nothing of vocabulary size ever goes to global memory; every CTA of a row goes over
// the row's whole history (a few KB from L2, tiles x 4 bytes per id) and counts its own tokens with integer
// atomics, whose order does not matter.  (Thread-block clusters that read the history once and count into each
// other's shared memory measured slower: 39 us against 25 at 64 x 152064 f32 with 768 ids, two cluster barriers
// and 31 clusters of 16 at a time.  So did CTAs that stay, with warps of their own for the counts: 44 us.)
//   word = (bias entry + 1) << 20 | n << 1 | in the prompt
// Few tokens are touched, but nearly every warp of a streaming pass would meet one and take its division along, so
// whoever changes a word first lists its token; the listed tokens are processed by themselves, a thread each, their
// words replaced by the values, and the streaming pass takes what its vectors' words hold.  (Where the list overflows,
// every word of the tile is looked at.)  A map of a bit per token in place of the words' look-up, and the list made from
// it by prefix sums, measured 5.05 / 25.6 / 30.0 us on the three cases below; places in the list by warp ballots
// 5.2 / 26.0 / 31.3.
// Each CTA issues the loads of its first logits before it counts, so that they arrive meanwhile.  The best of
// each tile goes to the scratch, and a second small kernel picks each row's.
// Measured with everything on: 1 x 151936 f32, 256 ids 4.65 us; 64 x 152064 f32, up to 768 ids 24.5 us (3.2 TB/s; the
// copy alone 13.4); 200 x 38017 bf16, up to 8000 ids 30.4 us (1 TB/s; the copy alone 8.3).  What bounds the last
// two is the counting, a chain of short phases (zeroes, ids, atomics, list, division) in each of a few CTAs per SM; five,
// six or eight smaller CTAs per SM read the ids more often: 33 to 37 us.
#include <atomic>
#include <string>

#include "saccade_qwen2.h"
#include "sc_device.cuh"
#include "sc_internal.h"

namespace sc {

constexpr int kLogitThreads = 256;
constexpr int kLogitWords = 10240;        // tokens of a tile at most (40 KB of words: four CTAs per SM)
constexpr int kLogitMinTile = 2048;
constexpr int kLogitList = 1024;
constexpr uint32_t kLogitDone = 0x7FC0DEADu;  // a processed value's flipped bits (a NaN's, which becomes another), so that no word is 0
constexpr int kLogitBatch = 6;            // 16-byte loads a thread has in flight
constexpr int64_t kLogitMaxHistory = (1 << 19) - 1;  // 19 bits of a word count occurrences
constexpr int64_t kLogitMaxRows = 1 << 20;
constexpr int kLogitMaxBias = (1 << 12) - 1;         // 12 bits name the bias entry

struct LogitArgs {
    const void* x;
    int64_t vocab, stride, begin;
    const int32_t* history;
    int64_t history_stride;
    const int32_t* prompt_len;
    const int32_t* hist_len;
    const float *rep, *pres, *freq;
    const int32_t *bias_ptr, *bias_ids;
    const float* bias_vals;
    int64_t num_bias;
    const uint32_t* mask;
    int64_t mask_words, mask_rows;
    const int32_t* mask_row;
    void* out;
    int64_t out_stride;
    int64_t* best;
    void* best_value;
    uint32_t* status;
    int tile, tiles;  // tokens of a tile, tiles of a row
    uint64_t* keys;   // [rows][tiles], or null
};

template <typename T>
struct LogitIo;
template <>
struct LogitIo<float> {
    static constexpr int kVec = 4;
    static __device__ __forceinline__ float get(float v) { return v; }
    static __device__ __forceinline__ float put(float v) { return v; }
};
template <>
struct LogitIo<__half> {
    static constexpr int kVec = 8;
    static __device__ __forceinline__ float get(__half v) { return __half2float(v); }
    static __device__ __forceinline__ __half put(float v) { return __float2half_rn(v); }
};
template <>
struct LogitIo<__nv_bfloat16> {
    static constexpr int kVec = 8;
    static __device__ __forceinline__ float get(__nv_bfloat16 v) { return __bfloat162float(v); }
    static __device__ __forceinline__ __nv_bfloat16 put(float v) { return __float2bfloat16_rn(v); }
};

// Orders (value, index) pairs as argmax does: NaN above all, equal values (-0 and 0 among them) by the
// lower index.  The largest key wins.
__device__ __forceinline__ uint64_t best_key(float v, uint32_t i) {
    const uint32_t b = __float_as_uint(__fadd_rn(v, 0.0f));  // -0 becomes 0
    const uint32_t ord = v != v ? 0xFFFFFFFFu : (b & 0x80000000u) ? ~b : b | 0x80000000u;
    return (static_cast<uint64_t>(ord) << 32) | (0xFFFFFFFFu - i);
}

// The larger of two, NaN if either is.
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// One logit.  Multiplications and subtractions round one by one.
__device__ __forceinline__ float process_one(float x, uint32_t word, float rep, float pres, float freq,
                                             const float* bias_row) {
    if (word & 0xFFFFFu) {
        x = x > 0.0f ? __fdiv_rn(x, rep) : __fmul_rn(x, rep);
        const uint32_t n = (word & 0xFFFFFu) >> 1;
        if (n) x = __fsub_rn(__fsub_rn(x, __fmul_rn(freq, static_cast<float>(n))), pres);
    }
    if (word >> 20) x = __fadd_rn(x, bias_row[(word >> 20) - 1]);
    return x;
}

template <typename T>
__global__ void __launch_bounds__(kLogitThreads, 4) k_process_logits(const LogitArgs a) {
    constexpr int kVec = LogitIo<T>::kVec;
    extern __shared__ __align__(16) uint32_t words[];  // one per token of the tile, from its first vector on
    __shared__ uint64_t s_best[kLogitThreads / 32];
    __shared__ uint16_t s_list[kLogitList];  // the tile's touched tokens, if they are so few
    __shared__ int s_count;                  // and how many there are
    pdl_launch_dependents();
    const uint32_t row32 = blockIdx.x / static_cast<uint32_t>(a.tiles);
    const int64_t row = row32;
    const int tid = threadIdx.x;
    // the tile's tokens [t0, t0 + len); vector j covers tokens t0 - lead + j * kVec .. + kVec, so that it starts on a
    // 16-byte boundary of the row; vectors [full0, full1) lie inside
    const int64_t t0 = static_cast<int64_t>(blockIdx.x - row32 * a.tiles) * a.tile;
    const int len = static_cast<int>(imin64(a.vocab - t0, a.tile));
    const T* x = static_cast<const T*>(a.x) + row * a.stride + t0;
    const int lead = static_cast<int>((reinterpret_cast<uintptr_t>(x) & 15u) / sizeof(T));
    const int nvec = (len + lead + kVec - 1) / kVec;
    const int full0 = lead ? 1 : 0, full1 = (len + lead) / kVec;
    const T* xb = x - lead;
    T* yb = static_cast<T*>(a.out) + row * a.out_stride + t0 - lead;
    const bool same = (reinterpret_cast<uintptr_t>(yb) & 15u) == 0;
    auto load = [&](int j) {
        uint4 r;
        if (j >= full0 && j < full1) {
            r = __ldcs(reinterpret_cast<const uint4*>(xb) + j);
        } else {
            __align__(16) T v[kVec];
#pragma unroll
            for (int k = 0; k < kVec; ++k) {
                const int e = j * kVec + k;
                v[k] = e >= lead && e < lead + len ? xb[e] : T(0.0f);
            }
            r = *reinterpret_cast<const uint4*>(v);
        }
        return r;
    };
    pdl_wait();

    // the row's parameters and first logits: every load is issued before the first is needed
    float rep = a.rep ? a.rep[row] : 1.0f, pres = a.pres ? a.pres[row] : 0.0f, freq = a.freq ? a.freq[row] : 0.0f;
    int hist = a.history ? a.hist_len[row] : 0, prompt = a.history && a.prompt_len ? a.prompt_len[row] : 0;
    int64_t b0 = a.bias_ptr ? a.bias_ptr[row] : 0, b1 = a.bias_ptr ? a.bias_ptr[row + 1] : 0;
    int64_t mrow = a.mask ? (a.mask_row ? a.mask_row[row] : row) : -1;
    uint4 batch[kLogitBatch];
#pragma unroll
    for (int i = 0; i < kLogitBatch; ++i) {
        const int j = tid + i * kLogitThreads;
        if (j < nvec) batch[i] = load(j);
    }
    bool bad = false;
    if (a.history) {
        const int width = static_cast<int>(a.history_stride);
        bad = hist < 0 || hist > width || prompt < 0 || prompt > hist;
        hist = min(max(hist, 0), width);
        prompt = min(max(prompt, 0), hist);
        if (rep == 1.0f && pres == 0.0f && freq == 0.0f) hist = prompt = 0;  // counts change nothing
    }
    if (a.bias_ptr) {
        bad = bad || b0 < 0 || b1 < b0 || b1 > a.num_bias || b1 - b0 > kLogitMaxBias;
        b0 = b0 < 0 ? 0 : imin64(b0, a.num_bias);
        b1 = b1 < b0 ? b0 : imin64(imin64(b1, a.num_bias), b0 + kLogitMaxBias);
    }
    if (a.mask && mrow >= a.mask_rows) {
        bad = true;
        mrow = -1;
    }
    if (bad && tid == 0) record_error(a.status, DEV_BAD_INDEX);
    const uint32_t* mask = mrow >= 0 ? a.mask + mrow * a.mask_words : nullptr;
    const int first = static_cast<int>(t0 + a.begin);  // the tile's first token id
    const int nb = static_cast<int>(b1 - b0);
    const bool touched = hist > 0 || nb > 0;
    if (touched) {
        for (int i = tid; i < nvec * (kVec / 4); i += kLogitThreads)
            reinterpret_cast<uint4*>(words)[i] = make_uint4(0, 0, 0, 0);
        if (tid == 0) s_count = 0;
        __syncthreads();
        auto push = [&](int at) {  // whoever changed the word first
            const int place = atomicAdd(&s_count, 1);
            if (place < kLogitList) s_list[place] = static_cast<uint16_t>(at);
        };
        for (int i = tid; i < nb; i += kLogitThreads) {
            const int v = a.bias_ids[b0 + i];
            if (v >= first && v - first < len) {
                const int at = v - first + lead;
                if (atomicMax(&words[at], static_cast<uint32_t>(i + 1) << 20) == 0) push(at);
            }
        }
        if (nb > 0) __syncthreads();  // an entry's number is settled before counts join it in the word
        const int32_t* h = a.history + row * a.history_stride;
        constexpr int kIds = 8;
        for (int i0 = tid; i0 < hist; i0 += kIds * kLogitThreads) {
            int id[kIds];
#pragma unroll
            for (int k = 0; k < kIds; ++k) {
                const int i = i0 + k * kLogitThreads;
                id[k] = i < hist ? h[i] : -1;
            }
#pragma unroll
            for (int k = 0; k < kIds; ++k) {
                if (id[k] < first || id[k] - first >= len) continue;
                const int at = id[k] - first + lead;
                const bool in_prompt = i0 + k * kLogitThreads < prompt;
                if ((in_prompt ? atomicOr(&words[at], 1u) : atomicAdd(&words[at], 2u)) == 0) push(at);
            }
        }
        __syncthreads();
        auto process = [&](int at) {
            const uint32_t y = __float_as_uint(process_one(LogitIo<T>::get(xb[at]), words[at], rep, pres, freq, a.bias_vals + b0));
            words[at] = y == kLogitDone ? 0x7FFFFFFFu ^ kLogitDone : y ^ kLogitDone;
        };
        const int total = s_count;
        if (total <= kLogitList) {
            for (int i = tid; i < total; i += kLogitThreads) process(s_list[i]);
        } else {
            for (int at = tid; at < nvec * kVec; at += kLogitThreads)
                if (words[at]) process(at);
        }
        __syncthreads();
    }
    const bool even = first >= lead && ((first - lead) & (kVec - 1)) == 0;  // no vector's bits reach into the next word
    auto mask_bits = [&](int j) {
        // (a first vector may begin before token 0, a last one end behind the last word: no tokens there)
        const int at = first - lead + j * kVec, g = max(at, 0), sh = g & 31;
        const uint32_t lo = __ldg(mask + (g >> 5));
        if (even) return lo >> sh;
        const uint32_t hi = sh + kVec > 32 && (g >> 5) + 1 < a.mask_words ? __ldg(mask + (g >> 5) + 1) : 0u;
        return __funnelshift_r(lo, hi, sh) << (g - at);
    };
    float best_v = 0.0f;  // the thread's best so far and the first vector it was in (they come in ascending order)
    int best_j = -1;
    for (int j0 = 0; j0 < nvec; j0 += kLogitBatch * kLogitThreads) {
        if (j0 > 0) {
#pragma unroll
            for (int i = 0; i < kLogitBatch; ++i) {
                const int j = j0 + tid + i * kLogitThreads;
                if (j < nvec) batch[i] = load(j);
            }
        }
        uint32_t allow[kLogitBatch];  // each vector's mask bits
        if (mask) {
#pragma unroll
            for (int i = 0; i < kLogitBatch; ++i) {
                const int j = j0 + tid + i * kLogitThreads;
                if (j < nvec) allow[i] = mask_bits(j);
            }
        }
#pragma unroll
        for (int i = 0; i < kLogitBatch; ++i) {
            const int j = j0 + tid + i * kLogitThreads;
            if (j >= nvec) break;
            __align__(16) T v[kVec];
            *reinterpret_cast<uint4*>(v) = batch[i];
            float f[kVec];
#pragma unroll
            for (int k = 0; k < kVec; ++k) f[k] = LogitIo<T>::get(v[k]);
            if (touched) {
#pragma unroll
                for (int k = 0; k < kVec; k += 4) {
                    const uint4 w = reinterpret_cast<const uint4*>(words)[(j * kVec + k) / 4];
                    if (w.x) f[k] = __uint_as_float(w.x ^ kLogitDone);
                    if (w.y) f[k + 1] = __uint_as_float(w.y ^ kLogitDone);
                    if (w.z) f[k + 2] = __uint_as_float(w.z ^ kLogitDone);
                    if (w.w) f[k + 3] = __uint_as_float(w.w ^ kLogitDone);
                }
            }
            if (mask) {
#pragma unroll
                for (int k = 0; k < kVec; ++k)
                    if (!(allow[i] & (1u << k))) f[k] = -INFINITY;
            }
#pragma unroll
            for (int k = 0; k < kVec; ++k) {
                v[k] = LogitIo<T>::put(f[k]);
                f[k] = LogitIo<T>::get(v[k]);
            }
            if (j >= full0 && j < full1 && same) {
                __stcs(reinterpret_cast<uint4*>(yb) + j, *reinterpret_cast<const uint4*>(v));
            } else {
#pragma unroll
                for (int k = 0; k < kVec; ++k) {
                    const int e = j * kVec + k;
                    if (e >= lead && e < lead + len) yb[e] = v[k];
                    else f[k] = -INFINITY;  // another tile's, or nobody's: no candidate
                }
            }
            float top = f[0];
#pragma unroll
            for (int k = 1; k < kVec; ++k) top = max_nan(top, f[k]);
            // once it is NaN it stays
            if (best_j < 0 || (!(top <= best_v) && best_v == best_v)) {
                best_v = top;
                best_j = j;
            }
        }
    }
    if (!a.keys) return;
    const uint64_t mine = best_j < 0 ? 0ull : best_key(best_v, static_cast<uint32_t>(best_j));
    uint64_t best = mine;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const uint64_t other = __shfl_xor_sync(0xffffffffu, best, o);
        best = other > best ? other : best;
    }
    if ((tid & 31) == 0) s_best[tid >> 5] = best;
    __syncthreads();
    best = s_best[0];
    for (int i = 1; i < kLogitThreads / 32; ++i) best = s_best[i] > best ? s_best[i] : best;
    if (mine == best) {  // the one thread with that vector finds the token in what it has written
        int at = -1;
        for (int k = 0; k < kVec; ++k) {
            const int e = best_j * kVec + k;
            if (at >= 0 || e < lead || e >= lead + len) continue;
            const float u = LogitIo<T>::get(yb[e]);
            if (u == best_v || (u != u && best_v != best_v)) at = e;
        }
        a.keys[blockIdx.x] = best_key(best_v, static_cast<uint32_t>(t0 + at - lead));
    }
}

// One warp per row: the best of its tiles.
template <typename T>
__global__ void __launch_bounds__(128) k_best_token(const uint64_t* __restrict__ keys, int64_t rows, int tiles,
                                                    int64_t begin, int64_t* __restrict__ best, T* __restrict__ value) {
    pdl_launch_dependents();
    pdl_wait();
    const int64_t row = blockIdx.x * 4ll + (threadIdx.x >> 5);
    if (row >= rows) return;
    uint64_t k = 0;
    for (int i = threadIdx.x & 31; i < tiles; i += 32) {
        const uint64_t other = keys[row * tiles + i];
        k = other > k ? other : k;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const uint64_t other = __shfl_xor_sync(0xffffffffu, k, o);
        k = other > k ? other : k;
    }
    if ((threadIdx.x & 31) == 0) {
        if (best) best[row] = begin + static_cast<int64_t>(0xFFFFFFFFu - static_cast<uint32_t>(k));
        if (value) {
            const uint32_t ord = static_cast<uint32_t>(k >> 32);
            const uint32_t bits = ord == 0xFFFFFFFFu ? 0x7FFFFFFFu : (ord & 0x80000000u) ? ord & 0x7FFFFFFFu : ~ord;
            value[row] = LogitIo<T>::put(__uint_as_float(bits));
        }
    }
}

// Tiles of a row: as many as fill the SMs (four CTAs each) a whole number of times with tiles that their words
// allow, and none below kLogitMinTile tokens.
static int logit_tiles(int64_t rows, int64_t vocab, int* tile) {
    const int64_t slots = 4ll * sm_count();
    int64_t tiles = 0;
    for (int64_t k = 1; tiles * kLogitWords < vocab; ++k) {
        tiles = k * slots / rows;
        if (k > 64) tiles = (vocab + kLogitWords - 1) / kLogitWords;  // very many rows: nothing to balance
    }
    const int64_t most = (vocab + kLogitMinTile - 1) / kLogitMinTile;
    if (tiles > most) tiles = most;
    *tile = static_cast<int>(((vocab + tiles - 1) / tiles + 7) / 8 * 8);
    return static_cast<int>((vocab + *tile - 1) / *tile);
}

template <typename T>
static cudaError_t launch_logits(const LogitArgs& a, int64_t rows, int64_t* best, void* value, cudaStream_t s) {
    const size_t smem = static_cast<size_t>(a.tile + 2 * LogitIo<T>::kVec) * 4;
    cudaError_t e = launch_pdl(k_process_logits<T>, dim3(static_cast<unsigned>(rows * a.tiles)), dim3(kLogitThreads), smem, s, a);
    if (e == cudaSuccess && a.keys)
        e = launch_pdl(k_best_token<T>, dim3(static_cast<unsigned>((rows + 3) / 4)), dim3(128), 0, s, a.keys, rows, a.tiles,
                       a.begin, best, static_cast<T*>(value));
    return e;
}

}  // namespace sc

using namespace sc;

extern "C" {

size_t sc_qwen2_process_logits_scratch(int64_t rows, int64_t vocab) {
    if (rows <= 0 || rows > kLogitMaxRows || vocab <= 0 || vocab > (1ll << 30)) return 0;
    int tile;
    return static_cast<size_t>(rows) * logit_tiles(rows, vocab, &tile) * 8;
}

sc_status sc_qwen2_process_logits(const void* logits, int dtype, int64_t rows, int64_t vocab, int64_t stride,
                                  int64_t vocab_begin, const int32_t* history, int64_t history_stride,
                                  const int32_t* prompt_len, const int32_t* hist_len, const float* repetition,
                                  const float* presence, const float* frequency, const int32_t* bias_ptr,
                                  const int32_t* bias_ids, const float* bias_vals, int64_t num_bias,
                                  const int32_t* mask, int64_t mask_words, int64_t mask_rows, const int32_t* mask_row,
                                  void* out, int64_t out_stride, int64_t* best, void* best_value, void* scratch,
                                  size_t scratch_bytes, uint32_t* status, void* stream) {
    auto bad = [](const char* what) {
        set_error(std::string("sc_qwen2_process_logits: ") + what);
        return SC_EINVAL;
    };
    if (dtype != SC_F32 && dtype != SC_F16 && dtype != SC_BF16) return bad("dtype is f32, f16 or bf16");
    if (rows < 0 || vocab <= 0 || vocab > (1ll << 30) || rows > kLogitMaxRows) return bad("rows or vocab out of range");
    if (vocab_begin < 0 || vocab_begin > (1ll << 30) - vocab) return bad("vocab_begin out of range");
    if (rows == 0) return SC_OK;
    if (!logits || !out) return bad("null logits or out");
    if (rows > 1 && (stride < vocab || out_stride < vocab)) return bad("rows overlap");
    if (history && (!hist_len || history_stride < 0)) return bad("a history needs its lengths");
    if (history && history_stride > kLogitMaxHistory) return bad("a history of more than 524287 tokens");
    if (bias_ptr && num_bias > 0 && (!bias_ids || !bias_vals)) return bad("bias entries need their ids and values");
    if (bias_ptr && num_bias < 0) return bad("a negative number of bias entries");
    if (mask && (mask_words < (vocab_begin + vocab + 31) / 32 || mask_rows < 0))
        return bad("a mask must cover the vocabulary");
    if (mask && !mask_row && mask_rows < rows) return bad("fewer masks than rows");
    const intptr_t size = dtype == SC_F32 ? 4 : 2;
    if (ranges_meet(logits, ((rows - 1) * stride + vocab) * size, out, ((rows - 1) * out_stride + vocab) * size)) {
        // in place, or columns of one buffer beside each other
        const intptr_t apart = reinterpret_cast<intptr_t>(out) - reinterpret_cast<intptr_t>(logits);
        intptr_t between = rows > 1 ? apart % (stride * size) : apart;
        if (between < 0) between += stride * size;
        if (rows > 1 && stride != out_stride) return bad("out lies over logits with another stride");
        if (apart != 0 && (rows == 1 || between < vocab * size || between > (stride - vocab) * size))
            return bad("out lies over logits, but not in place");
    }
    if ((reinterpret_cast<uintptr_t>(logits) | reinterpret_cast<uintptr_t>(out)) % size)
        return bad("logits and out must be aligned to their type");
    LogitArgs a = {};
    a.x = logits;
    a.vocab = vocab;
    a.stride = stride;
    a.begin = vocab_begin;
    a.history = history_stride > 0 ? history : nullptr;
    a.history_stride = history_stride;
    a.prompt_len = prompt_len;
    a.hist_len = hist_len;
    a.rep = repetition;
    a.pres = presence;
    a.freq = frequency;
    a.bias_ptr = num_bias > 0 ? bias_ptr : nullptr;
    a.bias_ids = bias_ids;
    a.bias_vals = bias_vals;
    a.num_bias = num_bias;
    a.mask = reinterpret_cast<const uint32_t*>(mask);
    a.mask_words = mask_words;
    a.mask_rows = mask_rows;
    a.mask_row = mask_row;
    a.out = out;
    a.out_stride = out_stride;
    a.status = status;
    a.tiles = logit_tiles(rows, vocab, &a.tile);
    if (rows * a.tiles > 0x7fffffff) return bad("rows or vocab out of range");
    if (best || best_value) {
        if (!scratch || reinterpret_cast<uintptr_t>(scratch) % 8) return bad("scratch must be 8-byte aligned");
        if (scratch_bytes < static_cast<size_t>(rows) * a.tiles * 8) {
            set_error("sc_qwen2_process_logits: scratch too small");
            return SC_ENOMEM;
        }
        a.keys = static_cast<uint64_t*>(scratch);
    }
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const cudaError_t e = dtype == SC_F32   ? launch_logits<float>(a, rows, best, best_value, s)
                          : dtype == SC_F16 ? launch_logits<__half>(a, rows, best, best_value, s)
                                            : launch_logits<__nv_bfloat16>(a, rows, best, best_value, s);
    return e == cudaSuccess ? SC_OK : cuda_fail(e, "sc_qwen2_process_logits");
}

}  // extern "C"
