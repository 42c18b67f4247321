// sc_logits.cu -- penalties, biases and grammar masks on logits, with the best token of each row.
//
// Per token v of a row, in f32 and rounded once to the logits' type:
//   x1 = seen(v) ? (x > 0 ? x / r : x * r) : x          seen: v occurs in the row's history
//   x2 = x1 - f * n(v) - (n(v) > 0 ? p : 0)             n: times v occurs among the generated tokens
//   x3 = x2 + b(v)                                      b: the last bias entry of v
//   y  = allowed(v) ? x3 : -inf
// One pass: each logit is read once and written once; the floor is rows * vocab * 2 * size bytes.
//
// A row belongs to one thread-block cluster, each CTA of it to a slice of the vocabulary.  The
// counts n(v) of a slice live in the CTA's shared memory, one word per token: history ids are read
// once per row (each CTA takes its share of them) and counted by remote shared-memory atomics into
// the CTA that owns the token, so nothing of vocabulary size ever goes to global memory.  Integer
// atomics only: the result does not depend on their order.
//   word = (bias entry + 1) << 20 | n << 1 | in the prompt
// Each CTA issues the loads of its first logits before it counts, so that they arrive meanwhile.
#include <cooperative_groups.h>

#include <atomic>
#include <string>

#include "saccade_qwen2.h"
#include "sc_device.cuh"
#include "sc_internal.h"

namespace sc {

constexpr int kLogitThreads = 512;
constexpr int kLogitWords = 20480;        // tokens of one CTA's slice at a time (80 KB of words: two CTAs per SM)
constexpr int kLogitBatch = 6;            // 16-byte loads a thread has in flight
constexpr int kLogitMaxCluster = 8;
constexpr int64_t kLogitMaxHistory = (1 << 19) - 1;  // 19 bits of a word count occurrences
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
    int64_t slice;    // tokens of one CTA and chunk, at most kLogitWords
    int chunks;       // chunks of cluster * slice tokens
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

__device__ __forceinline__ void red_add_cluster(uint32_t addr, uint32_t v) {
    asm volatile("red.relaxed.cluster.shared::cluster.add.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}
__device__ __forceinline__ void red_or_cluster(uint32_t addr, uint32_t v) {
    asm volatile("red.relaxed.cluster.shared::cluster.or.b32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}
__device__ __forceinline__ void st_cluster_u64(uint32_t addr, uint64_t v) {
    asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(addr), "l"(v) : "memory");
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
__global__ void __launch_bounds__(kLogitThreads, 2) k_process_logits(const LogitArgs a) {
    constexpr int kVec = LogitIo<T>::kVec;
    extern __shared__ __align__(16) uint32_t words[];  // [slice, rounded up to kVec, + kVec]
    __shared__ uint64_t s_best[kLogitThreads / 32];
    __shared__ uint64_t s_all[kLogitMaxCluster];
    pdl_launch_dependents();
    pdl_wait();
    const int rank = static_cast<int>(cluster_rank());
    const int cn = static_cast<int>(cooperative_groups::this_cluster().num_blocks());
    const int64_t row = blockIdx.x / cn;
    const int tid = threadIdx.x;
    const T* x = static_cast<const T*>(a.x) + row * a.stride;
    T* y = static_cast<T*>(a.out) + row * a.out_stride;

    // the row's parameters
    const float rep = a.rep ? a.rep[row] : 1.0f, pres = a.pres ? a.pres[row] : 0.0f, freq = a.freq ? a.freq[row] : 0.0f;
    int64_t hist = 0, prompt = 0;
    if (a.history) {
        hist = a.hist_len[row];
        prompt = a.prompt_len ? a.prompt_len[row] : 0;
        if (hist < 0 || hist > a.history_stride || prompt < 0 || prompt > hist) {
            if (tid == 0 && rank == 0) record_error(a.status, DEV_BAD_INDEX);
            hist = hist < 0 ? 0 : imin64(hist, a.history_stride);
            prompt = prompt < 0 ? 0 : imin64(prompt, hist);
        }
        if (rep == 1.0f && pres == 0.0f && freq == 0.0f) hist = prompt = 0;  // counts change nothing
    }
    int64_t b0 = 0, b1 = 0;
    if (a.bias_ptr) {
        b0 = a.bias_ptr[row];
        b1 = a.bias_ptr[row + 1];
        if (b0 < 0 || b1 < b0 || b1 > a.num_bias || b1 - b0 > kLogitMaxBias) {
            if (tid == 0 && rank == 0) record_error(a.status, DEV_BAD_INDEX);
            b0 = b0 < 0 ? 0 : imin64(b0, a.num_bias);
            b1 = b1 < b0 ? b0 : imin64(imin64(b1, a.num_bias), b0 + kLogitMaxBias);
        }
    }
    const uint32_t* mask = nullptr;
    if (a.mask) {
        int64_t m = a.mask_row ? a.mask_row[row] : row;
        if (m >= a.mask_rows) {
            if (tid == 0 && rank == 0) record_error(a.status, DEV_BAD_INDEX);
            m = -1;
        }
        if (m >= 0) mask = a.mask + m * a.mask_words;
    }
    const bool touched = hist > 0 || b1 > b0;  // the same in every CTA of the cluster

    uint64_t best = 0;
    for (int c = 0; c < a.chunks; ++c) {
        // this CTA's tokens [t0, t1) of the slice; vector j covers tokens t0 - lead + j * kVec .. + kVec, so
        // that it starts on a 16-byte boundary of the row
        const int64_t t0 = imin64(a.vocab, (static_cast<int64_t>(c) * cn + rank) * a.slice);
        const int64_t t1 = imin64(a.vocab, t0 + a.slice);
        const int lead = static_cast<int>((reinterpret_cast<uintptr_t>(x + t0) & 15u) / sizeof(T));
        const bool same = (reinterpret_cast<uintptr_t>(y + t0) & 15u) == lead * sizeof(T);
        const int nvec = t1 > t0 ? static_cast<int>((t1 - t0 + lead + kVec - 1) / kVec) : 0;
        auto load = [&](int j) {
            uint4 r = make_uint4(0, 0, 0, 0);
            const int64_t e = t0 - lead + static_cast<int64_t>(j) * kVec;
            if (e >= t0 && e + kVec <= t1) {
                r = __ldcs(reinterpret_cast<const uint4*>(x + e));
            } else {  // the slice's first or last vector
                __align__(16) T v[kVec];
#pragma unroll
                for (int k = 0; k < kVec; ++k) v[k] = (e + k >= t0 && e + k < t1) ? x[e + k] : T(0.0f);
                r = *reinterpret_cast<const uint4*>(v);
            }
            return r;
        };
        uint4 batch[kLogitBatch];
#pragma unroll
        for (int i = 0; i < kLogitBatch; ++i) {
            const int j = tid + i * kLogitThreads;
            if (j < nvec) batch[i] = load(j);
        }
        if (touched) {
            for (int i = tid; i < (nvec * kVec + 3) / 4; i += kLogitThreads)
                reinterpret_cast<uint4*>(words)[i] = make_uint4(0, 0, 0, 0);
            __syncthreads();
            // every CTA goes over all of the row's bias entries (at most 4095) for its own tokens
            for (int64_t i = b0 + tid; i < b1; i += kLogitThreads) {
                const int64_t v = a.bias_ids[i] - a.begin;
                if (v >= t0 && v < t1) atomicMax(&words[v - t0 + lead], static_cast<uint32_t>(i - b0 + 1) << 20);
            }
            __syncwarp();
            cluster_sync();
            // its share of the history goes to the owners' words
            const uint32_t base = smem_u32(words);
            const int64_t c0 = static_cast<int64_t>(c) * cn * a.slice;
            for (int64_t i = static_cast<int64_t>(rank) * kLogitThreads + tid; i < hist;
                 i += static_cast<int64_t>(cn) * kLogitThreads) {
                const int64_t v = a.history[row * a.history_stride + i] - a.begin;
                if (v < c0 || v >= a.vocab || v - c0 >= cn * a.slice) continue;
                const int owner = static_cast<int>((v - c0) / a.slice);
                const int64_t o0 = c0 + owner * a.slice;
                const int olead = static_cast<int>((reinterpret_cast<uintptr_t>(x + o0) & 15u) / sizeof(T));
                uint32_t addr;
                asm("mapa.shared::cluster.u32 %0, %1, %2;"
                    : "=r"(addr)
                    : "r"(base + static_cast<uint32_t>(v - o0 + olead) * 4), "r"(owner));
                if (i < prompt) red_or_cluster(addr, 1u);
                else red_add_cluster(addr, 2u);
            }
            __syncwarp();
            cluster_sync();
        }
        for (int j0 = 0; j0 < nvec; j0 += kLogitBatch * kLogitThreads) {
            if (j0 > 0) {
#pragma unroll
                for (int i = 0; i < kLogitBatch; ++i) {
                    const int j = j0 + tid + i * kLogitThreads;
                    if (j < nvec) batch[i] = load(j);
                }
            }
#pragma unroll
            for (int i = 0; i < kLogitBatch; ++i) {
                const int j = j0 + tid + i * kLogitThreads;
                if (j >= nvec) continue;
                __align__(16) T v[kVec];
                *reinterpret_cast<uint4*>(v) = batch[i];
                const int64_t e = t0 - lead + static_cast<int64_t>(j) * kVec;
                uint32_t w[kVec];
#pragma unroll
                for (int k = 0; k < kVec / 4; ++k)
                    *reinterpret_cast<uint4*>(w + 4 * k) =
                        touched ? reinterpret_cast<const uint4*>(words)[j * (kVec / 4) + k] : make_uint4(0, 0, 0, 0);
                uint32_t allowed = 0xFFFFFFFFu;
                if (mask) {  // bits e + begin .. + kVec (a first vector may begin before the slice)
                    const int64_t g = e + a.begin < 0 ? 0 : e + a.begin;
                    const uint32_t lo = mask[g >> 5];
                    const int sh = static_cast<int>(g & 31);
                    const uint32_t hi = sh + kVec > 32 && (g >> 5) + 1 < a.mask_words ? mask[(g >> 5) + 1] : 0u;
                    allowed = __funnelshift_r(lo, hi, sh) << (g - (e + a.begin));
                }
#pragma unroll
                for (int k = 0; k < kVec; ++k) {
                    float f = LogitIo<T>::get(v[k]);
                    if (w[k]) f = process_one(f, w[k], rep, pres, freq, a.bias_vals + b0);
                    if (!((allowed >> k) & 1u)) f = -INFINITY;
                    v[k] = LogitIo<T>::put(f);
                    if (a.best || a.best_value) {
                        if (e + k >= t0 && e + k < t1) {
                            const uint64_t key = best_key(LogitIo<T>::get(v[k]), static_cast<uint32_t>(e + k));
                            best = key > best ? key : best;
                        }
                    }
                }
                if (same && e >= t0 && e + kVec <= t1) {
                    __stcs(reinterpret_cast<uint4*>(y + e), *reinterpret_cast<const uint4*>(v));
                } else {
#pragma unroll
                    for (int k = 0; k < kVec; ++k)
                        if (e + k >= t0 && e + k < t1) y[e + k] = v[k];
                }
            }
        }
        // the words are zeroed again for the next chunk, and no CTA counts into them before that: its
        // cluster barrier after the zeroing
        if (c + 1 < a.chunks && touched) __syncthreads();
    }
    if (!a.best && !a.best_value) return;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const uint64_t other = __shfl_xor_sync(0xffffffffu, best, o);
        best = other > best ? other : best;
    }
    if ((tid & 31) == 0) s_best[tid >> 5] = best;
    __syncthreads();
    if (tid == 0) {
        for (int i = 1; i < kLogitThreads / 32; ++i) best = s_best[i] > best ? s_best[i] : best;
        st_cluster_u64(dsmem_addr(&s_all[rank], 0), best);
    }
    __syncwarp();
    cluster_sync();
    if (rank == 0 && tid == 0) {
        for (int i = 0; i < cn; ++i) best = s_all[i] > best ? s_all[i] : best;
        const int64_t at = static_cast<int64_t>(0xFFFFFFFFu - static_cast<uint32_t>(best));
        if (a.best) a.best[row] = at + a.begin;
        if (a.best_value) {
            const uint32_t ord = static_cast<uint32_t>(best >> 32);
            const uint32_t bits = ord == 0xFFFFFFFFu ? 0x7FFFFFFFu : (ord & 0x80000000u) ? ord & 0x7FFFFFFFu : ~ord;
            static_cast<T*>(a.best_value)[row] = LogitIo<T>::put(__uint_as_float(bits));
        }
    }
}

template <typename T>
static cudaError_t launch_logits(LogitArgs a, int64_t rows, int sms, cudaStream_t s) {
    // CTAs of a row: as many as its words need; more, down to slices of 2048 tokens, while the launch
    // leaves SMs without their two CTAs
    int cn = 1;
    while (cn < kLogitMaxCluster && (a.vocab > static_cast<int64_t>(cn) * kLogitWords ||
                                     (rows * cn < 2 * sms && a.vocab >= static_cast<int64_t>(cn) * 4096)))
        cn *= 2;
    constexpr int kVec = LogitIo<T>::kVec;
    int64_t slice = ((a.vocab + cn - 1) / cn + kVec - 1) / kVec * kVec;
    if (slice > kLogitWords) slice = kLogitWords;
    a.slice = slice;
    a.chunks = static_cast<int>((a.vocab + cn * slice - 1) / (cn * slice));
    const size_t smem = static_cast<size_t>(slice + 2 * kVec) * 4;
    static std::atomic<uint64_t> flags{0};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    const uint64_t bit = 1ull << (dev & 63);
    if (!(flags.load() & bit)) {
        e = cudaFuncSetAttribute(k_process_logits<T>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 (kLogitWords + 2 * kVec) * 4);
        if (e != cudaSuccess) return e;
        flags.fetch_or(bit);
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(rows * cn));
    cfg.blockDim = dim3(kLogitThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = static_cast<unsigned>(cn);
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    g_launches.fetch_add(1, std::memory_order_relaxed);
    return cudaLaunchKernelEx(&cfg, k_process_logits<T>, a);
}

}  // namespace sc

using namespace sc;

extern "C" {

sc_status sc_qwen2_process_logits(const void* logits, int dtype, int64_t rows, int64_t vocab, int64_t stride,
                                  int64_t vocab_begin, const int32_t* history, int64_t history_stride,
                                  const int32_t* prompt_len, const int32_t* hist_len, const float* repetition,
                                  const float* presence, const float* frequency, const int32_t* bias_ptr,
                                  const int32_t* bias_ids, const float* bias_vals, int64_t num_bias,
                                  const int32_t* mask, int64_t mask_words, int64_t mask_rows, const int32_t* mask_row,
                                  void* out, int64_t out_stride, int64_t* best, void* best_value, uint32_t* status,
                                  void* stream) {
    auto bad = [](const char* what) {
        set_error(std::string("sc_qwen2_process_logits: ") + what);
        return SC_EINVAL;
    };
    if (dtype != SC_F32 && dtype != SC_F16 && dtype != SC_BF16) return bad("dtype is f32, f16 or bf16");
    if (rows < 0 || vocab <= 0 || vocab > (1ll << 30) || rows > (1ll << 27)) return bad("rows or vocab out of range");
    if (vocab_begin < 0 || vocab_begin > (1ll << 30)) return bad("vocab_begin out of range");
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
    const uintptr_t size = dtype == SC_F32 ? 4 : 2;
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
    a.best = best;
    a.best_value = best_value;
    a.status = status;
    int dev = 0, sms = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    if (e == cudaSuccess) {
        cudaStream_t s = static_cast<cudaStream_t>(stream);
        e = dtype == SC_F32 ? launch_logits<float>(a, rows, sms, s)
            : dtype == SC_F16 ? launch_logits<__half>(a, rows, sms, s)
                              : launch_logits<__nv_bfloat16>(a, rows, sms, s);
    }
    return e == cudaSuccess ? SC_OK : cuda_fail(e, "sc_qwen2_process_logits");
}

}  // extern "C"
