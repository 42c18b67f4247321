// sc_paged.cuh -- the paged KV cache as the kernels see it.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "sc_device.cuh"
#include "sc_internal.h"

namespace sc {

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

}  // namespace sc
