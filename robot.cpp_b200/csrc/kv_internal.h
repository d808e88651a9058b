// kv_internal.h -- the key/value cache's kernels as the C-ABI layer sees them (not exported).
#pragma once

#include <cstdint>
#include <cuda_runtime.h>

#include "b2s_common.cuh"

namespace b2s {

constexpr unsigned int kErrIndex = 4u;  // device error word: an index read from device memory was out of range

// A cache as the kernels see it. Row (page * kv_heads + head) * page_size + token holds hd code bytes and one scale.
struct KvView {
    uint8_t *k, *v;
    float *ks, *vs;
    int64_t n_pages;
    int kv_heads, hd, page_shift;
    bool e4m3;
};

// Pairs of a rotary embedding: the factor that takes a position to its angle in units of pi, and the axis.
struct RopePairs {
    double turn[128];
    uint8_t axis[128];
};

cudaError_t launch_rope_axes(bool bf16, const void* x, int64_t ldx, int64_t M, int n_heads, int hd, const int32_t* pos,
                             int64_t ldpos, const RopePairs& pairs, void* y, int64_t ldy, cudaStream_t st);
cudaError_t launch_kv_write(const KvView& c, bool bf16, const void* k, int64_t ldk, const void* v, int64_t ldv, int64_t M,
                            const int64_t* slots, cudaStream_t st);
cudaError_t launch_kv_read(const KvView& c, const int64_t* slots, int64_t M, bool bf16, void* k, int64_t ldk, void* v,
                           int64_t ldv, cudaStream_t st);

// Softmax state of query rows, one record for each (piece, row of q, query head): the reference exponent m (log2
// units), the sum l of 2^(s - m), and the unnormalised output 2^(s - m) V of hd floats.
struct AttnState {
    float *m, *l, *o;
    int pieces;
};

// One attention pass over one key range per sequence.
struct KvAttnArgs {
    KvView c;
    const void* q;
    void* o;
    int64_t ldq, ldo;
    int64_t M;               // rows of q and o
    int64_t q_stride;        // sequence b's rows: q_start[b * q_stride] .. q_start[(b + 1) * q_stride] - 1
    const int32_t* q_start;
    const int32_t* kv_len;   // nullptr: every sequence has kv_const tokens
    int64_t kv_const;
    const int32_t* pages;
    int64_t ld_pages, max_pages;
    int batch, heads, group;
    uint32_t group_mul, group_shift;
    __device__ __forceinline__ int by_group(int n) const {  // n / group, n >= 0
        return (int)((__umulhi((uint32_t)n, group_mul) + (uint32_t)n) >> group_shift);
    }
    int min_rows, max_rows;  // sequences with min_rows < query rows x group <= max_rows are taken, the others left alone
    float scale_log2e;       // scale * log2(e): scores are in log2 units
    int causal;
    bool bf16;
    bool to_state;           // write `out` instead of o (kv_attention_tc.cu alone)
    AttnState out;           // where it goes, one piece for each split of the keys
    AttnState add;           // joined with the result before it is written; pieces = 0: none
    float* part;             // split units' partial results and borders (kv_attention.cu)
    // kv_attention.cu alone
    bool whole_units;               // no unit is split
    const int32_t* prefix_pages;    // tokens in front of every sequence, read with its own
    int prefix_len, prefix_pad;     // prefix_pad: in whole tiles
};

// The rows that a pass over a shared prefix takes, from 0 on: up to the batch's last entry of q_start, or, where that is out of
// range, all. Sequences that reach past it find no state there and are left out.
__device__ __forceinline__ int rows_used(const KvAttnArgs& a, int end) { return end < 0 || end > a.M ? (int)a.M : end; }

// Few rows (kv_attention.cu).
size_t kv_attn_part_bytes();
cudaError_t launch_kv_attention(const KvAttnArgs& a, cudaStream_t st);

// Many rows (kv_attention_tc.cu): blocks of 128 rows, or (pair, bf16 only) of 256; their keys are cut into `splits` pieces,
// of which more than one need to_state. The join of out's and add's pieces into o.
cudaError_t launch_kv_attention_tc(const KvAttnArgs& a, bool pair, int splits, cudaStream_t st);
cudaError_t launch_kv_state_join(const KvAttnArgs& a, cudaStream_t st);

}  // namespace b2s
