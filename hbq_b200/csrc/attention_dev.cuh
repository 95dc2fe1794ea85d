// What the attention kernels share: which keys a row sees, and the form in which parts of a row's sum are joined.
#pragma once
#include "common.cuh"
#include <cuda.h>

namespace hbq {

struct AttnArgs {
    const void *q, *k, *v, *pk, *pv;
    void* out;
    const int32_t *lengths, *starts;
    int64_t qs[3], ks[3], vs[3], os[3], pks[2], pvs[2];      // strides in elements
    int64_t S, P, window, sinks;
    uint32_t B, L, H, Hkv, G, D;
    float scale_log2;                                        // scale * log2(e)
    int nsplit;                                              // (tensor-core kernel) pieces of a block's keys
    float* part;                                             // [rows][parts][D] sums, then [rows][parts] (maximum, weight)
    int parts, part0;
    // The few-row kernel's division of work: `blocks` blocks of equal shares; its table and slots in the workspace.
    int blocks, shared;                                      // shared: shares may begin and end inside a row group
    int cluster;                                             // else: the blocks of a cluster, which share one group
    int beside;                                              // second kernel of a call: runs beside the first (begin_beside)
    int2* table;                                             // of each row group: its first block and how many; 0: undivided
    float* slots;                                            // [blocks][2][16][D] sums, then [blocks][2][16] (maximum, weight)
};

// Rows of sequence b: its keys, and the position of its first row.
__device__ __forceinline__ void sequence_of(const AttnArgs& a, uint32_t b, int64_t* n, int64_t* first)
{
    int64_t len = a.lengths ? (int64_t)__ldcg(a.lengths + b) : a.S;
    len = len < 0 ? 0 : len > a.S ? a.S : len;
    *n = len;
    *first = a.starts ? (int64_t)__ldcg(a.starts + b) : len - (int64_t)a.L;
}

// Weights are 2^(score - maximum + SHIFT), and up to 2^GROWTH more until the sums are rescaled.  In fp16 2^4 keeps 16 times smaller
// ones normal, and 2^(4 + 8) stays below the largest.  bf16 has room below, not above: its values go up to 2^128, and 2^24 of them
// at weights of 2^-24 sum up inside 32 bits.
constexpr float GROWTH = 8.f;
template <class E> struct Weights;
template <> struct Weights<__half> { static constexpr float SHIFT = 4.f; };
template <> struct Weights<__nv_bfloat16> { static constexpr float SHIFT = -24.f; };

__device__ __forceinline__ float exp2_fast(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// What a sum is multiplied by when its maximum is exceeded, or when it is joined: never zero, since the sum may be an infinity that a row
// sees.  The smallest number there is, 2^-149, adds below 2^-20 to others.
__device__ __forceinline__ float factor_of(float x) { return fmaxf(exp2_fast(x), __uint_as_float(1u)); }

// The second of a call's two attention kernels reads nothing that the first writes, and the first lets it start only behind its
// own wait, when all before it is complete: it need not wait for the first, and fills the SMs that the first leaves.  It
// waits at its end instead (its inputs come from L2, past what an SM's cache may hold of them from before), so that the kernel behind it, which joins both kernels' parts, finds both complete.
__device__ __forceinline__ void begin_beside(const AttnArgs& a)
{
    if (!a.beside) { grid_dependency_wait(); dependents_may_start(); }
}
__device__ __forceinline__ void end_beside(const AttnArgs& a)
{
    if (a.beside) { grid_dependency_wait(); dependents_may_start(); }
}

// A part's sums and (maximum, weight) of a row; rows are numbered (b * L + i) * H + h.
__device__ __forceinline__ float* part_sum(const AttnArgs& a, int64_t row, int part) { return a.part + (row * a.parts + part) * a.D; }
__device__ __forceinline__ float2* part_weight(const AttnArgs& a, int64_t row, int part)
{
    return reinterpret_cast<float2*>(a.part + (int64_t)a.B * a.L * a.H * a.parts * a.D) + row * a.parts + part;
}

// The few-row kernel's units of work: 64 keys of one row group (16 heads of a key head, one token).  A token's groups all
// have the same number of units.
// Block c of n has units total * c / n up to total * (c + 1) / n; no more blocks take part than there are units, so that each
// has some and a group's blocks follow one another.
__device__ __forceinline__ int64_t rows_takers(const AttnArgs& a, int64_t total) { return total < a.blocks ? total : a.blocks; }
__device__ __forceinline__ int rows_owner(int64_t unit, int64_t total, int64_t takers) { return (int)(((unit + 1) * takers - 1) / total); }
__device__ __forceinline__ float* slot_sum(const AttnArgs& a, int block, int which, int row) { return a.slots + ((int64_t)(block * 2 + which) * 16 + row) * a.D; }
__device__ __forceinline__ float2* slot_weight(const AttnArgs& a, int block, int which, int row)
{
    return reinterpret_cast<float2*>(a.slots + (int64_t)a.blocks * 2 * 16 * a.D) + (block * 2 + which) * 16 + row;
}

// attention_rows.cu
int attention_rows_launch(const AttnArgs& a, int dtype, cudaStream_t stream);
int attention_join_launch(const AttnArgs& a, int dtype, cudaStream_t stream);
int attention_rows_blocks(const hbq_attention* p, bool prefix, int* shared, int* cluster, bool* small);
// attention_tc.cu
int attention_tc_launch(AttnArgs& a, int dtype, bool prefix, cudaStream_t stream);
int attention_tc_parts(const hbq_attention* p, bool prefix);
int attention_cache_map(CUtensorMap* map, const void* ptr, int dtype, int64_t D, int rows, int64_t keys, int64_t key_stride, int64_t heads,
                        int64_t head_stride, int64_t seqs, int64_t seq_stride);

}  // namespace hbq
