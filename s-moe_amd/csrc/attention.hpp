// attention.hpp -- host-side launchers of the row, prompt and 4-bit-cache
// attention kernels (internal to libsmoe_hip.so; the public surface is
// include/smoe_hip.h).  The entry points (attention.cpp) have checked every
// size, stride and alignment; what only the device sees (offsets, slots,
// positions, lengths) the kernels check themselves and report in `err`.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace smoe {

// error word: a row offset, slot, position or length outside its buffer
constexpr uint32_t ERR_ATTN_RANGE = 8u;

// Scratch of a call whose keys are split: (maximum, sum) of every row and part, then
// (from a multiple of 16 bytes on) its weighted V.
__host__ __device__ constexpr size_t part_acc_at(size_t rows, uint32_t splits) { return (2 * rows * splits + 3) & ~size_t(3); }
__host__ __device__ constexpr size_t part_floats(size_t rows, uint32_t splits, uint32_t head_dim)
{
    return part_acc_at(rows, splits) + rows * splits * head_dim;
}

// RMSNorm and RoPE of n_rows query and key rows (attn_rows.hip); strides in elements
struct QkRows {
    const void* q;
    void* q_out;
    const void* k;
    void* k_out;
    const uint16_t* q_norm_w;
    const uint16_t* k_norm_w;
    const float* rope_cos;
    const float* rope_sin;
    const int32_t* positions;
    uint64_t q_stride, q_out_stride, k_stride, k_out_stride;
    uint32_t n_rows, n_positions, num_heads, num_kv_heads;   // heads 0: no such rows
    uint32_t* err;
};
hipError_t launch_qk_rows(const QkRows& a, uint32_t head_dim, uint32_t type, hipStream_t s);

// the 4-bit cache: codes [slot][KV head][position][head_dim / 2], scale and
// min pairs [slot][KV head][position][head_dim / 64][2] in bf16
struct Kv4 {
    uint8_t* codes[2];       // K, V
    uint16_t* params[2];
    uint32_t n_slots, capacity, num_kv_heads;
};
// packed rows of n_seqs sequences against cache positions from start[b] on (attn_rows.hip)
struct Kv4Rows {
    Kv4 c;
    void* rows[2];           // K, V
    uint64_t stride[2];      // elements
    const int32_t* offsets;  // [n_seqs + 1], or one row a sequence
    const int32_t* slots;    // [n_seqs], or sequence b in slot b
    const int32_t* start;    // [n_seqs]
    int32_t* lens_out;
    uint32_t n_seqs, n_rows;
    uint32_t* err;
};
hipError_t launch_kv4_append(const Kv4Rows& a, uint32_t head_dim, uint32_t type, hipStream_t s);
hipError_t launch_kv4_read(const Kv4Rows& a, uint32_t head_dim, uint32_t type, hipStream_t s);

// causal attention of packed sequences (attn_prompt.hip); strides in elements
struct PromptAttn {
    const void* q;
    const void* k;
    const void* v;
    void* out;
    const int32_t* q_offsets;   // [n_seqs + 1]
    const int32_t* k_offsets;
    uint64_t q_stride, k_stride, v_stride, out_stride;
    uint32_t n_seqs, q_rows, k_rows, num_kv_heads, group;
    float scale_log2;           // score scale times log2(e)
    uint32_t tiles;             // row tiles, at most (prompt_plan)
    uint32_t row_waves;         // waves of 32 rows of a block's row tile
    uint32_t key_groups;        // groups of such waves that take the tile's keys in turn
    uint32_t splits;            // parts of a sequence's keys, joined by a second launch
    float* part;                // rows = query rows times heads (part_floats)
    uint32_t plane_tiles;       // f32: tiles of 32 keys, at most, that share a power of two; else 0
    uint16_t* planes;           // f32: K hi, K lo, V hi, V lo [k_rows][KV heads][head_dim] f16
    int2* powers;               // f32: [KV heads][plane_tiles] powers of K and of V
    uint32_t* err;
};
// tiles and splits of a call (max_k: the longest sequence's keys as far as the caller knows), and its scratch
void prompt_plan(PromptAttn& a, uint32_t head_dim, uint32_t type, uint32_t max_k);
size_t prompt_scratch_bytes(const PromptAttn& a, uint32_t head_dim);
void prompt_scratch(PromptAttn& a, uint32_t head_dim, void* scratch);
hipError_t launch_attention_prompt(const PromptAttn& a, uint32_t head_dim, uint32_t type, hipStream_t s);

// attention of one token a sequence over the 4-bit cache (attn_kv4.hip); strides in elements
struct Kv4Attn {
    Kv4 c;
    const void* q;
    void* out;
    const int32_t* slots;       // [n_seqs], or sequence b in slot b
    const int32_t* lens;        // [n_seqs]
    uint64_t q_stride, out_stride;
    uint32_t n_seqs, group;     // group: query heads per KV head
    float scale_log2;
    uint32_t units;             // parts of all sequences' positions for a KV head, joined by a second launch;
                                // 0: each sequence whole
    uint32_t waves;             // of a block: 4 or 8
    float* part;                // rows = units times heads (part_floats, one part a row)
    uint32_t* err;
};
void kv4_plan(Kv4Attn& a, uint32_t head_dim, uint32_t max_len);
size_t kv4_scratch_bytes(const Kv4Attn& a, uint32_t head_dim);
hipError_t launch_attention_kv4(const Kv4Attn& a, uint32_t head_dim, uint32_t type, hipStream_t s);

}  // namespace smoe
