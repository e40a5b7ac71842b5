// C ABI of the operators that serve drafted tokens: a key/value cache of bf16 rows or of 8-bit codes, attention of a tree of
// drafts over it, the accepted branch kept, constraints on logits.
#pragma once
#include <stddef.h>
#include <stdint.h>
#ifdef __cplusplus
extern "C" {
#endif

// A layer's cache: k, v [B, kv_heads, max_seq, head_dim], bf16 (bits 16) or int8 codes (bits 8) with an fp32 scale per row,
// k_scale, v_scale [B, kv_heads, max_seq].  A stored row stands for code * scale.
typedef struct MeshKvCache {
  void* k; void* v; float* k_scale; float* v_scale;
  int B, kv_heads, max_seq, head_dim, bits;
} MeshKvCache;

// Row t of sequence b, k[b, t, h, :] (bf16; strides in elements, the last dimension dense), goes to slot pos[b] + t for
// t < counts[b] (NULL: T).  Rows whose slot lies outside [0, max_seq) are not written.
int mesh_kv_append(const MeshKvCache* c, const void* k, const void* v, long long k_sb, long long k_st, long long k_sh,
                   long long v_sb, long long v_st, long long v_sh, const int* pos, const int* counts, int T, void* stream);
// out[b, t, h, :] (bf16, dense) = the row in slot start[b] + t for t < counts[b] (NULL: T); zero elsewhere and outside the cache.
int mesh_kv_read(const MeshKvCache* c, void* k_out, void* v_out, const int* start, const int* counts, int T, void* stream);
// In every one of n caches of the same geometry: slot pos[b] + i gets what slot pos[b] + path[b, i] held before the call, for
// i < counts[b] (NULL: N); N <= 64.  An entry whose two slots do not both lie in the cache, or path < 0, is left out.
int mesh_kv_keep(const MeshKvCache* caches, int n, const int* pos, const int* path, const int* counts, int N, void* stream);

// Attention of T <= 64 drafted tokens per sequence.  q, out [B, T, q_heads, head_dim] bf16 (strides of b and t in elements,
// heads dense).  Node t of sequence b lies in slot pos[b] + t.  It sees the slots before pos[b] (with window > 0 only those
// of positions > p - window, p = pos[b] + max(1, bits set in visible[b, t]) - 1) and node j when bit j of visible[b, t] is
// set (NULL: j <= t), j < counts[b] (NULL: T).  A node that sees nothing gets zeros; rows t >= counts[b] are not written.
// scratch: mesh_draft_attention_scratch() floats for these arguments (0: none needed).
typedef struct MeshDraftAttention {
  const void* q; void* out; long long q_sb, q_st, o_sb, o_st;
  const int* pos; const int* counts; const long long* visible;
  int T, q_heads, window, splits;     // splits: CTAs among which all keys are shared out; 0: as it pays
  float scale; float* scratch; void* status;
} MeshDraftAttention;
long long mesh_draft_attention_scratch(const MeshKvCache* c, const MeshDraftAttention* a);
int mesh_draft_attention(const MeshKvCache* c, const MeshDraftAttention* a, void* stream);

// Logits of `rows` rows over a vocabulary (shard) of `vocab` ids that starts at vocab_offset, fp32 or bf16, row stride ldl:
//   l = l > 0 ? l / repetition : l * repetition      for ids among history[0 .. history_len)
//   l = l - frequency * n - (n > 0 ? presence : 0)   n: times the id stands in history[prompt_len .. history_len)
//   l = l + bias                                     for ids among bias_ids[0 .. bias_len); of equal ids the last counts
//   l = -inf                                         where the id's bit in `allowed` is clear
// in fp32, each step rounded.  out (may be the logits, may be NULL): the result, in the type of the logits.  tokens (may be
// NULL): the id (global) of the largest result before it is rounded to that type, the lowest of equal ones, -1 when none is
// above -inf; NaN is never chosen.  repetition, presence, frequency [rows]; NULL where not used.
typedef struct MeshLogits {
  const void* logits; long long ldl; void* out; long long ldo; int half;
  int rows, vocab, vocab_offset;
  const int* history; long long ldh; int hist; const int* history_len; const int* prompt_len;
  const float* repetition; const float* presence; const float* frequency;
  const int* bias_ids; const float* bias; long long ldb; int nbias; const int* bias_len;
  const uint32_t* allowed; long long ldw;
  int* tokens;
} MeshLogits;
int mesh_constrain_logits(const MeshLogits* a, void* stream);

#ifdef __cplusplus
}
#endif
