// A paged cache of keys and values in 8 bits (e4m3), with a scale for each block of 16 tokens of a head, and what its kernels share.
#pragma once

#include "ma_rotary.cuh"
#include "ma_sm100.cuh"

namespace ma {

constexpr int kScaleBlock = 16;       // tokens that share a scale
constexpr float kLeastLog = -40.0f;   // of a scale that is not zero, to base 2

// Strides in elements of each tensor; the features of a row lie next to one another.
struct CacheArgs {
  uint8_t *k, *v;         // (pages, heads, page size, D) e4m3
  float *k_scale, *v_scale;  // (pages, heads, page size / 16)
  long long k_sp, k_sh, k_st, v_sp, v_sh, v_st;
  long long ks_sp, ks_sh, vs_sp, vs_sh;
  int pages, heads, page_shift;  // page size = 1 << page_shift
  const int* table;  // (E, table_pages) page of each run of page-size tokens
  long long table_se;
  int table_pages;
  const int* lengths;  // (E) tokens of a sequence, those of the call among them
  const int* counts;   // (E) tokens of a sequence in the call, or nullptr: N
  int* status;         // mapped host word: what was wrong with a table, length or count
};

enum CacheFault { kBadLength = 1, kBadPage = 2, kBadParent = 3, kBadSource = 4, kNoPage = 5 };

__device__ __forceinline__ void report(int* status, int code) {
  if (status != nullptr) *reinterpret_cast<volatile int*>(status) = code;
}

// Tokens of sequence e and how many of them the call brings, held to what the table and the call have room for; false if they had to be.
__device__ __forceinline__ bool sequence_of(const CacheArgs& c, int e, int N, int* len, int* count) {
  const int room = (int)min((long long)c.table_pages << c.page_shift, 0x7fffff00LL);
  const int l = c.lengths[e], n = c.counts != nullptr ? c.counts[e] : N;
  *len = min(max(l, 0), room);
  *count = min(max(n, 0), N);
  return l == *len && n == *count;
}

// Page of the tokens from `position` on, or -1.
__device__ __forceinline__ int page_of(const CacheArgs& c, int e, int position) {
  const int i = position >> c.page_shift;
  if (i >= c.table_pages) return -1;
  const int page = c.table[e * c.table_se + i];
  return page >= 0 && page < c.pages ? page : -1;
}

constexpr int kTreeTokens = 512;  // most tokens of a tree

// Parent of token n of a tree (a row of `parents`): an earlier token, or -1; another value counts as -1.
__device__ __forceinline__ int parent_of(const int* parents, int n, int* status) {
  const int p = parents[n];
  if (p >= -1 && p < n) return p;
  report(status, kBadParent);
  return -1;
}

// softcap * tanh(score / softcap) of a score in units of log2 e, in the same units.  tanh y = 1 - 2 / (exp(2 y) + 1) is off by some 2^-22 whatever y is,
// too much next to a small y; below 1/8 its series takes over, whose first term left out is 2^-29 of it.
__device__ __forceinline__ float capped(float x, float softcap) {
  constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
  const float two = x * (2.0f / softcap), y2 = two * two * (0.25f * kLn2 * kLn2);
  const float large = softcap * kLog2e * (1.0f - __fdividef(2.0f, sm100::ex2(two) + 1.0f));
  const float small = x * fmaf(y2, fmaf(y2, fmaf(y2, -17.0f / 315.0f, 2.0f / 15.0f), -1.0f / 3.0f), 1.0f);
  return y2 < 1.0f / 64.0f ? small : large;
}

struct AppendArgs {
  CacheArgs cache;
  View4 k, v, q, q_out;
  int E, N, H;  // H: query heads, 0 = none
  RotaryArgs rotary;
  const int* parents;  // (E, N) of a tree, whose tokens are rotated at the positions of their depth, or nullptr
  long long parents_se;
};
cudaError_t launch_append(const AppendArgs& a, int dtype, int width, cudaStream_t stream);

// The caches of several layers: one shape, the same strides (in CacheArgs), other pointers.
struct LayerPointers {
  uint8_t *k, *v;
  float *k_scale, *v_scale;
};
constexpr int kMostLayers = 32;  // of a launch

struct AcceptArgs {
  CacheArgs cache;  // (without pointers to a pool)
  LayerPointers layer[kMostLayers];
  int layers, E, N;
  const int* parents;  // (E, N)
  long long parents_se;
  const void *drafted, *answers;  // (E, N) int32 or (ids64) int64
  long long drafted_se, answers_se;
  int ids64;
  int *lengths_out, *path_out;  // (E), (E, N); nullptr: not written
  void* answer_out;             // (E)
};
cudaError_t launch_accept(const AcceptArgs& a, int width, cudaStream_t stream);

struct ForkArgs {
  CacheArgs cache;  // (without pointers to a pool; the table and the lengths are written)
  LayerPointers layer[kMostLayers];
  int layers, E;
  int* uses;            // (pages)
  int *table, *lengths;
  const int *source, *room;  // (E) or nullptr: each row itself, room_all tokens
  int room_all;
  int* workspace;
};
size_t fork_workspace(int E, int table_pages, int pages);
cudaError_t launch_fork(const ForkArgs& a, int width, cudaStream_t stream);
// The copies of the same call in other layers.
cudaError_t launch_fork_copies(const ForkArgs& a, int width, cudaStream_t stream);

struct AttendArgs {
  CacheArgs cache;
  View4 q, out;
  int E, N, H, group;   // group: query heads of a key head
  int causal, window;   // window 0: none
  float scale, softcap;  // softcap 0: none
  int row_blocks;       // blocks of 8 * kernel tiles rows; row = token * group + head of the group
  uint32_t k16[3], v16[3];  // strides of a page, head and token in units of 16 bytes: products with them are one instruction
  float *part_o, *part_ml;  // of the pieces of split heads: two a CTA
  int4* split;              // where heads have been split: an entry a CTA or
  int split_by_head;        // (1) a head and block of rows
  int whole_heads;          // 1: no head is split
  const int* parents;       // (E, N) of a tree, or nullptr
  long long parents_se;
};
// Whether a row of the call's token n has a key at all; the others' results are zero, whatever the sums of their tile have caught.
__device__ __forceinline__ bool sees_keys(const AttendArgs& a, int len, int count, int n) { return n < count && (!a.causal || len - count + n >= 0); }

// Bytes of scratch.
size_t attend_workspace(int E, int N, int H, int kv_heads, int width, int window, long long longest);
// (wait_expiry, a self-test: a wait of the kernel for many rows runs out.)
cudaError_t launch_attend(AttendArgs a, int dtype, int width, void* workspace, long long longest, int* wait_status, bool wait_expiry, cudaStream_t stream);
// The same over a tree (a.parents).
size_t attend_tree_workspace(int E, int N, int H, int kv_heads, int width, int window, long long longest);
// The kernel for few rows over trees (ma_cache_attend_tree.cu): `nt` tiles of 8 rows, `warps` warps a CTA.
cudaError_t launch_few_tree(AttendArgs& a, int dtype, int width, int nt, int warps, long long grid, cudaStream_t stream);
// The pieces of `entries` heads and blocks of tile_rows rows (a.split, a.part_o, a.part_ml; a head's pieces `stride` slots apart) into a.out.
cudaError_t launch_join(const AttendArgs& a, int dtype, int width, int tile_rows, int entries, int stride, cudaStream_t stream);
// The kernel for many rows (ma_cache_prompt.cu).
size_t prompt_workspace(int E, int N, int H, int kv_heads, int width, long long longest);
size_t prompt_tree_workspace(int E, int N, int H, int kv_heads, int width, long long longest);
cudaError_t launch_prompt(AttendArgs a, int dtype, int width, void* workspace, long long longest, int* wait_status, bool wait_expiry, cudaStream_t stream);

}  // namespace ma
