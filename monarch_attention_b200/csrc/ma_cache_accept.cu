// Which drafted tokens of a tree stand, and the caches of all layers closed up over them.
//
// Token 0 of a sequence stands; another one does if its parent does and it is what the model answered the parent with (the first of several).  The
// line of tokens that stand, path[0] < path[1] < .., is moved to the slots start, start + 1, .. of the call.  A slot is never behind its token's
// (path[i] >= i), so that blocks of 16 slots are filled from the front on: a block's tokens come from itself or from behind it, and are all in
// registers before the first is written.  A block that tokens move into has the scale that the append would have given it, the smallest
// that holds them, or its own where older tokens stay in it and theirs is larger.
//
// A CTA finds the path of its sequence (two reads that depend on each other, a minimum in shared memory for each token's first fitting child, and a
// walk along it), then its warps take a head's keys or values of a layer each.  All layers are in one launch: the path is the same for them.
// Bound by latency: a chain of six reads (length, parent, answer, page, row, and the page's other rows) for some hundred bytes of a head.  Measured in a
// graph: one sequence of 7 tokens, 12 layers of 12 heads of 64 features 4.4 us, 64 of up to 61 tokens, 16 layers of 8 heads of 128 features 11.1 (14.6 where passes without a token look for their
// maximum too); a call from the host is 10.5 and 12, by its checks of all layers.
#include "ma_cache_codes.cuh"

namespace ma {
namespace {

constexpr int kWarps = 8, kThreads = 32 * kWarps;

template <typename Id>
__device__ __forceinline__ bool fits(const AcceptArgs& a, int e, int n, int parent) {
  return reinterpret_cast<const Id*>(a.drafted)[e * a.drafted_se + n] == reinterpret_cast<const Id*>(a.answers)[e * a.answers_se + parent];
}

// Largest magnitude of 16 codes; a NaN has none.
__device__ __forceinline__ float largest_code(const uint4& codes) {
  const uint32_t words[4] = {codes.x, codes.y, codes.z, codes.w};
  uint32_t most = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t m = words[i] & 0x7f7f7f7fu;
    most = __vmaxu4(most, m & ~__vcmpeq4(m, 0x7f7f7f7fu));
  }
  most = __vmaxu4(most, most >> 16);
  most = __vmaxu4(most, most >> 8) & 0xff;
  return __half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)most, __NV_E4M3)));
}
__device__ __forceinline__ uint4 moved16(const uint4& c, float ratio) { return make_uint4(moved(c.x, ratio), moved(c.y, ratio), moved(c.z, ratio), moved(c.w, ratio)); }

template <int D>
__global__ void __launch_bounds__(kThreads) accept_kernel(const __grid_constant__ AcceptArgs a) {
  constexpr int kLanes = D / 16, kRows = 32 / kLanes, kPasses = kScaleBlock / kRows;  // of a row; rows of a warp at once; passes of a block
  __shared__ int16_t path[kTreeTokens];
  __shared__ unsigned int first_child[kTreeTokens];
  __shared__ int2 from[kTreeTokens];  // page (-1: none) and row in it of the tokens that stand
  __shared__ int taken_s, in_place_s;
  const CacheArgs& c = a.cache;
  const int tid = threadIdx.x, w = tid >> 5, lane = tid & 31, e = blockIdx.x, N = a.N;
  grid_wait();
  int len, count;
  bool fine = sequence_of(c, e, N, &len, &count);
  if (count > len) fine = false;
  if (!fine) {
    if (tid == 0 && blockIdx.y == 0) report(c.status, kBadLength);
    count = 0;
  }
  const int start = len - count;
  for (int n = tid; n < count; n += kThreads) first_child[n] = 0xffffu;
  __syncthreads();
  for (int n = tid; n < count; n += kThreads) {
    const int parent = parent_of(a.parents + e * a.parents_se, n, c.status);
    if (parent >= 0 && (a.ids64 ? fits<long long>(a, e, n, parent) : fits<int>(a, e, n, parent))) atomicMin(&first_child[parent], (unsigned)n);
  }
  __syncthreads();
  if (tid == 0) {
    int taken = 0, in_place = 0;
    for (unsigned n = count > 0 ? 0u : 0xffffu; n != 0xffffu; n = first_child[n]) {
      path[taken] = (int16_t)n;
      in_place += (int)n == taken;
      ++taken;
    }
    taken_s = taken;
    in_place_s = in_place;
  }
  __syncthreads();
  const int taken = taken_s, in_place = in_place_s;
  if (blockIdx.y == 0 && a.lengths_out != nullptr) {
    for (int n = tid; n < N; n += kThreads) a.path_out[(long long)e * N + n] = n < taken ? path[n] : -1;
    if (tid == 0) {
      a.lengths_out[e] = start + taken;
      const long long at = e * a.answers_se + (taken > 0 ? path[taken - 1] : 0);
      if (a.ids64) reinterpret_cast<long long*>(a.answer_out)[e] = taken > 0 ? reinterpret_cast<const long long*>(a.answers)[at] : -1;
      else reinterpret_cast<int*>(a.answer_out)[e] = taken > 0 ? reinterpret_cast<const int*>(a.answers)[at] : -1;
    }
  }
  if (in_place == taken) return;
  const int page_mask = (1 << c.page_shift) - 1;
  for (int i = in_place + tid; i < taken; i += kThreads) {
    const int position = start + path[i];
    from[i] = make_int2(page_of(c, e, position), position & page_mask);
    if (from[i].x < 0) report(c.status, kBadPage);
  }
  __syncthreads();

  const int lane_row = lane / kLanes, piece = lane % kLanes, tasks = a.layers * 2 * c.heads;
  for (int task = blockIdx.y * kWarps + w; task < tasks; task += gridDim.y * kWarps) {
    const int head = task % c.heads, kind = task / c.heads & 1, layer = task / c.heads >> 1;
    const LayerPointers& l = a.layer[layer];
    uint8_t* const codes = (kind ? l.v + head * c.v_sh : l.k + head * c.k_sh) + piece * 16;
    float* const scales = kind ? l.v_scale + head * c.vs_sh : l.k_scale + head * c.ks_sh;
    const long long sp = kind ? c.v_sp : c.k_sp, st = kind ? c.v_st : c.k_st, ssp = kind ? c.vs_sp : c.ks_sp;
    for (int block = (start + in_place) / kScaleBlock; block * kScaleBlock < start + taken; ++block) {
      const int i0 = block * kScaleBlock - start;  // the path's number of the block's first slot
      const int page = page_of(c, e, block * kScaleBlock), row0 = (block * kScaleBlock) & page_mask;
      if (page < 0) {
        if (lane == 0) report(c.status, kBadPage);
        continue;
      }
      uint8_t* const rows = codes + page * sp + row0 * st;
      float* const scale_at = scales + page * ssp + row0 / kScaleBlock;
      uint4 x[kPasses];
      float xs[kPasses], amax = 0.0f;  // xs: the tokens' scales, -1 where there is none to move; NaN makes NaN of a token
#pragma unroll
      for (int p = 0; p < kPasses; ++p) {
        const int i = i0 + p * kRows + lane_row;
        const int2 src = i >= in_place && i < taken ? from[i] : make_int2(-1, 0);
        x[p] = make_uint4(0, 0, 0, 0);
        xs[p] = -1.0f;
        if (src.x >= 0) {
          x[p] = *reinterpret_cast<const uint4*>(codes + src.x * sp + src.y * st);
          xs[p] = scales[src.x * ssp + src.y / kScaleBlock];
        }
      }
      const bool older = i0 < in_place;  // tokens stay in the block
      const float before = older ? *scale_at : 0.0f;
#pragma unroll
      for (int p = 0; p < kPasses; ++p) amax = fmaxf(amax, xs[p] < 0.0f ? 0.0f : largest_code(x[p]) * xs[p]);  // (a NaN asks for no scale)
      const float scale = fmaxf(scale_for(__uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(amax)))), before);
      __syncwarp();  // (all of the block's tokens, and the scales that they come with, have been read)
#pragma unroll
      for (int p = 0; p < kPasses; ++p) {
        const int slot = p * kRows + lane_row;
        uint4* const at = reinterpret_cast<uint4*>(rows + slot * st);
        if (!(xs[p] < 0.0f)) *at = moved16(x[p], xs[p] / scale);
        else if (i0 + slot < in_place && scale != before) *at = moved16(*at, before / scale);
      }
      if (lane == 0) *scale_at = scale;
      __syncwarp();
    }
  }
}

}  // namespace

cudaError_t launch_accept(const AcceptArgs& a, int width, cudaStream_t stream) {
  void* args[] = {(void*)&a};
  // (every CTA finds the path anew: no more of them than run at a time)
  const int tasks = (2 * a.layers * a.cache.heads + kWarps - 1) / kWarps, most = (8 * sm_count() + a.E - 1) / a.E;
  return launch_kernel(width == 128 ? (const void*)accept_kernel<128> : (const void*)accept_kernel<64>, dim3(a.E, tasks < most ? tasks : most), dim3(kThreads), args, 0, stream);
}

}  // namespace ma
