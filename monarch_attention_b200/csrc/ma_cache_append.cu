// New keys and values into a paged cache in 8 bits, the keys (and the call's queries) rotated on the way.
//
// A block of 16 tokens of a head shares a scale 2^n, the smallest with which 448 (the largest e4m3 value) holds the block's largest
// magnitude.  A power of two costs a floating-point format nothing but range, and a block that is filled over several calls can
// raise its scale without a second rounding: older codes move by whole exponents, exact but for subnormal ones.  n is held to [-40, 60]: the
// attention's sums are in units of the largest weight times scale, and scales further apart than 2^100 would leave 32 bits.
//
// A lane holds 8 neighbouring features of a row (16 bytes), so that the partner of a rotated feature is in the same lane (interleaved
// pairs) or a shuffle away (half); the sines of a CTA's tokens are computed once into shared memory.
//  * Prompts: a CTA takes a block of 16 tokens and some heads, a lane one of the tokens, whose sines it keeps in registers while it
//    walks over the heads, several rows in flight.  A block's largest magnitude is a reduction over each warp and a maximum in shared
//    memory; rows stay in registers in 16 bits until the scale is known.  Bound by memory.
//  * Single tokens: a row is all there is of a block, so rows of different heads are spread over the warps, and nothing is exchanged
//    between them.  Bound by latency: the row's load does not wait for the length and the page.
// Measured: 8 prompts of up to 1999 tokens, 4 heads of 128 features and 16 query heads, 123 MB in 32 us, 3.8 TB/s; the SMs issue in 52 % of their
// cycles, 16 warps of 128 registers each.  (24 warps of 80 registers, or four heads in flight, take longer.)  One token of 256 sequences of 8 + 32
// heads 4.7 us back to back, of 8 sequences 2.5, which is a launch.
#include "ma_cache_codes.cuh"
#include "ma_sm100.cuh"

namespace ma {
namespace {

constexpr int kWarps = 8, kThreads = 32 * kWarps;
constexpr int F = 8;  // features of a lane

__device__ __forceinline__ uint2 to_codes(const float (&x)[F]) { return make_uint2(four_codes(x[0], x[1], x[2], x[3]), four_codes(x[4], x[5], x[6], x[7])); }
template <typename T>
__device__ __forceinline__ void widen(const uint4& raw, float (&x)[F]) {
  const uint32_t words[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = sm100::unpack2<T>(words[i]);
    x[2 * i] = f.x;
    x[2 * i + 1] = f.y;
  }
}
template <typename T>
__device__ __forceinline__ uint4 narrow(const float (&x)[F]) {
  return make_uint4(sm100::pack2<T>(x[0], x[1]), sm100::pack2<T>(x[2], x[3]), sm100::pack2<T>(x[4], x[5]), sm100::pack2<T>(x[6], x[7]));
}
// (of the numbers: a NaN, also a row of nothing else, asks for no scale)
__device__ __forceinline__ float largest(const float (&x)[F]) {
  float m = 0.0f;
#pragma unroll
  for (int i = 0; i < F; ++i) m = fmaxf(m, fabsf(x[i]));
  return m;
}

// How the lane's features f0 .. f0 + 7 are rotated at one position.
struct Turn {
  float2 cs[F];  // half: of each feature, the sine with its sign; interleaved: of its four pairs
  int partner;   // lane that holds the other half
  bool turned;   // else the features stay what they are: a product with a sine of zero would make a NaN of the partner's infinity
};
// `sines`: those of the position, by pair; not looked at where `real` is false, which turns nothing.
template <int D>
__device__ __forceinline__ Turn turn_of(const RotaryArgs& r, const float2* sines, bool real, int lane, int f0) {
  Turn t;
  t.turned = real && f0 < 2 * r.pairs;
  const bool upper = f0 >= r.pairs;
  constexpr int kLanes = D / F;  // of a row
  t.partner = !t.turned || r.interleaved ? lane : (lane & ~(kLanes - 1)) | ((lane & (kLanes - 1)) + (upper ? -r.pairs / F : r.pairs / F));
#pragma unroll
  for (int i = 0; i < F; ++i) {
    t.cs[i] = make_float2(1.0f, 0.0f);
    if (!t.turned) continue;
    if (!r.interleaved) {
      t.cs[i] = sines[f0 + i - (upper ? r.pairs : 0)];
      if (!upper) t.cs[i].y = -t.cs[i].y;
    } else if (i < F / 2) {
      t.cs[i] = sines[f0 / 2 + i];
    }
  }
  return t;
}
// Features of a row turned in place (the whole warp takes part).
__device__ __forceinline__ void apply(const RotaryArgs& r, const Turn& t, float (&x)[F]) {
  if (r.interleaved) {
    if (!t.turned) return;
#pragma unroll
    for (int i = 0; i < F; i += 2) {
      const float u = x[i], w = x[i + 1];
      x[i] = u * t.cs[i / 2].x - w * t.cs[i / 2].y;
      x[i + 1] = u * t.cs[i / 2].y + w * t.cs[i / 2].x;
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < F; ++i) {
    const float w = __shfl_sync(0xffffffffu, x[i], t.partner);
    if (t.turned) x[i] = x[i] * t.cs[i].x + w * t.cs[i].y;
  }
}

// What a call has to know of sequence e; counts that cannot be are taken as none.
__device__ __forceinline__ void span_of(const CacheArgs& c, int e, int N, bool reports, int* len, int* count) {
  bool fine = sequence_of(c, e, N, len, count);
  if (*count > *len) fine = false;
  if (fine) return;
  if (reports) report(c.status, kBadLength);
  *count = 0;
}

// kTree: the call's tokens are a tree (a.parents): they lie in the cache as they come, and are rotated at the positions of their depth.
template <typename T, int D, bool kTree>
__global__ void __launch_bounds__(kThreads, 2) append_kernel(const __grid_constant__ AppendArgs a) {
  constexpr int kLanes = D / F, kRows = 32 / kLanes;               // rows of a warp at once
  constexpr int kTeam = kScaleBlock / kRows, kTeams = kWarps / kTeam;  // warps that hold the 16 tokens of a head between them
  constexpr int kHeads = 2;                                        // of keys, and of values, that a team has in flight
  __shared__ float2 table[kScaleBlock * D / 2];
  __shared__ unsigned int most[3][kTeams][2][kHeads];
  __shared__ int16_t parents[kTree ? kTreeTokens : 1];
  __shared__ int places[kTree ? kScaleBlock : 1];
  const CacheArgs& c = a.cache;
  const int tid = threadIdx.x, lane = tid & 31, f0 = (lane & (kLanes - 1)) * F;
  const int team = (tid >> 5) / kTeam, slot = ((tid >> 5) % kTeam) * kRows + lane / kLanes;  // the lane's token of the block
  grid_wait();
  const int blocks = (a.N + kScaleBlock - 2) / kScaleBlock + 1;  // that N tokens can touch
  const int e = blockIdx.x / blocks;
  int len, count;
  span_of(c, e, a.N, tid == 0 && blockIdx.y == 0, &len, &count);
  const int start = len - count;
  const int base = (start / kScaleBlock + blockIdx.x % blocks) * kScaleBlock;  // position of the block's first token
  const int pairs = a.rotary.pairs;
  // slots [first, last) of the block take new tokens
  const int first = max(start - base, 0), last = min(max(len - base, 0), kScaleBlock);
  const bool any = first < last;
  const bool fresh = slot >= first && slot < last;  // the lane's token is new
  const int n = base + slot - start;                // the call's number of it
  const int stride = gridDim.y * kTeams * kHeads, g_first = blockIdx.y * kTeams * kHeads;
  uint4 raw[2][kHeads];
  auto load = [&](int h0) {
#pragma unroll
    for (int kind = 0; kind < 2; ++kind)
#pragma unroll
      for (int h = 0; h < kHeads; ++h) {
        const View4& view = kind == 0 ? a.k : a.v;
        raw[kind][h] = make_uint4(0, 0, 0, 0);
        if (fresh && h0 + h < c.heads)
          raw[kind][h] = *reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(view.ptr) + e * view.se + (h0 + h) * view.sh + n * view.sn + f0);
      }
  };
  constexpr int kInFlight = 8;
  const int q_first = (blockIdx.y * kTeams + team) * kInFlight;
  uint4 rows[kInFlight];  // of queries
  auto load_q = [&](int h0) {
    const T* const src = reinterpret_cast<const T*>(a.q.ptr) + e * a.q.se + n * a.q.sn + f0;
#pragma unroll
    for (int i = 0; i < kInFlight; ++i) {
      rows[i] = make_uint4(0, 0, 0, 0);
      if (fresh && h0 + i < a.H) rows[i] = *reinterpret_cast<const uint4*>(src + (h0 + i) * a.q.sh);
    }
  };
  load(g_first + team * kHeads);  // (on their way while the sines are computed)
  load_q(q_first);
  if constexpr (kTree) {
    const int behind = min(base + last - start, count);  // (a token's ancestors are in front of it)
    for (int i = tid; any && i < behind; i += kThreads) parents[i] = (int16_t)parent_of(a.parents + e * a.parents_se, i, c.status);
    __syncthreads();
    if (any && pairs > 0 && tid >= first && tid < last) {
      int depth = -1;
      for (int i = base + tid - start; i >= 0; i = parents[i]) ++depth;
      places[tid] = start + depth;
    }
    __syncthreads();
  }
  if (any)
    for (int i = first * pairs + tid; i < last * pairs; i += kThreads) table[i] = rotary_turn(a.rotary, i % pairs, kTree ? places[i / pairs] : base + i / pairs);
  if (tid < 3 * kTeams * 2 * kHeads) (&most[0][0][0][0])[tid] = 0;
  const int page = any ? page_of(c, e, base) : -1;
  if (any && page < 0 && tid == 0 && blockIdx.y == 0) report(c.status, kBadPage);
  const int in_page = base & ((1 << c.page_shift) - 1);
  __syncthreads();
  const Turn turn = turn_of<D>(a.rotary, table + slot * pairs, fresh, lane, f0);

  // --- keys and values, kHeads at a time
  if (page >= 0) {
    int round = 0;
    for (int g0 = g_first; g0 < c.heads; g0 += stride, round = round == 2 ? 0 : round + 1) {  // (the same for all teams)
      const int h0 = g0 + team * kHeads;
      if (g0 != g_first) load(h0);
      float before[2][kHeads];
#pragma unroll
      for (int kind = 0; kind < 2; ++kind)
#pragma unroll
        for (int h = 0; h < kHeads; ++h) {
          before[kind][h] = 0.0f;
          if (first > 0 && h0 + h < c.heads)  // the block has older tokens, and a scale
            before[kind][h] = (kind == 0 ? c.k_scale + page * c.ks_sp + (h0 + h) * c.ks_sh : c.v_scale + page * c.vs_sp + (h0 + h) * c.vs_sh)[in_page / kScaleBlock];
        }
#pragma unroll
      for (int kind = 0; kind < 2; ++kind)
#pragma unroll
        for (int h = 0; h < kHeads; ++h) {
          float x[F];
          widen<T>(raw[kind][h], x);
          if (kind == 0 && pairs > 0) apply(a.rotary, turn, x);
          const unsigned int bits = __reduce_max_sync(0xffffffffu, __float_as_uint(largest(x)));  // (slots without a new token are zero)
          if (lane == 0) atomicMax(&most[round][team][kind][h], bits);
        }
      // the maxima of the round after next are zero again for all behind this barrier: their last readers were before the one before it
      if (tid < kTeams * 2 * kHeads) (&most[round == 2 ? 0 : round + 1][0][0][0])[tid] = 0;
      __syncthreads();
#pragma unroll
      for (int kind = 0; kind < 2; ++kind)
#pragma unroll
        for (int h = 0; h < kHeads; ++h) {
          const float scale = fmaxf(scale_for(__uint_as_float(most[round][team][kind][h])), before[kind][h]);
          float x[F];
          widen<T>(raw[kind][h], x);
          if (kind == 0 && pairs > 0) apply(a.rotary, turn, x);
          if (h0 + h >= c.heads) continue;
          uint2* const row = reinterpret_cast<uint2*>((kind == 0 ? c.k + page * c.k_sp + (h0 + h) * c.k_sh + (in_page + slot) * c.k_st
                                                                 : c.v + page * c.v_sp + (h0 + h) * c.v_sh + (in_page + slot) * c.v_st) + f0);
          if (fresh) {
            const float inverse = 1.0f / scale;
#pragma unroll
            for (int i = 0; i < F; ++i) x[i] *= inverse;
            *row = to_codes(x);
          } else if (slot < first && scale != before[kind][h]) {
            const uint2 codes = *row;
            const float ratio = before[kind][h] / scale;
            *row = make_uint2(moved(codes.x, ratio), moved(codes.y, ratio));
          }
          if (slot == first && f0 == 0)
            (kind == 0 ? c.k_scale + page * c.ks_sp + (h0 + h) * c.ks_sh : c.v_scale + page * c.vs_sp + (h0 + h) * c.vs_sh)[in_page / kScaleBlock] = scale;
        }
    }
  }

  // --- queries; rows behind the sequence's tokens become zeros
  const bool mine = n >= 0 && n < a.N;
  T* const dst = reinterpret_cast<T*>(const_cast<void*>(a.q_out.ptr)) + e * a.q_out.se + n * a.q_out.sn + f0;
  for (int h0 = q_first; h0 < a.H; h0 += gridDim.y * kTeams * kInFlight) {
    if (h0 != q_first) load_q(h0);
#pragma unroll
    for (int i = 0; i < kInFlight; ++i) {
      float x[F];
      widen<T>(rows[i], x);
      if (pairs > 0) apply(a.rotary, turn, x);
      if (mine && h0 + i < a.H) *reinterpret_cast<uint4*>(dst + (h0 + i) * a.q_out.sh) = narrow<T>(x);
    }
  }
}

// One token of each sequence: a row of 128 features, two to a warp, or of 64, four.  (Six CTAs of an SM, 40 registers: 256 sequences of 8 + 32 heads
// are one round of them, 4.7 us; with 47 registers and five 6.1.)
// kTree: the token is a tree, whose parent can only be none: the position is that of its place, and another parent is reported.
template <typename T, int D, bool kTree>
__global__ void __launch_bounds__(kThreads, 6) append_token_kernel(const __grid_constant__ AppendArgs a) {
  constexpr int kLanes = D / F, kRows = 32 / kLanes;
  __shared__ float2 table[D / 2];
  const CacheArgs& c = a.cache;
  const int lane = threadIdx.x & 31, f0 = (lane & (kLanes - 1)) * F, e = blockIdx.x;
  const int task = (blockIdx.y * kWarps + (threadIdx.x >> 5)) * kRows + lane / kLanes, tasks = 2 * c.heads + a.H;
  const int kind = task < c.heads ? 0 : task < 2 * c.heads ? 1 : 2;  // keys, values, queries
  const int h = task - kind * c.heads;
  grid_wait();
  uint4 raw = make_uint4(0, 0, 0, 0);
  if (task < tasks) {
    const View4& view = kind == 0 ? a.k : kind == 1 ? a.v : a.q;
    raw = *reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(view.ptr) + e * view.se + h * view.sh + f0);
  }
  int len, count;
  span_of(c, e, 1, threadIdx.x == 0 && blockIdx.y == 0, &len, &count);
  if constexpr (kTree) {
    if (count > 0 && threadIdx.x == 0 && blockIdx.y == 0) (void)parent_of(a.parents + e * a.parents_se, 0, c.status);
  }
  const int position = max(len - 1, 0), first = position & (kScaleBlock - 1), pairs = a.rotary.pairs;
  const int page = count > 0 ? page_of(c, e, position) : -1;
  if (threadIdx.x < pairs) table[threadIdx.x] = rotary_turn(a.rotary, threadIdx.x, position);
  if (count > 0 && page < 0 && threadIdx.x == 0 && blockIdx.y == 0) report(c.status, kBadPage);
  const bool cached = task < 2 * c.heads && page >= 0;
  const int in_page = position & ((1 << c.page_shift) - 1);
  float* at = nullptr;
  float before = 0.0f;
  if (cached) {
    at = (kind == 0 ? c.k_scale + page * c.ks_sp + h * c.ks_sh : c.v_scale + page * c.vs_sp + h * c.vs_sh) + in_page / kScaleBlock;
    if (first > 0) before = *at;
  }
  __syncthreads();  // (also: the row's lanes have read the older scale)
  float x[F];
  widen<T>(raw, x);
  if (pairs > 0) apply(a.rotary, turn_of<D>(a.rotary, table, kind != 1, lane, f0), x);  // (values, next to keys in a warp, are not turned)
  float amax = largest(x);
#pragma unroll
  for (int m = kLanes / 2; m > 0; m >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, m));
  if (task < tasks && kind == 2) {
    T* const dst = reinterpret_cast<T*>(const_cast<void*>(a.q_out.ptr)) + e * a.q_out.se + h * a.q_out.sh + f0;
    *reinterpret_cast<uint4*>(dst) = count > 0 ? narrow<T>(x) : make_uint4(0, 0, 0, 0);
  }
  if (!cached) return;
  const float scale = fmaxf(scale_for(amax), before);
  const long long st = kind == 0 ? c.k_st : c.v_st;
  uint8_t* const block = (kind == 0 ? c.k + page * c.k_sp + h * c.k_sh : c.v + page * c.v_sp + h * c.v_sh) + (in_page - first) * st + f0;
  if (f0 == 0) *at = scale;
  const float inverse = 1.0f / scale;
#pragma unroll
  for (int i = 0; i < F; ++i) x[i] *= inverse;
  *reinterpret_cast<uint2*>(block + first * st) = to_codes(x);
  if (first > 0 && scale != before) {
    const float ratio = before / scale;
    for (int t = 0; t < first; ++t) {
      uint2* const row = reinterpret_cast<uint2*>(block + t * st);
      *row = make_uint2(moved(row->x, ratio), moved(row->y, ratio));
    }
  }
}

}  // namespace

cudaError_t launch_append(const AppendArgs& a, int dtype, int width, cudaStream_t stream) {
  void* args[] = {(void*)&a};
  const bool bf = dtype == MA_B200_BF16;
  // us, the kernel for single tokens / the other: 8 sequences of 4 heads 3.5 / 9.9, 256 of 8 heads 5.4 / 20.1
  if (a.N == 1) {
    const int rows = kWarps * 32 * F / width;  // of a CTA
    const void* fn = bf ? (width == 128 ? (const void*)append_token_kernel<__nv_bfloat16, 128, false> : (const void*)append_token_kernel<__nv_bfloat16, 64, false>)
                        : (width == 128 ? (const void*)append_token_kernel<__half, 128, false> : (const void*)append_token_kernel<__half, 64, false>);
    if (a.parents != nullptr)
      fn = bf ? (width == 128 ? (const void*)append_token_kernel<__nv_bfloat16, 128, true> : (const void*)append_token_kernel<__nv_bfloat16, 64, true>)
              : (width == 128 ? (const void*)append_token_kernel<__half, 128, true> : (const void*)append_token_kernel<__half, 64, true>);
    return launch_kernel(fn, dim3(a.E, (2 * a.cache.heads + a.H + rows - 1) / rows), dim3(kThreads), args, 0, stream);
  }
  const void* fn = bf ? (width == 128 ? (const void*)append_kernel<__nv_bfloat16, 128, false> : (const void*)append_kernel<__nv_bfloat16, 64, false>)
                      : (width == 128 ? (const void*)append_kernel<__half, 128, false> : (const void*)append_kernel<__half, 64, false>);
  if (a.parents != nullptr)  // (also where nothing is rotated: parents that cannot be are reported)
    fn = bf ? (width == 128 ? (const void*)append_kernel<__nv_bfloat16, 128, true> : (const void*)append_kernel<__nv_bfloat16, 64, true>)
            : (width == 128 ? (const void*)append_kernel<__half, 128, true> : (const void*)append_kernel<__half, 64, true>);
  const long long blocks = (long long)a.E * ((a.N + kScaleBlock - 2) / kScaleBlock + 1);
  // Few blocks: their heads are spread over more CTAs, each of which computes the sines again; four for each SM where a block's sines are few, else one.
  // us, all heads together / four / one: 17 tokens of 8 sequences 11.2 / 7.8 / 7.7; 5 tokens of 64 sequences and 12 heads of 64 features 10.2 / 8.3 / 9.5; a
  // prompt of 1999 and 4 heads 11.0 / 9.9 / 10.0; two of them 17.6 / 17.6 / 14.1, four 27 / 32 / 27.
  const int per = width == 128 ? 2 : 4;
  const int groups = (a.cache.heads + per - 1) / per;
  const long long sms = sm_count(), ctas = (a.N < kScaleBlock ? 4LL : 1LL) * sms;
  long long wanted = (ctas + blocks - 1) / blocks;
  // Trees come by the batch.  With more blocks than SMs and many heads it counts how many of the blocks have a token (not every sequence's tokens touch all of its blocks): up to one an SM,
  // two groups of heads keep both of its places busy; up to 1.35, groups smaller than the most there can be even the SMs with two blocks out with those of one; more than both places and up to 2.8, two
  // groups, so that the second round is not half empty.  (128 features, where a CTA is long: as soon as there are more blocks than places, with or without a token.)
  // us, one group / so many, tokens x sequences, 8 + 32 heads of 128 features: 61 x 30 22.1 / 16.1 (two), 61 x 38 24.1 / 22.0 (three), 25 x 74 22.3 / 21.1 (three), 61 x 64 40.7 / 35.9 (two), 61 x 80
  // 46.8 / 41.0, 25 x 147 43.5 / 38.4; 12 + 12 of 64 features: 25 x 64 13.2 / 11.4 (two), 25 x 123 21.7 / 19.6.  Between and behind, where one group is taken, one / two: 61 x 48 25.2 / 27.6, 61 x 59
  // 26.1 / 29.2, 61 x 100 49.3 / 51.2; 64 features: 25 x 93 13.7 / 15.4, 25 x 117 16.6 / 18.5, 25 x 197 25.9 / 29.3; 24 + 8 heads, 40 x 56 12.7 / 14.8.
  if (a.parents != nullptr && blocks > sms && 2 * a.cache.heads + a.H >= 32) {
    const long long full = (long long)a.E * (a.N + kScaleBlock - 1) / kScaleBlock;  // blocks with a token, as a mean over where sequences end
    if (full <= sms) wanted = 2;
    else if (20 * full <= 27 * sms) wanted = groups <= 2 ? 1 : groups == 3 ? 2 : 3;
    else wanted = 20 * (width == 128 ? blocks : full) > 41 * sms && 5 * full <= 14 * sms ? 2 : 1;
  }
  return launch_kernel(fn, dim3((unsigned)blocks, (unsigned)(wanted < groups ? wanted : groups)), dim3(kThreads), args, 0, stream);
}

}  // namespace ma
