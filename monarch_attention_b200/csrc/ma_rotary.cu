// Rotary positions of queries and keys in one launch.
//
// Bound by memory: each element is read and written once, 4 operations per pair.  A CTA takes 16 tokens of one batch element and a
// number of heads: the sines of its tokens are computed once into shared memory (about 40 instructions a pair) and shared by the heads.
// A thread owns one piece of a row, V pairs (16 bytes of each half of the head, or of neighbouring pairs) or V copied features, and walks
// over the rows in the order in which they lie in memory, four in flight, so that a CTA reads and writes long runs.
// Measured: 20 heads of 128 features, 65536 tokens, bf16 interleaved, 671 MB in 120 us, 5.6 TB/s, 85 % of a copy; with a thread to a head
// 163 us, and 142 with the sines in an order in which lanes met in banks.  What is left is the wait for a row and then for its sines.
#include "ma_rotary.cuh"
#include "ma_sm100.cuh"

namespace ma {

const char* rotary_args(const ma_b200_rotary* r, int width, RotaryArgs* a) {
  a->pairs = 0;
  a->interleaved = 0;
  a->magnitude = a->sign = 1.0f;
  if (r == nullptr) return nullptr;
  if (r->dim <= 0 || r->dim % 2 != 0) return "rotary: dim must be even and positive";
  if (r->dim > width) return "rotary: dim exceeds the head width";
  if (r->dim > 2 * kMaxPairs) return "rotary: dim is above 256";
  if (r->pairs != MA_B200_PAIRS_HALF && r->pairs != MA_B200_PAIRS_INTERLEAVED) return "rotary: unknown layout of pairs";
  if (r->turns == nullptr) return "rotary: turns is NULL";
  a->pairs = r->dim / 2;
  a->interleaved = r->pairs == MA_B200_PAIRS_INTERLEAVED;
  a->magnitude = r->magnitude;
  for (int i = 0; i < a->pairs; ++i) a->turns[i] = r->turns[i];
  return nullptr;
}

namespace {

constexpr int kTokens = 16, kThreads = 256;

struct RotateArgs {
  View4 in[2], out[2];  // queries, keys
  int heads[2];
  int E, N, D, heads_per_cta;
  int tokens_first;  // 1: tokens of a head lie closer together than heads of a token
  const void* positions;
  int positions_i64;
  long long pos_se, pos_sn;
  RotaryArgs rotary;
};

template <typename T, int V>
struct alignas(sizeof(T) * V) Pack {
  T x[V];
};

template <typename T, int V>
__device__ __forceinline__ void widen(const Pack<T, V>& p, float* x) {
  if constexpr (sizeof(T) == 2 && V > 1) {
#pragma unroll
    for (int j = 0; j < V; j += 2) {
      const float2 f = sm100::unpack2<T>(reinterpret_cast<const uint32_t*>(&p)[j / 2]);
      x[j] = f.x;
      x[j + 1] = f.y;
    }
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) x[j] = Cvt<T>::to_f(p.x[j]);
  }
}
template <typename T, int V>
__device__ __forceinline__ void narrow(const float* x, Pack<T, V>& p) {
  if constexpr (sizeof(T) == 2 && V > 1) {
#pragma unroll
    for (int j = 0; j < V; j += 2) reinterpret_cast<uint32_t*>(&p)[j / 2] = sm100::pack2<T>(x[j], x[j + 1]);
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) p.x[j] = Cvt<T>::from_f(x[j]);
  }
}

// One row's piece, V features in x and V in y.  Interleaved: pair j is features 2 j and 2 j + 1 of the two together.  Its sines come two pairs
// at a time, `stride` apart.
template <typename T, int V, bool kInterleaved>
__device__ __forceinline__ void turn(Pack<T, V>& x, Pack<T, V>& y, const float2* sines, int stride) {
  float2 cs[V];
  if constexpr (V == 1) {
    cs[0] = sines[0];
  } else {
#pragma unroll
    for (int j = 0; j < V; j += 2) {
      const float4 two = *reinterpret_cast<const float4*>(sines + (j / 2) * stride);
      cs[j] = make_float2(two.x, two.y);
      cs[j + 1] = make_float2(two.z, two.w);
    }
  }
  float f[2 * V];
  widen<T, V>(x, f);
  widen<T, V>(y, f + V);
#pragma unroll
  for (int j = 0; j < V; ++j) {
    float& a = f[kInterleaved ? 2 * j : j];
    float& b = f[kInterleaved ? 2 * j + 1 : j + V];
    const float u = a, w = b;
    a = u * cs[j].x - w * cs[j].y;
    b = u * cs[j].y + w * cs[j].x;
  }
  narrow<T, V>(f, x);
  narrow<T, V>(f + V, y);
}

template <typename T, int V, bool kInterleaved>
__global__ void __launch_bounds__(kThreads, 4) rotate_kernel(const __grid_constant__ RotateArgs a) {
  using P = Pack<T, V>;
  constexpr int kRows = 4;  // in flight
  __shared__ __align__(16) float2 table[kTokens * kMaxPairs];
  // pieces of a row: rotated ones (half: V features of each half; interleaved: 2 V features), then copied ones of V features
  const int pairs = a.rotary.pairs, turned = pairs / V, pieces = turned + (a.D - 2 * pairs) / V;
  const int tiles = (a.N + kTokens - 1) / kTokens;
  const int e = blockIdx.x / tiles, n0 = (blockIdx.x - e * tiles) * kTokens, tokens = min(kTokens, a.N - n0);
  grid_wait();
  for (int i = threadIdx.x; i < tokens * pairs; i += kThreads) {
    const int t = i / pairs;
    long long p = n0 + t;
    if (a.positions != nullptr) {
      const long long at = e * a.pos_se + p * a.pos_sn;
      p = a.positions_i64 ? reinterpret_cast<const long long*>(a.positions)[at] : reinterpret_cast<const int*>(a.positions)[at];
    }
    // two pairs, 16 bytes, at a time, those of a piece `turned` apart: what neighbouring threads read at once lies next to one another
    const int pair = i - t * pairs, j = pair % V;
    table[t * pairs + (V == 1 ? pair : ((j / 2) * turned + pair / V) * 2 + (j & 1))] = rotary_turn(a.rotary, pair, p);
  }
  __syncthreads();
  const int slots = min(pieces, kThreads), per_pass = kThreads / slots;  // rows of a pass
  const int slot = threadIdx.x / slots, piece = blockIdx.z * kThreads + threadIdx.x - slot * slots;
  if (slot >= per_pass || piece >= pieces) return;
  const bool turns = piece < turned;
  const int fa = !turns ? 2 * pairs + (piece - turned) * V : kInterleaved ? 2 * piece * V : piece * V;
  const int fb = kInterleaved ? fa + V : fa + pairs;
  const int h0 = blockIdx.y * a.heads_per_cta, heads = min(a.heads_per_cta, a.heads[0] + a.heads[1] - h0);
  // rows are numbered with the closer of tokens and heads first
  const int inner = a.tokens_first ? tokens : heads, rows = tokens * heads;
  const int step_out = per_pass / inner, step_in = per_pass - step_out * inner;
  int out = slot / inner, in = slot - out * inner;
  const T *const src_q = reinterpret_cast<const T*>(a.in[0].ptr) + e * a.in[0].se + n0 * a.in[0].sn,
          *const src_k = reinterpret_cast<const T*>(a.in[1].ptr) + e * a.in[1].se + n0 * a.in[1].sn;
  T *const dst_q = reinterpret_cast<T*>(const_cast<void*>(a.out[0].ptr)) + e * a.out[0].se + n0 * a.out[0].sn,
    *const dst_k = reinterpret_cast<T*>(const_cast<void*>(a.out[1].ptr)) + e * a.out[1].se + n0 * a.out[1].sn;
  for (int row = slot; row < rows; row += kRows * per_pass) {
    P x[kRows], y[kRows];
    T* dst[kRows];
    int token[kRows];
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      if (row + i * per_pass >= rows) break;
      const int t = a.tokens_first ? in : out, h = h0 + (a.tokens_first ? out : in);
      const bool key = h >= a.heads[0];
      const T* const src = key ? src_k + (h - a.heads[0]) * a.in[1].sh + t * a.in[1].sn : src_q + h * a.in[0].sh + t * a.in[0].sn;
      dst[i] = key ? dst_k + (h - a.heads[0]) * a.out[1].sh + t * a.out[1].sn : dst_q + h * a.out[0].sh + t * a.out[0].sn;
      token[i] = t;
      x[i] = *reinterpret_cast<const P*>(src + fa);
      if (turns) y[i] = *reinterpret_cast<const P*>(src + fb);
      in += step_in;
      out += step_out;
      if (in >= inner) {
        in -= inner;
        ++out;
      }
    }
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      if (row + i * per_pass >= rows) break;
      if (turns) {
        turn<T, V, kInterleaved>(x[i], y[i], table + token[i] * pairs + piece * (V == 1 ? 1 : 2), 2 * turned);
        *reinterpret_cast<P*>(dst[i] + fb) = y[i];
      }
      *reinterpret_cast<P*>(dst[i] + fa) = x[i];
    }
  }
}

template <typename T, int V>
const void* kernel_of(bool interleaved) {
  return interleaved ? (const void*)rotate_kernel<T, V, true> : (const void*)rotate_kernel<T, V, false>;
}

// Features that a thread takes at once: the most (up to 16 bytes) that divide the pieces of a row, and all row starts.
int vector_of(const RotateArgs& a, size_t size) {
  int v = (int)(16 / size);
  auto fits = [&](int n) {
    if (a.rotary.pairs % n != 0 || (a.D - 2 * a.rotary.pairs) % n != 0) return false;
    for (int i = 0; i < 2; ++i)
      for (const View4* t : {&a.in[i], &a.out[i]})
        if (a.heads[i] > 0 && (reinterpret_cast<uintptr_t>(t->ptr) % (n * size) != 0 || t->se % n != 0 || t->sh % n != 0 || t->sn % n != 0))
          return false;
    return true;
  };
  while (v > 1 && !fits(v)) v /= 2;
  return v;
}

}  // namespace

cudaError_t launch_rotary(const ma_b200_rotation* p, const RotaryArgs& rotary, cudaStream_t stream) {
  RotateArgs a{};
  const ma_b200_tensor* in[2] = {&p->q, &p->k};
  const ma_b200_tensor* out[2] = {&p->q_out, &p->k_out};
  for (int i = 0; i < 2; ++i) {
    a.in[i] = View4{in[i]->ptr, in[i]->stride_e, in[i]->stride_h, in[i]->stride_n};
    a.out[i] = View4{out[i]->ptr, out[i]->stride_e, out[i]->stride_h, out[i]->stride_n};
  }
  a.heads[0] = p->H; a.heads[1] = p->Hk;
  a.E = p->E; a.N = p->N; a.D = p->D;
  const int first = p->H > 0 ? 0 : 1;
  a.tokens_first = a.out[first].sn < a.out[first].sh || a.heads[0] + a.heads[1] == 1;
  a.positions = p->positions;
  a.positions_i64 = p->positions_i64;
  a.pos_se = p->pos_stride_e; a.pos_sn = p->pos_stride_n;
  a.rotary = rotary;
  const int heads = p->H + p->Hk;
  const size_t size = p->dtype == MA_B200_F32 ? 4 : 2;
  const int v = vector_of(a, size);
  const int pieces = rotary.pairs / v + (p->D - 2 * rotary.pairs) / v;
  const long long tiles = (long long)p->E * ((p->N + kTokens - 1) / kTokens);
  // Few tokens: the heads are spread over more CTAs, each of which computes the sines again, until half the SMs have one.  us, 24 heads of 64
  // features, all heads together / until half / until four a SM: 128 tokens 5.4 / 3.6 / 3.6, 1024 5.5 / 4.4 / 8.2, 4096 7.6 / 7.6 / 10.7; 40 heads of 128,
  // 1024 tokens 11.0 / 7.6 / 13.5.
  a.heads_per_cta = heads;
  while (a.heads_per_cta > 2 && tiles * ((heads + a.heads_per_cta - 1) / a.heads_per_cta) < sm_count() / 2) a.heads_per_cta = (a.heads_per_cta + 1) / 2;
  const bool il = rotary.interleaved;
  const void* fn = nullptr;
  if (p->dtype == MA_B200_F32)
    fn = v == 4 ? kernel_of<float, 4>(il) : v == 2 ? kernel_of<float, 2>(il) : kernel_of<float, 1>(il);
  else if (p->dtype == MA_B200_BF16)
    fn = v == 8 ? kernel_of<__nv_bfloat16, 8>(il) : v == 4 ? kernel_of<__nv_bfloat16, 4>(il) : v == 2 ? kernel_of<__nv_bfloat16, 2>(il) : kernel_of<__nv_bfloat16, 1>(il);
  else
    fn = v == 8 ? kernel_of<__half, 8>(il) : v == 4 ? kernel_of<__half, 4>(il) : v == 2 ? kernel_of<__half, 2>(il) : kernel_of<__half, 1>(il);
  void* args[] = {(void*)&a};
  return launch_kernel(fn, dim3((unsigned)tiles, (heads + a.heads_per_cta - 1) / a.heads_per_cta, (pieces + kThreads - 1) / kThreads), dim3(kThreads), args, 0, stream);
}

}  // namespace ma
