// Rotary positions of queries and keys in one launch.
//
// Bound by memory: each element is read and written once, 4 operations per pair.  A CTA takes 16 tokens of one batch element and a
// number of heads: the sines and cosines of its tokens are computed once into shared memory (about 40 instructions a pair) and shared by
// the heads.  A thread takes V pairs at a time (16 bytes of each half of the head, or of neighbouring pairs); tokens go before heads
// where they lie next to each other in memory, so that a warp's accesses are whole lines either way.
#include "ma_rotary.cuh"

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

template <typename T, int V, bool kInterleaved>
__global__ void __launch_bounds__(kThreads) rotate_kernel(const __grid_constant__ RotateArgs a) {
  __shared__ float2 table[kTokens * kMaxPairs];
  using P = Pack<T, V>;
  grid_wait();
  const int tiles = (a.N + kTokens - 1) / kTokens;
  const int e = blockIdx.x / tiles, n0 = (blockIdx.x % tiles) * kTokens;
  const int tokens = min(kTokens, a.N - n0), pairs = a.rotary.pairs;
  for (int i = threadIdx.x; i < tokens * pairs; i += kThreads) {
    const int t = i / pairs;
    long long p = n0 + t;
    if (a.positions != nullptr) {
      const long long at = e * a.pos_se + p * a.pos_sn;
      p = a.positions_i64 ? reinterpret_cast<const long long*>(a.positions)[at] : reinterpret_cast<const int*>(a.positions)[at];
    }
    table[i] = rotary_turn(a.rotary, i - t * pairs, p);
  }
  __syncthreads();
  // pieces of a row: rotated ones of V pairs (half: V features of each half; interleaved: 2 of V features), then copied ones of V features
  const int turned = pairs / V, copied = (a.D - 2 * pairs) / V, pieces = turned + copied;
  const int h0 = blockIdx.y * a.heads_per_cta, heads = min(a.heads_per_cta, a.heads[0] + a.heads[1] - h0);
  const int total = tokens * heads * pieces;
  for (int i = threadIdx.x; i < total; i += kThreads) {
    const int row = i / pieces, piece = i - row * pieces;
    const int t = a.tokens_first ? row % tokens : row / heads;
    int h = h0 + (a.tokens_first ? row / tokens : row - t * heads);
    const int which = h >= a.heads[0];
    h -= which ? a.heads[0] : 0;
    const View4 &vi = which ? a.in[1] : a.in[0], &vo = which ? a.out[1] : a.out[0];
    const T* src = reinterpret_cast<const T*>(vi.ptr) + e * vi.se + h * vi.sh + (n0 + t) * vi.sn;
    T* dst = reinterpret_cast<T*>(const_cast<void*>(vo.ptr)) + e * vo.se + h * vo.sh + (n0 + t) * vo.sn;
    if (piece >= turned) {
      const int f = 2 * pairs + (piece - turned) * V;
      *reinterpret_cast<P*>(dst + f) = *reinterpret_cast<const P*>(src + f);
      continue;
    }
    const float2* cs = table + t * pairs + piece * V;
    const int fa = kInterleaved ? 2 * piece * V : piece * V, fb = kInterleaved ? fa + V : fa + pairs;
    P x = *reinterpret_cast<const P*>(src + fa), y = *reinterpret_cast<const P*>(src + fb);
    if constexpr (kInterleaved && V == 1) {
      const float u = Cvt<T>::to_f(x.x[0]), w = Cvt<T>::to_f(y.x[0]);
      x.x[0] = Cvt<T>::from_f(u * cs[0].x - w * cs[0].y);
      y.x[0] = Cvt<T>::from_f(u * cs[0].y + w * cs[0].x);
    } else if constexpr (kInterleaved) {
#pragma unroll
      for (int j = 0; j < V; j += 2) {
        float u = Cvt<T>::to_f(x.x[j]), w = Cvt<T>::to_f(x.x[j + 1]);
        x.x[j] = Cvt<T>::from_f(u * cs[j / 2].x - w * cs[j / 2].y);
        x.x[j + 1] = Cvt<T>::from_f(u * cs[j / 2].y + w * cs[j / 2].x);
        u = Cvt<T>::to_f(y.x[j]), w = Cvt<T>::to_f(y.x[j + 1]);
        y.x[j] = Cvt<T>::from_f(u * cs[(V + j) / 2].x - w * cs[(V + j) / 2].y);
        y.x[j + 1] = Cvt<T>::from_f(u * cs[(V + j) / 2].y + w * cs[(V + j) / 2].x);
      }
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float u = Cvt<T>::to_f(x.x[j]), w = Cvt<T>::to_f(y.x[j]);
        x.x[j] = Cvt<T>::from_f(u * cs[j].x - w * cs[j].y);
        y.x[j] = Cvt<T>::from_f(u * cs[j].y + w * cs[j].x);
      }
    }
    *reinterpret_cast<P*>(dst + fa) = x;
    *reinterpret_cast<P*>(dst + fb) = y;
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
  a.tokens_first = a.out[first].sn < a.out[first].sh || p->H + p->Hk == 1;
  a.positions = p->positions;
  a.positions_i64 = p->positions_i64;
  a.pos_se = p->pos_stride_e; a.pos_sn = p->pos_stride_n;
  a.rotary = rotary;
  const long long tiles = (long long)p->E * ((p->N + kTokens - 1) / kTokens);
  const int heads = p->H + p->Hk;
  // few tokens: the heads are spread over more CTAs, each of which computes the sines again
  a.heads_per_cta = heads;
  while (a.heads_per_cta > 2 && tiles * ((heads + a.heads_per_cta - 1) / a.heads_per_cta) < 2 * sm_count()) a.heads_per_cta = (a.heads_per_cta + 1) / 2;
  const size_t size = p->dtype == MA_B200_F32 ? 4 : 2;
  const int v = vector_of(a, size);
  const bool il = rotary.interleaved;
  const void* fn = nullptr;
  if (p->dtype == MA_B200_F32)
    fn = v == 4 ? kernel_of<float, 4>(il) : v == 2 ? kernel_of<float, 2>(il) : kernel_of<float, 1>(il);
  else if (p->dtype == MA_B200_BF16)
    fn = v == 8 ? kernel_of<__nv_bfloat16, 8>(il) : v == 4 ? kernel_of<__nv_bfloat16, 4>(il) : v == 2 ? kernel_of<__nv_bfloat16, 2>(il) : kernel_of<__nv_bfloat16, 1>(il);
  else
    fn = v == 8 ? kernel_of<__half, 8>(il) : v == 4 ? kernel_of<__half, 4>(il) : v == 2 ? kernel_of<__half, 2>(il) : kernel_of<__half, 1>(il);
  void* args[] = {(void*)&a};
  return launch_kernel(fn, dim3((unsigned)tiles, (heads + a.heads_per_cta - 1) / a.heads_per_cta), dim3(kThreads), args, 0, stream);
}

}  // namespace ma
