// New keys and values into a paged cache in 8 bits, the keys (and the call's queries) rotated on the way.
//
// A block of 16 tokens of a head shares a scale 2^n, the smallest with which 448 (the largest e4m3 value) holds the block's largest
// magnitude.  A power of two costs a floating-point format nothing but range, and a block that is filled over several calls can
// raise its scale without a second rounding: older codes move by whole exponents, exact but for subnormal ones.  n is held to [-40, 60]: the
// attention's sums are in units of the largest weight times scale, and scales further apart than 2^100 would leave 32 bits.
//
// A warp takes one head of one block, for the keys, the values or the queries: lane l holds features [l D/32, (l+1) D/32) of the 16 tokens in
// registers, so that a row is one coalesced access, the partner of a rotated feature is in the same lane (interleaved pairs) or a
// shuffle away (half), and the block's magnitude is a reduction over the warp.  The sines of the block's positions are computed once for
// the CTA's warps.  Bound by memory for prompts (16-bit rows in, 8-bit rows out), by latency for single tokens.
#include <cuda_fp8.h>

#include "ma_cache.cuh"

namespace ma {
namespace {

constexpr int kWarps = 8;

template <int F>
struct Word;
template <>
struct Word<4> {
  using Half = uint2;
  using Code = uint32_t;
};
template <>
struct Word<2> {
  using Half = uint32_t;
  using Code = uint16_t;
};

// The smallest n in [-40, 60] with amax <= 448 * 2^n, as 2^n: 448 = 1.75 * 2^8, so a mantissa above 1.75 takes one more.
__device__ __forceinline__ float scale_for(float amax) {
  const int n = (int)((__float_as_uint(amax) + 0x1fffffu) >> 23) - 127 - 8;
  return __uint_as_float((uint32_t)(min(max(n, -40), 60) + 127) << 23);
}

template <int F>
__device__ __forceinline__ typename Word<F>::Code to_codes(const float (&x)[F]) {
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < F; i += 2) w |= (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(x[i], x[i + 1]), __NV_SATFINITE, __NV_E4M3) << (8 * i);
  return (typename Word<F>::Code)w;
}
template <int F>
__device__ __forceinline__ void from_codes(typename Word<F>::Code w, float (&x)[F]) {
#pragma unroll
  for (int i = 0; i < F; i += 2) {
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)((uint32_t)w >> (8 * i)), __NV_E4M3);
    const float2 f = __half22float2(__half2(h));
    x[i] = f.x;
    x[i + 1] = f.y;
  }
}

template <typename T, int D>
__global__ void __launch_bounds__(kWarps * 32) append_kernel(const __grid_constant__ AppendArgs a) {
  constexpr int F = D / 32;
  using Half = typename Word<F>::Half;
  using Code = typename Word<F>::Code;
  __shared__ float2 table[kScaleBlock * D / 2];
  const CacheArgs& c = a.cache;
  grid_wait();
  const int blocks = (a.N + kScaleBlock - 2) / kScaleBlock + 1;  // that N tokens can touch
  const int e = blockIdx.x / blocks;
  int len, count;
  bool fine = sequence_of(c, e, a.N, &len, &count);
  if (count > len) fine = false;
  if (!fine) {  // nothing is appended
    if (threadIdx.x == 0 && blockIdx.y == 0) report(c.status, kBadLength);
    count = 0;
  }
  const int start = len - count;
  const int base = (start / kScaleBlock + blockIdx.x % blocks) * kScaleBlock;  // position of the block's first token
  const int pairs = a.rotary.pairs;
  // slots [first, last) of the block take new tokens
  const int first = max(start - base, 0), last = min(max(len - base, 0), kScaleBlock);
  if (first < last)
    for (int i = threadIdx.x; i < (last - first) * pairs; i += kWarps * 32) {
      const int t = first + i / pairs, j = i % pairs;
      table[t * pairs + j] = rotary_turn(a.rotary, j, base + t);
    }
  __syncthreads();
  const int page = first < last ? page_of(c, e, base) : -1;
  if (first < last && page < 0 && threadIdx.x == 0 && blockIdx.y == 0) report(c.status, kBadPage);
  const int in_page = base & ((1 << c.page_shift) - 1);
  const int lane = threadIdx.x & 31, f0 = lane * F;
  const int tasks = 2 * c.heads + a.H;
  for (int task = blockIdx.y * kWarps + (threadIdx.x >> 5); task < tasks; task += gridDim.y * kWarps) {
    const int kind = task < c.heads ? 0 : task < 2 * c.heads ? 1 : 2;  // keys, values, queries
    const int h = task - kind * c.heads;
    const View4& view = kind == 0 ? a.k : kind == 1 ? a.v : a.q;
    const T* src = reinterpret_cast<const T*>(view.ptr) + e * view.se + h * view.sh + f0;
    Half raw[kScaleBlock];
#pragma unroll
    for (int t = 0; t < kScaleBlock; ++t)
      raw[t] = t >= first && t < last ? *reinterpret_cast<const Half*>(src + (base + t - start) * view.sn) : Half{};
    float x[kScaleBlock][F];
#pragma unroll
    for (int t = 0; t < kScaleBlock; ++t) {
      const T* r = reinterpret_cast<const T*>(&raw[t]);
#pragma unroll
      for (int i = 0; i < F; ++i) x[t][i] = Cvt<T>::to_f(r[i]);
    }
    if (kind != 1 && pairs > 0) {
      const bool turned = f0 < 2 * pairs;
      if (a.rotary.interleaved) {
#pragma unroll
        for (int t = 0; t < kScaleBlock; ++t) {
          if (t < first || t >= last || !turned) continue;
#pragma unroll
          for (int i = 0; i < F; i += 2) {
            const float2 cs = table[t * pairs + (f0 + i) / 2];
            const float u = x[t][i], w = x[t][i + 1];
            x[t][i] = u * cs.x - w * cs.y;
            x[t][i + 1] = u * cs.y + w * cs.x;
          }
        }
      } else {
        const bool upper = f0 >= pairs;
        const int other = (lane + (upper ? -pairs / F : pairs / F)) & 31, j = upper ? f0 - pairs : f0;
#pragma unroll
        for (int t = 0; t < kScaleBlock; ++t) {
          if (t < first || t >= last) continue;  // (the same for the whole warp)
#pragma unroll
          for (int i = 0; i < F; ++i) {
            const float w = __shfl_sync(0xffffffffu, x[t][i], other);
            if (turned) {
              const float2 cs = table[t * pairs + j + i];
              x[t][i] = upper ? w * cs.y + x[t][i] * cs.x : x[t][i] * cs.x - w * cs.y;
            }
          }
        }
      }
    }
    if (kind == 2) {
      T* dst = reinterpret_cast<T*>(const_cast<void*>(a.q_out.ptr)) + e * a.q_out.se + h * a.q_out.sh + f0;
#pragma unroll
      for (int t = 0; t < kScaleBlock; ++t) {
        const int n = base + t - start;  // rows behind the sequence's tokens become zeros
        if (n < 0 || n >= a.N) continue;
        Half out;
        T* r = reinterpret_cast<T*>(&out);
#pragma unroll
        for (int i = 0; i < F; ++i) r[i] = Cvt<T>::from_f(t < last ? x[t][i] : 0.0f);
        *reinterpret_cast<Half*>(dst + n * a.q_out.sn) = out;
      }
      continue;
    }
    if (page < 0) continue;
    float amax = 0.0f;
#pragma unroll
    for (int t = 0; t < kScaleBlock; ++t)
#pragma unroll
      for (int i = 0; i < F; ++i) amax = fmaxf(amax, fabsf(x[t][i]));  // (slots without a new token are zero)
#pragma unroll
    for (int m = 16; m > 0; m >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, m));
    float* at = kind == 0 ? c.k_scale + page * c.ks_sp + h * c.ks_sh : c.v_scale + page * c.vs_sp + h * c.vs_sh;
    at += in_page / kScaleBlock;
    float scale = scale_for(amax), before = scale;
    if (first > 0) {  // the block has older tokens
      before = *at;
      scale = fmaxf(scale, before);
    }
    __syncwarp();
    if (lane == 0) *at = scale;
    uint8_t* rows = kind == 0 ? c.k + page * c.k_sp + h * c.k_sh : c.v + page * c.v_sp + h * c.v_sh;
    const long long pitch = kind == 0 ? c.k_st : c.v_st;
    rows += in_page * pitch + f0;
    if (scale != before) {
      const float ratio = before / scale;
      for (int t = 0; t < first; ++t) {
        float y[F];
        from_codes<F>(*reinterpret_cast<const Code*>(rows + t * pitch), y);
#pragma unroll
        for (int i = 0; i < F; ++i) y[i] *= ratio;
        *reinterpret_cast<Code*>(rows + t * pitch) = to_codes<F>(y);
      }
    }
    const float inverse = 1.0f / scale;
#pragma unroll
    for (int t = 0; t < kScaleBlock; ++t) {
      if (t < first || t >= last) continue;
#pragma unroll
      for (int i = 0; i < F; ++i) x[t][i] *= inverse;
      *reinterpret_cast<Code*>(rows + t * pitch) = to_codes<F>(x[t]);
    }
  }
}

}  // namespace

cudaError_t launch_append(const AppendArgs& a, int dtype, int width, cudaStream_t stream) {
  const long long blocks = (a.N + kScaleBlock - 2) / kScaleBlock + 1;
  const int rounds = (2 * a.cache.heads + a.H + kWarps - 1) / kWarps;
  // few blocks: a round of tasks for each CTA, so that no warp takes a second
  const long long wanted = 4LL * sm_count() / (a.E * blocks) + 1;
  const unsigned y = (unsigned)(wanted < rounds ? wanted : rounds);
  const void* fn = dtype == MA_B200_BF16 ? (width == 128 ? (const void*)append_kernel<__nv_bfloat16, 128> : (const void*)append_kernel<__nv_bfloat16, 64>)
                                         : (width == 128 ? (const void*)append_kernel<__half, 128> : (const void*)append_kernel<__half, 64>);
  void* args[] = {(void*)&a};
  return launch_kernel(fn, dim3((unsigned)(a.E * blocks), y), dim3(kWarps * 32), args, 0, stream);
}

}  // namespace ma
