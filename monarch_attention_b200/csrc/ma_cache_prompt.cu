// Softmax attention of many query rows (a prompt, or a piece of one) over a paged cache in 8 bits, on the tcgen05 tensor cores.
//
// Bound by the tensor cores and by the exponentials (as many cycles at 128 features: 2 x 256 x 128 x 128 x 2 operations of a step are 2048 cycles,
// its 256 x 128 exponentials 2048 of the special function units).  A CTA takes 256 rows (tokens times heads of a group) of a key head and
// walks over its keys, 128 at a step:
//  * Four warps bring keys and values: bytes from global memory into registers, half a step ahead, and from there, widened to f16 (exact),
//    into swizzled tiles in shared memory.  Two tiles of rows share them, so that the conversion and the shared memory's traffic, which a
//    single tile would be bound by, count half.
//  * Two warpgroups have a row a thread: the row's 128 scores go from tensor memory to registers in one go, and the maximum, the weights and
//    their sum need no other thread.  Scales of blocks are applied as in the kernel for few rows (ma_cache_attend.cu): the keys' to the
//    scores, the values' to the weights, with a reference that is raised (and O multiplied) only when a weight would pass 2^15.
//  * One warp issues the products: O += P V, the weights P read from tensor memory, where they have taken the place of their scores, and
//    the next step's scores S = Q K^T.  While one tile's rows are exponentiated the other's products run.
// Measured: 1024 tokens of 2 sequences over 16384 keys, 4 heads of 128 features, 281 us, 947 TFLOP/s, 57 % of a library product; 64 features 495.  (A call
// lasts as long as its longest sequence: one of 16384 beside one of 1024 takes the same 281.)  A step takes 4200 cycles, of which the row warps' weights are
// 2300 a tile: without any exponential they would take 80 % of the time, without the conversion of keys and values all of it, and with scores that never
// wait for the products of the step before (64 features leave the room) 99 %.
// Slower were (beside 304 us): two threads a row 343, scores of 64 keys in two buffers 358, scores loaded a quarter at a time 347; eight warps that
// bring keys and values, which leave the rows 160 registers each, took the 304.
// Every wait is bounded; one that gives up ends the CTA's others, and the next call on the device reports it.
#include <math_constants.h>

#include <type_traits>

#include "ma_cache.cuh"
#include "ma_sm100.cuh"

namespace ma {
namespace {

using namespace sm100;

constexpr int kKeys = 128, kTileRows = 128, kRows = 2 * kTileRows;
constexpr int kThreads = 512, kBringers = 128;  // warps 0-3, 4-7: rows; 8-11: keys and values; 12: products (13-15 make it a warpgroup)
constexpr int kLaunchRegs = 128, kRowRegs = 184, kBringerRegs = 104, kIssuerRegs = 40;
static_assert(256 * kRowRegs + kBringers * kBringerRegs + 128 * kIssuerRegs <= kThreads * kLaunchRegs, "setmaxnreg draws on the launch's registers");
constexpr int kRing = 8;  // steps whose pages and scales are kept
constexpr float kBelow = 7.0f, kSlack = 15.0f;  // (ma_cache_attend.cu)
// Scores beyond this (in units of log2) have references in two parts (rows_apart).
constexpr float kApart = 8192.0f;

enum Bar { kQ0, kQ1, kKFull, kKEmpty = kKFull + 2, kVFull = kKEmpty + 2, kVEmpty = kVFull + 2, kS0 = kVEmpty + 2, kS1, kP0, kP1, kO, kDrain, kBars };

// What the rows need of a step's 8 blocks.
struct alignas(16) Blocks {
  float k_scale[8], v_inverse[8], v_log[8];  // the values' scales as their inverse and logarithm
  int page[2][8];  // of keys and of values; -1: zeros
};

template <int D>
struct Layout {
  static constexpr int kTileBytes = 128 * D * 2;  // 128 rows in f16: panels of 64 features
  static constexpr int kQ = 0, kK = 2 * kTileBytes, kV = kK + 2 * kTileBytes, kBlocks = kV + 2 * kTileBytes;
  static constexpr int kBarriers = kBlocks + kRing * (int)sizeof(Blocks), kFlags = kBarriers + 8 * kBars, kBytes = kFlags + 16;
  static constexpr int kSmem = kBytes + 1024;  // (tiles start on 1024-byte boundaries)
};

struct PromptArgs {
  AttendArgs a;
  int pieces;        // that the keys of a CTA's rows are cut into
  int* wait_status;  // mapped host word: a wait that gave up
};

template <int N>
__device__ __forceinline__ void regs_inc() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void regs_dec() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

__device__ __forceinline__ uint32_t widen2(uint32_t codes) {
  uint32_t r;
  asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\t}" : "=r"(r) : "r"(codes));
  return r;
}
__device__ __forceinline__ uint32_t widen2_upper(uint32_t codes) {
  uint32_t r;
  asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, hi;\n\t}" : "=r"(r) : "r"(codes));
  return r;
}
// The larger of the two, NaN if one is: a key of NaN takes its rows with it.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
// 2^x on the multipliers, for x up to 2^7: the special function units are what the weights wait for.  x = n + f with f in [-1/2, 1/2], 2^f by a
// polynomial of degree 5 (minimax in the relative error, found by exchange; 2^-22.7 with the coefficients in 32 bits), times 2^n.
constexpr int kByProducts = 1;  // of 4 pairs of weights, these (us of 16384 keys: none 295, one 288, two 320)
__device__ __forceinline__ float2 exp2_by_products(float2 x) {
  x = make_float2(max_nan(x.x, -126.0f), max_nan(x.y, -126.0f));
  const float2 round = make_float2(12582912.0f, 12582912.0f);  // 1.5 * 2^23: its last bits are n
  const float2 t = add2(x, round), f = sub2(x, sub2(t, round));
  auto both = [](float c) { return make_float2(c, c); };
  float2 p = fma2(f, both(1.3277939e-3f), both(9.6757580e-3f));
  p = fma2(p, f, both(5.5507097e-2f));
  p = fma2(p, f, both(2.4022114e-1f));
  p = fma2(p, f, both(6.9314694e-1f));
  p = fma2(p, f, both(1.0000001f));
  // times 2^n, a product, in which a NaN stays one (added to its bits n would make a number of it)
  return mul2(p, make_float2(__int_as_float((__float_as_int(t.x) << 23) + 0x3f800000), __int_as_float((__float_as_int(t.y) << 23) + 0x3f800000)));
}
// What a row needs for its scores: those of keys [low, high) count.
struct RowScores {
  float factor, softcap;
  int low, high;
};
// A step's weights of a row whose scores are far from zero, of the 128 scores at t_s (t0: the first one's key), in place of them, and into the row's sum.
//
// The kernel's loop has a weight as the exponential of fma(score, f, log - reference), with the logarithm of the value's scale in the reference: where
// the last bit of a score is worth more than a unit, such a difference is anything, the weights leave f16 and the logarithm is lost.  Here a score is
// rounded first and a reference is a score S and a logarithm L: (score - S) + (log - L) is exact for the keys that count, however large S is.
// A few scores are in registers at a time, read and scaled twice: 1276 us for the loop's 281 (2 x 1024 tokens over 16384 keys of 128 features).
template <typename T, int D>
__device__ __forceinline__ void rows_apart(const RowScores& r, const Blocks& b, int t0, uint32_t t_s, uint32_t t_o, bool has_sums, float* sum, float* S_row, float* L_row) {
  // (What leaves the kernel's loop as it was; us of 2 x 1024 tokens over 16384 keys with 1 / 2 / 4: 128 features, bf16 281 / 288 / 285, f16 285 / 282 / 278; 64
  // features, bf16 273 / 266 / 277, f16 275 / 270 / 271.)
  constexpr int kUnroll = D == 64 ? 2 : std::is_same<T, __half>::value ? 4 : 1;
  auto load = [&](int q, float (&x)[32]) {
    tmem_ld32_nowait(t_s + 32 * q, x);
    tmem_wait_ld(x);
#pragma unroll
    for (int j = 0; j < 32; ++j) {
      const float f = r.factor * b.k_scale[2 * q + j / 16];
      x[j] = r.softcap > 0.0f ? capped(x[j] * f, r.softcap) : __fmul_rn(x[j], fmaxf(f, 1e-37f));
      const int t = t0 + 32 * q + j;
      if (t < r.low || t >= r.high) x[j] = -CUDART_INF_F;
    }
  };
  float S = *S_row, L = *L_row, best = -CUDART_INF_F, best_log = 0.0f;
#pragma unroll kUnroll
  for (int q = 0; q < 4; ++q) {
    float x[32];
    load(q, x);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float most = x[16 * h];
#pragma unroll
      for (int j = 1; j < 16; ++j) most = fmaxf(most, x[16 * h + j]);
      const float log = b.v_log[2 * q + h];
      if ((most - best) + (log - best_log) > 0.0f) {
        best = most;
        best_log = log;
      }
    }
  }
  const bool raise = (best - S) + (best_log - L) > kSlack;
  if (__any_sync(0xffffffffu, raise)) {
    const float S0 = S, L0 = L;
    if (raise) {
      S = best;
      L = best_log - kBelow;
    }
    const float shrink = raise ? ex2((S0 - S) + (L0 - L)) : 1.0f;
    *sum *= shrink;
    if (has_sums) {
#pragma unroll 1
      for (int q = 0; q < D / 16; ++q) {
        float o[16];
        uint32_t z[16];
        tmem_ld16_nowait(t_o + 16 * q, o);
        tmem_wait_ld16(o);
#pragma unroll
        for (int j = 0; j < 16; ++j) z[j] = __float_as_uint(o[j] * shrink);
        tmem_st16(t_o + 16 * q, z);
      }
    }
  }
  *S_row = S;
  *L_row = L;
  const float base = S == -CUDART_INF_F ? 0.0f : S;
  float all = 0.0f;
#pragma unroll kUnroll
  for (int q = 0; q < 4; ++q) {  // (the weights of 32 keys take the place of 16 scores that have been read)
    float x[32];
    uint32_t y[16];
    load(q, x);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float log = b.v_log[2 * q + h] - L;
      float part = 0.0f;
#pragma unroll
      for (int j = 0; j < 16; j += 2) {
        const float p0 = ex2((x[16 * h + j] - base) + log), p1 = ex2((x[16 * h + j + 1] - base) + log);
        part += p0 + p1;
        y[8 * h + j / 2] = pack2<__half>(p0, p1);
      }
      all = fmaf(part, b.v_inverse[2 * q + h], all);
    }
    tmem_st16(t_s + 16 * q, y);
  }
  *sum += all;
}
// 16 codes as two 16-byte chunks of a row.
__device__ __forceinline__ void put_codes(uint32_t panel, uint32_t row, uint32_t chunk, const uint4& c) {
  st_shared_v4(panel + swz(row, chunk), widen2(c.x), widen2_upper(c.x), widen2(c.y), widen2_upper(c.y));
  st_shared_v4(panel + swz(row, chunk + 1), widen2(c.z), widen2_upper(c.z), widen2(c.w), widen2_upper(c.w));
}

// kExpire: of the self-test, in which the values of a CTA's first step never arrive.
template <typename T, int D, bool kExpire = false>
__global__ void __launch_bounds__(kThreads, 1) prompt_kernel(const __grid_constant__ PromptArgs args) {
  using L = Layout<D>;
  constexpr int kPanel = 128 * 128;  // bytes of 128 rows of 64 features
  constexpr uint32_t kTmemS = 0, kTmemO = 256;  // columns: S (and P) of both tiles, then O of both
  extern __shared__ uint8_t smem_raw[];
  const AttendArgs& a = args.a;
  const CacheArgs& c = a.cache;
  const uint32_t base = (smem_u32(smem_raw) + 1023) & ~1023u;
  uint8_t* const smem = smem_raw + (base - smem_u32(smem_raw));
  Blocks* const blocks = reinterpret_cast<Blocks*>(smem + L::kBlocks);
  volatile int* const abort_flag = reinterpret_cast<volatile int*>(smem + L::kFlags);
  const int tid = threadIdx.x, warp = tid >> 5;
  auto bar = [&](int i) { return base + L::kBarriers + 8 * i; };
  // (the vote brings the lanes of a warp back together, and of one mind)
  constexpr int kTries = kExpire ? 4096 : 1 << 21;
  auto wait = [&](int b, uint32_t phase, int tries = 1 << 21) {
    const bool r = __all_sync(0xffffffffu, mbar_wait_abortable(bar(b), phase & 1u, abort_flag, tries));
    if (!r) *abort_flag = 1;
    return r;
  };

  grid_wait();
  // --- the CTA's rows and keys; row blocks with more keys come first
  const int piece = blockIdx.x % args.pieces, unit = blockIdx.x / args.pieces;  // unit: (block from the last on, sequence, head)
  const int e_head = unit % (a.E * c.heads), block = a.row_blocks - 1 - unit / (a.E * c.heads);
  const int e = e_head / c.heads, head = e_head % c.heads, row0 = block * kRows;
  int len, count;
  const bool fine = sequence_of(c, e, a.N, &len, &count);
  if (!fine && tid == 0) report(c.status, kBadLength);
  const int first_token = row0 / a.group, last_token = min((row0 + kRows - 1) / a.group, count - 1);
  const bool two = row0 + kTileRows < count * a.group;  // the second tile has rows
  int lo = 0, hi = len;
  if (a.causal) hi = min(len, len - count + last_token + 1);
  if (a.window > 0) lo = max(max(len - count + first_token, 0) - a.window + 1, 0) & ~(kScaleBlock - 1);
  if (first_token >= count) hi = lo;
  const int all_steps = max((hi - lo + kKeys - 1) / kKeys, 0);
  const int step0 = (int)((long long)piece * all_steps / args.pieces), steps = (int)((long long)(piece + 1) * all_steps / args.pieces) - step0;
  lo += step0 * kKeys;

  if (tid == 0) {
    mbar_init(bar(kQ0), 128);
    mbar_init(bar(kQ1), 128);
    for (int i = 0; i < 2; ++i) {
      mbar_init(bar(kKFull + i), kBringers);
      mbar_init(bar(kVFull + i), kBringers);
      mbar_init(bar(kKEmpty + i), 1);
      mbar_init(bar(kVEmpty + i), 1);
      mbar_init(bar(kS0 + i), 1);
      mbar_init(bar(kP0 + i), 128);
    }
    mbar_init(bar(kO), 1);
    mbar_init(bar(kDrain), 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 12) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(base + L::kFlags + 4), "r"(512) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(smem + L::kFlags + 4);

  if (warp < 8) {
    // =========================== a row a thread ======================================================================
    regs_inc<kRowRegs>();
    const int tile = warp >> 2, r = tid & 127, row = row0 + tile * kTileRows + r;
    const int token = row / a.group, h = head * a.group + row - token * a.group;
    const bool exists = token < a.N, real = token < count;
    const uint32_t lanes = (uint32_t)(warp & 3) << 21;  // the warp's 32 lanes of tensor memory
    const uint32_t t_s = tmem + kTmemS + tile * 128 + lanes, t_o = tmem + kTmemO + tile * 128 + lanes;
    const bool works = steps > 0 && (tile == 0 || two), idle = !__any_sync(0xffffffffu, real);
    int keyed = sees_keys(a, len, count, token);
    asm volatile("" : "+r"(keyed));  // (else its four operands take registers through the loop)
    float factor = fabsf(a.scale) * kLog2e, top = -CUDART_INF_F, top_log = 0.0f, sum = 0.0f;  // top_log: of references in two parts
    bool ok = true;
    if (works) {
      // the query row in f16, brought to magnitudes of 1 to 2 by a power of two (bf16), with the sign of the scale
      const uint4* src = reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(a.q.ptr) + (real ? e * a.q.se + h * a.q.sh + token * a.q.sn : 0));
      uint4 raw[D / 8];
#pragma unroll
      for (int i = 0; i < D / 8; ++i) raw[i] = real ? src[i] : make_uint4(0, 0, 0, 0);
      float down = 1.0f;
      if constexpr (!std::is_same<T, __half>::value) {
        float amax = 0.0f;
#pragma unroll
        for (int i = 0; i < D / 8; ++i) {
          const uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float2 x = unpack2<T>(w[j]);
            amax = fmaxf(amax, fmaxf(fabsf(x.x), fabsf(x.y)));
          }
        }
        const int exponent = min(max((int)(__float_as_uint(amax) >> 23), 27), 253);  // biased
        down = __uint_as_float((uint32_t)(254 - exponent) << 23);
        factor *= __uint_as_float((uint32_t)exponent << 23);
      }
      if (a.scale < 0.0f) down = -down;
      const uint32_t to = base + L::kQ + tile * L::kTileBytes;
#pragma unroll
      for (int i = 0; i < D / 8; ++i) {
        const uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
        uint32_t y[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 x = unpack2<T>(w[j]);
          y[j] = pack2<__half>(x.x * down, x.y * down);
        }
        st_shared_v4(to + (i >> 3) * kPanel + swz(r, i & 7), y[0], y[1], y[2], y[3]);
      }
      fence_async_smem();
      mbar_arrive(bar(kQ0 + tile));
      const int place = len - count + token;
      // (rows of padding, whose results are not looked at, ask for no mask)
      const int high = !real ? 0x7fffffff : a.causal ? place + 1 : len, low = real && a.window > 0 ? max(place, 0) - a.window + 1 : 0;
      // Warps of nothing but padding leave the schedulers to the others: 64 rows of 64 heads over 16384 keys 189 -> 138 us.
      for (int i = 0; i < steps && idle && ok; ++i) {
        ok = wait(kS0 + tile, i);
        if (ok) mbar_arrive(bar(kP0 + tile));
      }
      int i = 0;
      for (; i < steps && !idle; ++i) {
        ok = wait(kS0 + tile, i);
        if (!ok) break;
        tc_fence_after();
        const Blocks& b = blocks[i & (kRing - 1)];
        const int t0 = lo + i * kKeys;
        uint32_t y[4][16];
        float more;
        // The weights are found with the reference as it is, next to the maximum that says whether it would do; where not, once more.
#pragma unroll 1
        for (;;) {
          float v[4][32];
#pragma unroll
          for (int q = 0; q < 4; ++q) tmem_ld32_nowait(t_s + 32 * q, v[q]);
#pragma unroll
          for (int q = 0; q < 4; ++q) tmem_wait_ld(v[q]);
          // (scores in units of log2 e) = f * S, and never zero: a mask is minus infinity times f, and rows of zeros, small keys and a small
          // scale together leave 32 bits.  (S is 2^17 at most of bf16 rows, 2^32 of f16.)
          auto f = [&](int j) { return a.softcap > 0.0f ? 1.0f : fmaxf(factor * b.k_scale[j], 1e-37f); };
          if (a.softcap > 0.0f) {
#pragma unroll
            for (int q = 0; q < 4; ++q)
#pragma unroll
              for (int j = 0; j < 32; ++j)
                v[q][j] = capped(v[q][j] * (factor * b.k_scale[2 * q + j / 16]), a.softcap);
          }
          if (t0 < low || t0 + kKeys > high) {
#pragma unroll
            for (int q = 0; q < 4; ++q)
#pragma unroll
              for (int j = 0; j < 32; ++j)
                if (t0 + 32 * q + j < low || t0 + 32 * q + j >= high) v[q][j] = -CUDART_INF_F;
          }
          const float ref = top == -CUDART_INF_F ? 0.0f : top;
          float most = -CUDART_INF_F;
          more = 0.0f;
          // weights times the values' scale; the sum of the weights takes it out again, block by block
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            float* x = &v[j / 2][(j & 1) * 16];
            float m0 = max3(x[0], x[1], x[2]), m1 = max3(x[3], x[4], x[5]);
            m0 = max3(m0, x[6], x[7]);
            m1 = max3(m1, x[8], x[9]);
            m0 = max3(m0, x[10], x[11]);
            m1 = max3(m1, x[12], x[13]);
            m0 = max3(m0, x[14], x[15]);
            const float fj = f(j), log = b.v_log[j], shift = log - ref;
            most = fmaxf(most, fmaf(fmaxf(m0, m1), fj, log));
            float2 part = make_float2(0.0f, 0.0f);
#pragma unroll
            for (int k = 0; k < 16; k += 2) {
              float2 p = fma2(make_float2(x[k], x[k + 1]), make_float2(fj, fj), make_float2(shift, shift));
              p = k % 8 < 8 - 2 * kByProducts ? make_float2(ex2(p.x), ex2(p.y)) : exp2_by_products(p);
              part = k == 0 ? p : add2(part, p);
              y[j / 2][(j & 1) * 8 + k / 2] = pack2<__half>(p.x, p.y);
            }
            more = fmaf(part.x + part.y, b.v_inverse[j], more);
          }
          if (!__any_sync(0xffffffffu, most > top + kSlack)) break;
          if (__any_sync(0xffffffffu, fabsf(most) > kApart && most > -CUDART_INF_F)) goto apart;
          const float before = top;
          top = fmaxf(top, most - kBelow);
          const float shrink = ex2(before - (top == -CUDART_INF_F ? 0.0f : top));
          sum *= shrink;
          if (i > 0) {  // (the scores of this step are there, so the products of the one before are done)
#pragma unroll 1
            for (int q = 0; q < D / 16; ++q) {
              float o[16];
              uint32_t z[16];
              tmem_ld16_nowait(t_o + 16 * q, o);
              tmem_wait_ld16(o);
#pragma unroll
              for (int j = 0; j < 16; ++j) z[j] = __float_as_uint(o[j] * shrink);
              tmem_st16(t_o + 16 * q, z);
            }
          }
        }
        sum += more;
#pragma unroll
        for (int q = 0; q < 4; ++q) tmem_st16(t_s + 16 * q, y[q]);
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(bar(kP0 + tile));
      }
      // From the first step on in which a row of the warp has a score far from zero, its rows go this way: a path of its own, of which the loop above knows a jump
      // and no state (a flag in its place costs 4 to 6 % of all calls, the same inside the loop 15).
      if (false) {
      apart:
#pragma unroll 1
        for (bool there = true;; there = false) {  // (the first step's scores have been waited for)
          if (!there) ok = wait(kS0 + tile, i);
          if (!ok) break;
          tc_fence_after();
          rows_apart<T, D>({factor, a.softcap, low, high}, blocks[i & (kRing - 1)], lo + i * kKeys, t_s, t_o, i > 0, &sum, &top, &top_log);
          tmem_wait_st();
          tc_fence_before();
          mbar_arrive(bar(kP0 + tile));
          if (++i == steps) break;
        }
      }
      if (ok) {
        ok = wait(kO, 0);
        tc_fence_after();
      }
    }
    // --- result: rows without a key, and of padding, are zero
    if (ok) {
      const float unit_of = ex2(top_log);  // (a piece's reference is one number)
      const float inverse = top > -CUDART_INF_F ? 1.0f / sum : 0.0f;  // (no key, no reference)
      const size_t slot = ((size_t)unit * args.pieces + piece) * kRows + tile * kTileRows + r;
      T* const dst = reinterpret_cast<T*>(const_cast<void*>(a.out.ptr)) + e * a.out.se + h * a.out.sh + token * a.out.sn;
#pragma unroll
      for (int q = 0; q < D / 32; ++q) {
        float o[32];
        if (works) tmem_ld32(t_o + 32 * q, o);
        if (!works || !keyed) {
#pragma unroll
          for (int j = 0; j < 32; ++j) o[j] = 0.0f;
        }
        if (!exists) continue;
        if (args.pieces == 1) {
#pragma unroll
          for (int j = 0; j < 32; j += 8)
            *reinterpret_cast<uint4*>(dst + 32 * q + j) =
                make_uint4(pack2<T>(o[j] * inverse, o[j + 1] * inverse), pack2<T>(o[j + 2] * inverse, o[j + 3] * inverse),
                           pack2<T>(o[j + 4] * inverse, o[j + 5] * inverse), pack2<T>(o[j + 6] * inverse, o[j + 7] * inverse));
        } else {
#pragma unroll
          for (int j = 0; j < 32; j += 4)
            *reinterpret_cast<float4*>(a.part_o + slot * D + 32 * q + j) = make_float4(o[j] * unit_of, o[j + 1] * unit_of, o[j + 2] * unit_of, o[j + 3] * unit_of);
        }
      }
      if (args.pieces > 1 && exists) *reinterpret_cast<float2*>(a.part_ml + 2 * slot) = make_float2(top, sum * unit_of);
    }
    if (args.pieces > 1 && tid == 0 && piece == 0)
      a.split[unit] = make_int4((e * c.heads + head) * a.row_blocks + block, unit * args.pieces, (unit + 1) * args.pieces - 1, 0);
  } else if (warp < 12) {
    // =========================== keys and values =====================================================================
    regs_dec<kBringerRegs>();
    const int t = tid - 256, page_mask = (1 << c.page_shift) - 1;
    // Threads 0-7 look after a block each: its page two steps ahead of its scales, those a step ahead of the bytes.
    auto page_at = [&](int i) {
      const int at = lo + i * kKeys + t * kScaleBlock;
      if (i >= steps || at >= len) return -1;
      const int page = page_of(c, e, at);
      if (page < 0) report(c.status, kBadPage);
      return page;
    };
    auto scale_at = [&](const float* scales, long long sp, long long sh, int i, int page) {
      return page < 0 ? 1.0f : scales[page * sp + head * sh + ((lo + i * kKeys + t * kScaleBlock) & page_mask) / kScaleBlock];
    };
    auto put_blocks = [&](int i, int page, float ks, float vs) {
      Blocks& b = blocks[i & (kRing - 1)];
      // (a scale of zero is another one before zeros, since a mask is minus infinity times the keys' scale and a weight is divided by the values': one for keys,
      // the smallest that there is for values, whose weights are not to be above those of any other block's)
      b.page[0][t] = ks == 0.0f ? -1 : page;
      b.page[1][t] = vs == 0.0f ? -1 : page;
      b.k_scale[t] = ks == 0.0f ? 1.0f : ks;
      b.v_inverse[t] = vs == 0.0f ? exp2f(-kLeastLog) : 1.0f / vs;
      b.v_log[t] = vs == 0.0f ? kLeastLog : __log2f(vs);
    };
    auto meet = [&]() { asm volatile("bar.sync 1, %0;" ::"n"(kBringers) : "memory"); };
    int page_next = -1;
    if (t < 8) {
      for (int i = 0; i < 2; ++i) {
        const int page = page_at(i);
        put_blocks(i, page, scale_at(c.k_scale, c.ks_sp, c.ks_sh, i, page), scale_at(c.v_scale, c.vs_sp, c.vs_sh, i, page));
      }
      page_next = page_at(2);
    }
    meet();
    // A thread has a 16-byte piece of 4 in each panel of rows t / 4 + 32 j: eight threads write 4 pieces of two rows, an even and an
    // odd one, whose chunks the swizzle puts on different banks.
    constexpr int kPanels = D / 64;
    uint4 raw[2][4][kPanels];  // keys and values on their way
    auto load = [&](int which, int i) {
      const uint8_t* const all = which ? c.v : c.k;
      const uint32_t sp = which ? a.v16[0] : a.k16[0], sh = which ? a.v16[1] : a.k16[1], st = which ? a.v16[2] : a.k16[2];
      const Blocks& b = blocks[i & (kRing - 1)];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int row = (t >> 2) + 32 * j, token = lo + i * kKeys + row, page = b.page[which][row / kScaleBlock];
        const uint8_t* const src = all + 16 * ((uint32_t)page * (uint64_t)sp + (uint32_t)head * (uint64_t)sh + (uint32_t)(token & page_mask) * (uint64_t)st + (t & 3));
#pragma unroll
        for (int x = 0; x < kPanels; ++x)
          raw[which][j][x] = token < len && page >= 0 ? *reinterpret_cast<const uint4*>(src + 64 * x) : make_uint4(0, 0, 0, 0);
      }
    };
    auto put = [&](int which, uint32_t to) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int x = 0; x < kPanels; ++x) put_codes(to + x * kPanel, (t >> 2) + 32 * j, 2 * (t & 3), raw[which][j][x]);
      fence_async_smem();
    };
    if (steps > 0) {
      load(0, 0);
      load(1, 0);
    }
    bool ok = true;  // (whatever happens, all meet at each step)
    for (int i = 0; i < steps; ++i) {
      float ks = 1.0f, vs = 1.0f;
      int page_after = -1;
      if (t < 8) {
        ks = scale_at(c.k_scale, c.ks_sp, c.ks_sh, i + 2, page_next);
        vs = scale_at(c.v_scale, c.vs_sp, c.vs_sh, i + 2, page_next);
        page_after = page_at(i + 3);
      }
      const int stage = i & 1;
      ok = ok && (i < 2 || wait(kKEmpty + stage, (i >> 1) - 1));
      if (ok) {
        put(0, base + L::kK + stage * L::kTileBytes);
        mbar_arrive(bar(kKFull + stage));
      }
      if (i + 1 < steps) load(0, i + 1);
      ok = ok && (i < 2 || wait(kVEmpty + stage, (i >> 1) - 1));
      if (ok) {
        put(1, base + L::kV + stage * L::kTileBytes);
        if (!kExpire || i > 0) mbar_arrive(bar(kVFull + stage));
      }
      if (i + 1 < steps) load(1, i + 1);
      if (t < 8) {
        put_blocks(i + 2, page_next, ks, vs);
        page_next = page_after;
      }
      meet();
    }
  } else {
    regs_dec<kIssuerRegs>();
  }
  if (warp == 12) {
    // =========================== products ============================================================================
    constexpr uint32_t kScores = instr_desc(0, 0, 0, kKeys, kTileRows), kSums = instr_desc(0, 0, 1, D, kTileRows);
    constexpr uint32_t kTileUnits = L::kTileBytes >> 4, kPanelUnits = kPanel >> 4;
    auto scores = [&](int tile, int i) {
      const uint32_t da = smem_desc_lo(base + L::kQ, 16) + tile * kTileUnits, db = smem_desc_lo(base + L::kK, 16) + (i & 1) * kTileUnits;
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk)
        mma_f16_lo(tmem + kTmemS + tile * 128, da + (kk >> 2) * kPanelUnits + (kk & 3) * 2, db + (kk >> 2) * kPanelUnits + (kk & 3) * 2, kScores, kk > 0);
      mma_commit(bar(kS0 + tile));
    };
    auto sums = [&](int tile, int i) {
      const uint32_t db = smem_desc_lo(base + L::kV, kPanel) + (i & 1) * kTileUnits;
#pragma unroll
      for (int kk = 0; kk < kKeys / 16; ++kk)
        mma_f16_ts(tmem + kTmemO + tile * 128, tmem + kTmemS + tile * 128 + kk * 8, db + kk * 128, kSums, i > 0 || kk > 0);
    };
    const int tiles = two ? 2 : 1;
    bool ok = steps > 0 && wait(kKFull, 0);
    for (int tile = 0; tile < tiles && ok; ++tile) {
      ok = wait(kQ0 + tile, 0);
      if (!ok) break;
      tc_fence_after();
      if (elect_one()) {
        scores(tile, 0);
        if (tile == tiles - 1) mma_commit(bar(kKEmpty));
      }
      __syncwarp();
    }
    for (int i = 0; i < steps && ok; ++i) {
      ok = wait(kVFull + (i & 1), i >> 1, kTries) && (i + 1 == steps || wait(kKFull + ((i + 1) & 1), (i + 1) >> 1));
      for (int tile = 0; tile < tiles && ok; ++tile) {
        ok = wait(kP0 + tile, i);
        if (!ok) break;
        tc_fence_after();
        if (elect_one()) {
          sums(tile, i);
          if (tile == tiles - 1) mma_commit(bar(kVEmpty + (i & 1)));
          if (i + 1 < steps) {
            scores(tile, i + 1);
            if (tile == tiles - 1) mma_commit(bar(kKEmpty + ((i + 1) & 1)));
          } else if (tile == tiles - 1) {
            mma_commit(bar(kO));
          }
        }
        __syncwarp();
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (*abort_flag != 0) {
    if (tid == 0 && args.wait_status != nullptr) *reinterpret_cast<volatile int*>(args.wait_status) = 800;
    // products that were issued have read their operands and written tensor memory before the CTA leaves
    if (warp == 12 && elect_one()) {
      mma_commit(bar(kDrain));
      (void)mbar_wait(bar(kDrain), 0);
    }
    __syncwarp();
  }
  if (warp == 12) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
}

}  // namespace

// Pieces that the keys of 256 rows are cut into: with fewer blocks of rows than SMs, what brings them to all SMs, as long as a piece has
// four steps at least.  us, pieces / none: 4 heads x 256 rows over 16384 keys 34 / 275, over 4096 28 / 80, over 1500 27 / 38; 32 heads over 16384 94 / 286, 64
// over 8000 97 / 150.
int prompt_pieces(int E, int N, int H, int kv_heads, long long longest) {
  const long long units = (long long)E * kv_heads * (((long long)H / kv_heads * N + kRows - 1) / kRows);
  const long long fill = sm_count() / units, most = longest / (4 * kKeys);
  return (int)(fill < 2 || most < 2 ? 1 : fill < most ? fill : most);
}

size_t prompt_workspace(int E, int N, int H, int kv_heads, int width, long long longest) {
  const long long pieces = prompt_pieces(E, N, H, kv_heads, longest);
  if (pieces == 1) return 256;
  const size_t units = (size_t)E * kv_heads * (((size_t)H / kv_heads * N + kRows - 1) / kRows);
  return (units * sizeof(int4) + 255) / 256 * 256 + units * pieces * kRows * (width + 2) * sizeof(float);
}

cudaError_t launch_prompt(AttendArgs a, int dtype, int width, void* workspace, long long longest, int* wait_status, bool wait_expiry, cudaStream_t stream) {
  a.row_blocks = (a.group * a.N + kRows - 1) / kRows;
  const long long units = (long long)a.E * a.cache.heads * a.row_blocks;
  PromptArgs args{a, prompt_pieces(a.E, a.N, a.H, a.cache.heads, longest), wait_status};
  char* at = reinterpret_cast<char*>(workspace);
  args.a.split = reinterpret_cast<int4*>(at);
  args.a.part_o = reinterpret_cast<float*>(at + ((size_t)units * sizeof(int4) + 255) / 256 * 256);
  args.a.part_ml = args.a.part_o + (size_t)units * args.pieces * kRows * width;
  const bool bf = dtype == MA_B200_BF16;
  const void* fn = width == 128 ? (bf ? (const void*)prompt_kernel<__nv_bfloat16, 128> : (const void*)prompt_kernel<__half, 128>)
                                : (bf ? (const void*)prompt_kernel<__nv_bfloat16, 64> : (const void*)prompt_kernel<__half, 64>);
  if (wait_expiry) fn = width == 128 ? (const void*)prompt_kernel<__nv_bfloat16, 128, true> : (const void*)prompt_kernel<__nv_bfloat16, 64, true>;
  const size_t smem = width == 128 ? Layout<128>::kSmem : Layout<64>::kSmem;
  // a build whose launch does not cover the roles' registers must not start: setmaxnreg would wait for them without end
  static std::atomic<unsigned long long> checked[6];
  int dev = 0;
  cudaError_t err = cudaGetDevice(&dev);
  if (err != cudaSuccess) return err;
  std::atomic<unsigned long long>& done = checked[(width == 128) * 3 + (wait_expiry ? 2 : bf)];
  if (dev >= 64 || !(done.load(std::memory_order_relaxed) >> dev & 1)) {
    cudaFuncAttributes fa;
    err = cudaFuncGetAttributes(&fa, fn);
    if (err != cudaSuccess) return err;
    if (fa.numRegs != kLaunchRegs) return cudaErrorLaunchOutOfResources;
    if (dev < 64) done.fetch_or(1ull << dev, std::memory_order_relaxed);
  }
  err = allow_dynamic_smem(fn, smem);
  if (err != cudaSuccess) return err;
  void* params[] = {(void*)&args};
  err = launch_kernel(fn, dim3((unsigned)(units * args.pieces)), dim3(kThreads), params, smem, stream);
  if (err != cudaSuccess || args.pieces == 1) return err;
  return launch_join(args.a, dtype, width, kRows, (int)units, 1, stream);
}

}  // namespace ma
