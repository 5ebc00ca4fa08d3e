// Softmax attention of a few query rows over a paged cache in 8 bits.
//
// Bound by memory: a key/value pair of a head is 2 D bytes and takes part in 4 D operations a row, so that up to some 30 rows the cache's
// bytes are all that counts.  The kernel is built around them:
//  * The keys of all sequences and heads are one list of steps of 128 tokens, shared out evenly: CTA c takes steps [c S / G, (c + 1) S / G)
//    whatever the lengths are, so that a ragged batch and a single long sequence both fill the GPU.  Lengths are read on the device; a
//    head whose steps lie in several CTAs has its pieces joined by a second small kernel.
//  * A warp takes 32 of a step's tokens, through a ring of its own in shared memory that is filled asynchronously, steps ahead and
//    across the ends of heads; nothing in the loop waits for another warp.
//  * Scores are taken as (keys x rows): the keys are the 16-row operand of the 16 x 8 x 16 matrix instruction and up to 8 query rows (the heads
//    of a group, times tokens) its 8 columns, so that no part of it is padding when 8 rows share a key head.  Bytes go from shared memory
//    straight into operand registers: the order of features in a contraction is free, and a lane's 16 bytes of a row are taken
//    as they lie.  The weighted values are (features x rows) in the same way, two tokens' bytes interleaved by byte permutation; the
//    weights change sides by an 8 x 8 transpose between lanes.
//  * e4m3 is exact in f16, so the products are f16 with 32-bit sums whatever the queries' type; a bf16 row is scaled by a power of two to
//    magnitudes of 1 to 2 first (exact but for elements 2^-23 below the row's largest).  A block's key scale multiplies its scores; its value
//    scale goes into the weights, and the running maximum is taken over weight times scale, so that f16 weights are at most 2^kSlack (kBelow).
// Measured, a token each: 32 sequences of up to 8192 tokens, 8 heads of 128 features, 270 MB in 59 us; every further byte comes at 6.3 TB/s, 96 %
// of a copy (64 features: 4.9, the bytes' conversion and the weights bind), and some 12 us go to the start, the unequal finish of the CTAs and the
// join.  One sequence of 131071 tokens and 2 heads, 67 MB in 23 us; of 500 tokens and 12 heads of 64 features 7.4 us.
#include <math_constants.h>

#include <type_traits>

#include "ma_cache.cuh"
#include "ma_sm100.cuh"

namespace ma {
namespace {

using sm100::ex2;
using sm100::kLog2e;
using sm100::smem_u32;

// Weights in f16 (times their value's scale): the reference is kBelow under the largest when it is set, and raised when one would pass 2^kSlack, so that the largest are
// 2^7 to 2^15, under the 65504 of the type, and only those below 2^-21 to 2^-29 of the largest have fewer bits than 11.
// (Beside a score of 2^27 and more the logarithm of a value's scale is lost from the reference, and a weight is anything from the scale itself to 2^(7 +- 16).  A
// reference of two numbers, score and logarithm, as the kernel for many rows has it there, costs every call of this one 3 to 5 %, and the shortest 0.8 us of 6.7:
// in the loop, as a rare branch in it and as a call from there.  So there the scales are asked to be from 2^-14 to 2^15.)
constexpr float kBelow = 7.0f, kSlack = 15.0f;
constexpr int kSlice = 32;  // tokens of a warp at a time
constexpr int kWide = 12;   // warps of a CTA that has an SM to itself: as many as fit in with two tiles of rows

template <int D, int NT, int W>
struct Shape {
  static constexpr int kStep = W * kSlice;  // tokens of a CTA at a time
  static constexpr int kStages = D == 128 ? 2 : W == 4 ? 3 : 4;
  static constexpr int kStageBytes = 2 * kSlice * D + 16;  // keys, values and their two scales each
  static constexpr int kRows = 8 * NT;
  static constexpr bool kSharedRows = NT > 1;  // the query rows' operands are in shared memory: there are no registers for them
  static constexpr int kRing = W * kStages * kStageBytes;
  static constexpr int kOperandBytes = kSharedRows ? kRows * D * 2 : 0;
  static constexpr int kSmem = kRing + kOperandBytes;
  static constexpr int kCtas = W > 4 ? 1 : NT > 2 ? 2 : D == 64 && NT == 1 ? 4 : 3;  // of an SM: what registers and shared memory allow
};

// Byte offset of 16-byte piece `piece` of token t in a slice: pieces are permuted so that neither the reads of the keys (8 rows x 4 pieces)
// nor those of the values (tokens 0, 2, 4, 6 x 8 pieces) meet in a bank.
template <int D>
__device__ __forceinline__ uint32_t piece_at(uint32_t t, uint32_t piece) {
  if constexpr (D == 128) return t * 128 + ((piece ^ ((t & 2) ^ ((((t >> 2) ^ t) & 1) << 2))) << 4);
  return (t >> 1) * 128 + (((((t & 1) << 2) | piece) ^ (((t >> 1) & 3) << 1)) << 4);
}

__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool real) {  // else zeros
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(real ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t dst, const void* src, bool real) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(real ? 4 : 0) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Two e4m3 values as two f16, exactly.
__device__ __forceinline__ uint32_t widen(uint32_t two) {
  uint32_t r;
  asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\t}" : "=r"(r) : "r"(two));
  return r;
}
__device__ __forceinline__ uint32_t widen_upper(uint32_t two) {
  uint32_t r;
  asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, hi;\n\t}" : "=r"(r) : "r"(two));
  return r;
}
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}
// What a sequence's keys look like to the call.
struct Sequence {
  int len, count, lo, steps;  // keys [lo, len) are looked at, in `steps` steps (one at least)
};
template <int kStep>
__device__ __forceinline__ Sequence sequence(const AttendArgs& a, int e) {
  Sequence s;
  sequence_of(a.cache, e, a.N, &s.len, &s.count);
  s.lo = a.window > 0 ? max(max(s.len - s.count, 0) - a.window + 1, 0) & ~(kScaleBlock - 1) : 0;
  s.steps = max((s.len - s.lo + kStep - 1) / kStep, 1);
  return s;
}

// The steps of a call in `parts` shares that differ by one at most, the longer ones spread evenly: share i begins at i * whole + i * rest / parts.
// (Divisions of 64 bits take longer than all else in front of the first load.)
struct Share {
  long long whole;
  int rest, parts;
  __device__ Share(long long total, int n) : parts(n) {
    whole = total < 0x7fffffff ? (int)total / n : total / n;
    rest = (int)(total - whole * n);
  }
  __device__ long long first(int i) const { return i * whole + (int)((long long)i * rest < 0x7fffffff ? i * rest / parts : (long long)i * rest / parts); }
  __device__ int of(long long step) const {  // the share that a step is in
    int i = min((int)((float)step / ((float)whole + (float)rest / (float)parts)) + 1, parts - 1);  // (within a share or two)
    while (first(i) > step) --i;
    while (i + 1 < parts && first(i + 1) <= step) ++i;
    return i;
  }
};

// A place in the list of steps.
struct Place {
  int e, head, block, step;  // block: of rows
  Sequence s;
};
template <int kStep>
__device__ __forceinline__ void advance(const AttendArgs& a, Place* p) {
  if (++p->step < p->s.steps) return;
  p->step = 0;
  if (++p->block < a.row_blocks) return;
  p->block = 0;
  if (++p->head < a.cache.heads) return;
  p->head = 0;
  if (++p->e < a.E) p->s = sequence<kStep>(a, p->e);
}

template <typename T, int D, int NT, int W>
__global__ void __launch_bounds__(W * 32, Shape<D, NT, W>::kCtas) attend_kernel(const __grid_constant__ AttendArgs a) {
  using S = Shape<D, NT, W>;
  constexpr int kStep = S::kStep;
  constexpr int kWords = D / 16;   // 32-bit words of a key row that a lane holds; also products of 16 features, and feature tiles of 16
  constexpr int kValueWords = D / 32;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ long long warp_sum[W];
  __shared__ __align__(16) float row_scale[S::kRows];
  __shared__ __align__(16) int2 row_keys[S::kRows];  // keys [x, y) that a row sees
  __shared__ float2 tops[W][S::kRows];           // running maximum and sum of each warp
  __shared__ int where_e;
  __shared__ long long where_at;
  const CacheArgs& c = a.cache;
  const int tid = threadIdx.x, w = tid >> 5, lane = tid & 31, g = lane >> 2, q4 = lane & 3;
  const int units = c.heads * a.row_blocks;
  if (!a.whole_heads) dependents_may_start();  // (the joining kernel may come up where there is room)
  grid_wait();

  // --- this CTA's share of the steps
  Place now;
  long long total = 0, ctas = gridDim.x, end = 0;  // steps of the call, CTAs that have some, and the end of this one's
  Share share(0, 1);
  int steps = 0, unit;
  if (a.whole_heads) {  // as many heads (and blocks of rows) as another CTA
    const long long heads = (long long)a.E * units, u0 = blockIdx.x * heads / ctas, u1 = (blockIdx.x + 1) * heads / ctas;
    now.e = (int)(u0 / units);
    unit = (int)(u0 - (long long)now.e * units);
    now.s = sequence<kStep>(a, now.e);
    now.step = 0;
    for (long long u = u0; u < u1;) {
      const int e = (int)(u / units);
      const long long next = min(u1, (long long)(e + 1) * units);
      steps += (int)(next - u) * sequence<kStep>(a, e).steps;
      u = next;
    }
    int x, y;
    for (int e = blockIdx.x * W * 32 + tid; e < a.E; e += gridDim.x * W * 32)
      if (!sequence_of(c, e, a.N, &x, &y)) report(c.status, kBadLength);
  } else {  // prefix sums over the sequences, a run of them per thread
    const int run = (a.E + W * 32 - 1) / (W * 32);
    long long mine = 0;
    for (int e = tid * run; e < min(a.E, (tid + 1) * run); ++e) {
      mine += sequence<kStep>(a, e).steps;
      int x, y;
      if (blockIdx.x == 0 && !sequence_of(c, e, a.N, &x, &y)) report(c.status, kBadLength);
    }
    long long upto = mine;
#pragma unroll
    for (int m = 1; m < 32; m <<= 1) {
      const long long o = __shfl_up_sync(0xffffffffu, upto, m);
      if (lane >= m) upto += o;
    }
    if (lane == 31) warp_sum[w] = upto;
    __syncthreads();
    for (int i = 0; i < w; ++i) upto += warp_sum[i];
    for (int i = 0; i < W; ++i) total += warp_sum[i];
    total *= units;
    ctas = min(ctas, total);
    if (blockIdx.x >= ctas) {
      if (tid == 0 && !a.split_by_head) a.split[blockIdx.x] = make_int4(-1, 0, 0, 0);
      return;
    }
    share = Share(total, (int)ctas);
    const long long begin = share.first(blockIdx.x);
    end = share.first(blockIdx.x + 1);
    steps = (int)(end - begin);
    if ((upto - mine) * units <= begin && begin < upto * units) {
      long long at = (upto - mine) * units;
      int e = tid * run;
      for (;; ++e) {
        const long long n = (long long)sequence<kStep>(a, e).steps * units;
        if (begin < at + n) break;
        at += n;
      }
      where_e = e;
      where_at = begin - at;
    }
    __syncthreads();
    now.e = where_e;
    now.s = sequence<kStep>(a, now.e);
    unit = where_at < 0x7fffffff ? (int)where_at / now.s.steps : (int)(where_at / now.s.steps);
    now.step = (int)(where_at - (long long)unit * now.s.steps);
  }
  now.head = unit / a.row_blocks;
  now.block = unit - now.head * a.row_blocks;
  Place ahead = now;

  // --- the warp's ring of slices
  const uint32_t ring = smem_u32(smem) + w * S::kStages * S::kStageBytes;
  uint2* const shared_rows = reinterpret_cast<uint2*>(smem + S::kRing);
  constexpr int kLanesPerRow = D / 16, kRowsPerPass = 32 / kLanesPerRow, kPasses = kScaleBlock / kRowsPerPass;  // passes of 16 tokens
  const int lane_row = lane / kLanesPerRow, piece = lane % kLanesPerRow;
  const int page_mask = (1 << c.page_shift) - 1;
  // Pages of the slice that is fetched next: looked up a slice earlier, so that the copies do not wait for the table.
  int pages[2] = {-1, -1};
  auto look_up = [&]() {
    const int t0 = ahead.s.lo + ahead.step * kStep + w * kSlice;
#pragma unroll
    for (int b = 0; b < 2; ++b) pages[b] = t0 + b * kScaleBlock < ahead.s.len ? page_of(c, ahead.e, t0 + b * kScaleBlock) : -1;
  };
  auto fetch = [&](int stage) {
    const int t0 = ahead.s.lo + ahead.step * kStep + w * kSlice;
    const int left = ahead.s.len - t0;
    if (left <= 0) return;
    const uint32_t at = ring + stage * S::kStageBytes;
    const bool whole = left >= kSlice && pages[0] >= 0 && pages[1] >= 0;
    if (!whole && lane == 0 && (pages[0] < 0 || (left > kScaleBlock && pages[1] < 0))) report(c.status, kBadPage);
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const uint32_t page = max(pages[b], 0), row = ((t0 + b * kScaleBlock) & page_mask) + lane_row;
      const uint8_t* k = c.k + 16 * (page * (uint64_t)a.k16[0] + ahead.head * (uint64_t)a.k16[1] + row * (uint64_t)a.k16[2] + piece);
      const uint8_t* v = c.v + 16 * (page * (uint64_t)a.v16[0] + ahead.head * (uint64_t)a.v16[1] + row * (uint64_t)a.v16[2] + piece);
#pragma unroll
      for (int i = 0; i < kPasses; ++i, k += a.k16[2] * (16ull * kRowsPerPass), v += a.v16[2] * (16ull * kRowsPerPass)) {
        const int t = b * kScaleBlock + i * kRowsPerPass + lane_row;
        const uint32_t to = at + piece_at<D>(t, piece);
        if (whole) {
          copy16(to, k);
          copy16(to + kSlice * D, v);
        } else {
          const bool real = t < left && pages[b] >= 0;
          copy16(to, real ? k : c.k, real);
          copy16(to + kSlice * D, real ? v : c.v, real);
        }
      }
    }
    if (lane < 4) {  // scales: keys of both blocks, values of both
      const int page = lane & 1 ? pages[1] : pages[0], row = (t0 + (lane & 1) * kScaleBlock) & page_mask;
      const long long p = max(page, 0);
      const float* src = lane < 2 ? c.k_scale + p * c.ks_sp + ahead.head * c.ks_sh : c.v_scale + p * c.vs_sp + ahead.head * c.vs_sh;
      copy4(at + 2 * kSlice * D + lane * 4, src + (page >= 0 ? row / kScaleBlock : 0), page >= 0);
    }
  };
  look_up();
#pragma unroll
  for (int i = 0; i < S::kStages - 1; ++i) {
    if (i < steps) {
      fetch(i);
      advance<kStep>(a, &ahead);
      if (i + 1 < steps) look_up();
    }
    copies_commit();
  }

  uint32_t qf[S::kSharedRows ? 1 : NT][kWords][2];  // query rows as the second operand
  float o[NT][kWords][4], top[NT][2], sum[NT][2];   // of rows 2 q4, 2 q4 + 1 of each tile
  int full_low = 0, full_high = 0;                  // keys that all rows see
  bool fresh = true, later = false;                 // a head begins; the CTA has finished (a piece of) one
  int stage = 0;
  for (int i = 0; i < steps; ++i) {
    const int row0 = now.block * S::kRows;
    if (fresh) {
      fresh = false;
      // Rows 8 n + g as operands, and what their scores are multiplied by (units of log2 e).
      auto load_rows = [&](int n, uint32_t (&to)[kWords][2]) {
        const int r = row0 + n * 8 + g, token = r / a.group, h = now.head * a.group + r - token * a.group;
        const bool real = token < now.s.count;
        const T* src = reinterpret_cast<const T*>(a.q.ptr) + (real ? now.e * a.q.se + h * a.q.sh + token * a.q.sn : 0);
        float factor = a.scale * kLog2e;
        uint2 raw[kWords];
#pragma unroll
        for (int k = 0; k < kWords; ++k)
          raw[k] = real ? *reinterpret_cast<const uint2*>(src + (k >> 2) * 64 + q4 * 16 + (k & 3) * 4) : make_uint2(0, 0);
        if constexpr (!std::is_same<T, __half>::value) {
          float amax = 0.0f;
#pragma unroll
          for (int k = 0; k < kWords; ++k) {
            const float2 x = sm100::unpack2<T>(raw[k].x), y = sm100::unpack2<T>(raw[k].y);
            amax = fmaxf(fmaxf(amax, fmaxf(fabsf(x.x), fabsf(x.y))), fmaxf(fabsf(y.x), fabsf(y.y)));
          }
          amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
          amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
          const int exponent = min(max((int)(__float_as_uint(amax) >> 23), 27), 253);  // biased
          const float down = __uint_as_float((uint32_t)(254 - exponent) << 23);
          factor *= __uint_as_float((uint32_t)exponent << 23);
#pragma unroll
          for (int k = 0; k < kWords; ++k) {
            const float2 x = sm100::unpack2<T>(raw[k].x), y = sm100::unpack2<T>(raw[k].y);
            to[k][0] = sm100::pack2<__half>(x.x * down, x.y * down);
            to[k][1] = sm100::pack2<__half>(y.x * down, y.y * down);
          }
        } else {
#pragma unroll
          for (int k = 0; k < kWords; ++k) {
            to[k][0] = raw[k].x;
            to[k][1] = raw[k].y;
          }
        }
        return factor;
      };
      if constexpr (S::kSharedRows) {  // a tile of rows a warp
        if (w < NT) {
          const float factor = load_rows(w, qf[0]);
#pragma unroll
          for (int k = 0; k < kWords; ++k) shared_rows[(w * kWords + k) * 32 + lane] = make_uint2(qf[0][k][0], qf[0][k][1]);
          if (q4 == 0) row_scale[w * 8 + g] = factor;
        }
      } else {
        const float factor = load_rows(0, qf[0]);
        if (w == 0 && q4 == 0) row_scale[g] = factor;
      }
      if (tid < S::kRows) {
        const int token = (row0 + tid) / a.group, place = now.s.len - now.s.count + token;
        row_keys[tid] = make_int2(a.window > 0 ? max(place, 0) - a.window + 1 : 0, token >= now.s.count ? 0 : a.causal ? place + 1 : now.s.len);
      }
      __syncthreads();
      // rows are in the order of their tokens; those of padding have results of zero whatever they see
      full_low = 0;
      full_high = now.s.len;
      if (a.causal && row0 / a.group < now.s.count) {
        const int last = min((row0 + S::kRows - 1) / a.group, now.s.count - 1);
        full_high = row_keys[0].y;
        if (a.window > 0) full_low = max(now.s.len - now.s.count + last, 0) - a.window + 1;
      }
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        top[n][0] = top[n][1] = -CUDART_INF_F;
        sum[n][0] = sum[n][1] = 0.0f;
#pragma unroll
        for (int m = 0; m < kWords; ++m)
#pragma unroll
          for (int j = 0; j < 4; ++j) o[n][m][j] = 0.0f;
      }
    }
    copies_wait<S::kStages - 2>();
    __syncwarp();
    if (i + S::kStages - 1 < steps) {
      fetch(stage == 0 ? S::kStages - 1 : stage - 1);
      advance<kStep>(a, &ahead);
      if (i + S::kStages < steps) look_up();
    }
    copies_commit();
    const int t0 = now.s.lo + now.step * kStep + w * kSlice;
    if (t0 < now.s.len) {
      const uint8_t* const keys = smem + (w * S::kStages + stage) * S::kStageBytes;
      const uint8_t* const values = keys + kSlice * D;
      float s[2][NT][4];
      uint32_t kw[2][2][kWords];
#pragma unroll
      for (int mt = 0; mt < 2; ++mt)
#pragma unroll
        for (int r = 0; r < 2; ++r)
#pragma unroll
          for (int h = 0; h < kWords / 4; ++h) {
            const uint4 v = *reinterpret_cast<const uint4*>(keys + piece_at<D>(mt * 16 + r * 8 + g, q4 + 4 * h));
            kw[mt][r][4 * h] = v.x; kw[mt][r][4 * h + 1] = v.y; kw[mt][r][4 * h + 2] = v.z; kw[mt][r][4 * h + 3] = v.w;
          }
#pragma unroll
      for (int mt = 0; mt < 2; ++mt)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int j = 0; j < 4; ++j) s[mt][n][j] = 0.0f;
      // (the two blocks' products take turns: a product waits for the one before it in its sum)
#pragma unroll
      for (int k = 0; k < kWords; ++k)
#pragma unroll
        for (int mt = 0; mt < 2; ++mt) {
          const uint32_t a0 = widen(kw[mt][0][k]), a1 = widen(kw[mt][1][k]), a2 = widen_upper(kw[mt][0][k]), a3 = widen_upper(kw[mt][1][k]);
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            if constexpr (S::kSharedRows) {
              const uint2 b = shared_rows[(n * kWords + k) * 32 + lane];
              mma(s[mt][n], a0, a1, a2, a3, b.x, b.y);
            } else {
              mma(s[mt][n], a0, a1, a2, a3, qf[n][k][0], qf[n][k][1]);
            }
          }
        }
      const float4 scales = *reinterpret_cast<const float4*>(keys + 2 * kSlice * D);
      const float ks[2] = {scales.x, scales.y}, vs[2] = {scales.z, scales.w};
      // (values of scale zero count as of the smallest scale there is: their keys have weights, which the reference has to stand for, but no more than that)
      const float vl[2] = {fmaxf(__log2f(scales.z), kLeastLog), fmaxf(__log2f(scales.w), kLeastLog)};
      uint32_t weights[2][NT][2];
      const bool whole = t0 >= full_low && t0 + kSlice <= full_high;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const float2 rs = *reinterpret_cast<const float2*>(row_scale + n * 8 + 2 * q4);
        float most[2] = {-CUDART_INF_F, -CUDART_INF_F};
#pragma unroll
        for (int mt = 0; mt < 2; ++mt)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            float x = s[mt][n][j] * (ks[mt] * (j & 1 ? rs.y : rs.x));
            if (a.softcap > 0.0f) x = capped(x, a.softcap);
            s[mt][n][j] = x;
          }
        if (!whole) {
          const int4 seen = *reinterpret_cast<const int4*>(row_keys + n * 8 + 2 * q4);
#pragma unroll
          for (int mt = 0; mt < 2; ++mt)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const int t = t0 + mt * 16 + g + (j >> 1) * 8;
              if (t < (j & 1 ? seen.z : seen.x) || t >= (j & 1 ? seen.w : seen.y)) s[mt][n][j] = -CUDART_INF_F;
            }
        }
#pragma unroll
        for (int mt = 0; mt < 2; ++mt)
#pragma unroll
          for (int j = 0; j < 4; ++j) most[j & 1] = fmaxf(most[j & 1], s[mt][n][j] + vl[mt]);
        // The rows' reference is raised only when a weight would pass 2^kSlack: seldom once a head's first keys have been seen, and until then
        // no lane has to know the others' scores.  (A difference, which is exact; a reference plus kSlack is rounded to the last bit of a large reference, and a weight could
        // pass 2^16.)
        if (__any_sync(0xffffffffu, most[0] - top[n][0] > kSlack || most[1] - top[n][1] > kSlack)) {
#pragma unroll
          for (int j = 0; j < 2; ++j) {
#pragma unroll
            for (int m = 4; m < 32; m <<= 1) most[j] = fmaxf(most[j], __shfl_xor_sync(0xffffffffu, most[j], m));
            const float before = top[n][j];
            top[n][j] = fmaxf(before, most[j] - kBelow);
            const float shrink = ex2(before - (top[n][j] == -CUDART_INF_F ? 0.0f : top[n][j]));
            sum[n][j] *= shrink;
#pragma unroll
            for (int m = 0; m < kWords; ++m) {
              o[n][m][j] *= shrink;
              o[n][m][2 + j] *= shrink;
            }
          }
        }
        float base[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) base[j] = top[n][j] == -CUDART_INF_F ? 0.0f : top[n][j];
#pragma unroll
        for (int mt = 0; mt < 2; ++mt) {
          float p[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            p[j] = ex2(s[mt][n][j] - base[j & 1]);
            sum[n][j & 1] += p[j];
            p[j] *= vs[mt];
          }
          weights[mt][n][0] = transpose8(sm100::pack2<__half>(p[0], p[1]));
          weights[mt][n][1] = transpose8(sm100::pack2<__half>(p[2], p[3]));
        }
      }
#pragma unroll
      for (int mt = 0; mt < 2; ++mt) {
        uint32_t vw[4][kValueWords];  // tokens 2 q4, 2 q4 + 1, 2 q4 + 8, 2 q4 + 9
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int t = mt * 16 + 2 * q4 + (j & 1) + (j >> 1) * 8;
          if constexpr (D == 128) {
            const uint4 v = *reinterpret_cast<const uint4*>(values + piece_at<D>(t, g));
            vw[j][0] = v.x; vw[j][1] = v.y; vw[j][2] = v.z; vw[j][3] = v.w;
          } else {
            const uint2 v = *reinterpret_cast<const uint2*>(values + piece_at<D>(t, g >> 1) + (g & 1) * 8);
            vw[j][0] = v.x; vw[j][1] = v.y;
          }
        }
#pragma unroll
        for (int k = 0; k < kValueWords; ++k) {
          const uint32_t x0 = __byte_perm(vw[0][k], vw[1][k], 0x5140), x1 = __byte_perm(vw[0][k], vw[1][k], 0x7362);
          const uint32_t y0 = __byte_perm(vw[2][k], vw[3][k], 0x5140), y1 = __byte_perm(vw[2][k], vw[3][k], 0x7362);
          const uint32_t a0 = widen(x0), a1 = widen_upper(x0), a2 = widen(y0), a3 = widen_upper(y0);
          const uint32_t b0 = widen(x1), b1 = widen_upper(x1), b2 = widen(y1), b3 = widen_upper(y1);
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            mma(o[n][2 * k], a0, a1, a2, a3, weights[mt][n][0], weights[mt][n][1]);
            mma(o[n][2 * k + 1], b0, b1, b2, b3, weights[mt][n][0], weights[mt][n][1]);
          }
        }
      }
    }

    const bool last_of_head = now.step + 1 == now.s.steps;
    if (last_of_head || i + 1 == steps) {
      // --- the warps' sums into one: each brings its own to the common maximum and leaves it in its ring, in the stage that it has just
      // used up, a tile of rows at a time (by turns in its two halves); warp w < 4 then adds up rows 2 w and 2 w + 1
      fresh = true;
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
#pragma unroll
          for (int m = 4; m < 32; m <<= 1) sum[n][j] += __shfl_xor_sync(0xffffffffu, sum[n][j], m);
          if (g == 0) tops[w][n * 8 + 2 * q4 + j] = make_float2(top[n][j], sum[n][j]);
        }
      __syncthreads();
      const bool alone = last_of_head && i >= now.step;  // all of the head's steps were this CTA's
      const int slot = 2 * blockIdx.x + (later ? 1 : 0);
      float* const mine = reinterpret_cast<float*>(smem + (w * S::kStages + stage) * S::kStageBytes);
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float most = -CUDART_INF_F;
#pragma unroll
          for (int v = 0; v < W; ++v) most = fmaxf(most, tops[v][n * 8 + 2 * q4 + j].x);
          const float x = ex2(top[n][j] - (most == -CUDART_INF_F ? 0.0f : most));
#pragma unroll
          for (int m = 0; m < kWords; ++m) {
            mine[(n & 1) * 8 * D + (m * 4 + j) * 32 + lane] = o[n][m][j] * x;
            mine[(n & 1) * 8 * D + (m * 4 + 2 + j) * 32 + lane] = o[n][m][2 + j] * x;
          }
        }
        __syncthreads();
        // 8 neighbouring features of a row a lane (64 features: 4), in the places where the lanes of the product had them
        constexpr int kRun = D / 16;
        const int j = lane >> 4, u = lane & 15, r = n * 8 + 2 * w + j;
        if (w < 4 && row0 + r < a.N * a.group) {
          float x[kRun];
#pragma unroll
          for (int f = 0; f < kRun; ++f) x[f] = 0.0f;
#pragma unroll
          for (int v = 0; v < W; ++v) {
            const float* theirs = reinterpret_cast<const float*>(smem + (v * S::kStages + stage) * S::kStageBytes);
#pragma unroll
            for (int f = 0; f < kRun; ++f) x[f] += theirs[(n & 1) * 8 * D + (((u & 1) * (kWords / 2) + f / 2) * 4 + j + 2 * (f & 1)) * 32 + (u >> 1) * 4 + w];
          }
          float most = -CUDART_INF_F, all = 0.0f;
#pragma unroll
          for (int v = 0; v < W; ++v) most = fmaxf(most, tops[v][r].x);
          const float base = most == -CUDART_INF_F ? 0.0f : most;
#pragma unroll
          for (int v = 0; v < W; ++v) all += tops[v][r].y * ex2(tops[v][r].x - base);
          if (alone) {
            const int token = (row0 + r) / a.group, h = now.head * a.group + row0 + r - token * a.group;
            const float inverse = all > 0.0f ? 1.0f / all : 0.0f;
            if (!sees_keys(a, now.s.len, now.s.count, token)) {
#pragma unroll
              for (int f = 0; f < kRun; ++f) x[f] = 0.0f;
            }
            T* dst = reinterpret_cast<T*>(const_cast<void*>(a.out.ptr)) + now.e * a.out.se + h * a.out.sh + token * a.out.sn + u * kRun;
            if constexpr (D == 128)
              *reinterpret_cast<uint4*>(dst) = make_uint4(sm100::pack2<T>(x[0] * inverse, x[1] * inverse), sm100::pack2<T>(x[2] * inverse, x[3] * inverse),
                                                          sm100::pack2<T>(x[4] * inverse, x[5] * inverse), sm100::pack2<T>(x[6] * inverse, x[7] * inverse));
            else
              *reinterpret_cast<uint2*>(dst) = make_uint2(sm100::pack2<T>(x[0] * inverse, x[1] * inverse), sm100::pack2<T>(x[2] * inverse, x[3] * inverse));
          } else {
            float* dst = a.part_o + ((size_t)slot * S::kRows + r) * D + u * kRun;
#pragma unroll
            for (int f = 0; f < kRun; f += 4) *reinterpret_cast<float4*>(dst + f) = make_float4(x[f], x[f + 1], x[f + 2], x[f + 3]);
            if (u == 0) *reinterpret_cast<float2*>(a.part_ml + ((size_t)slot * S::kRows + r) * 2) = make_float2(most, all);
          }
        }
      }
      __syncthreads();
      if (tid == 0 && !a.whole_heads && (a.split_by_head ? i >= now.step : i + 1 == steps)) {
        // a head that began here and goes on in the next CTA: the entry names it, this CTA, and the CTA of its last step
        const int which = (now.e * c.heads + now.head) * a.row_blocks + now.block;
        int4 entry = make_int4(-1, 0, 0, 0);
        if (!last_of_head && i >= now.step) {
          const long long last = end - 1 + (now.s.steps - 1 - now.step);
          entry = make_int4(which, blockIdx.x, share.of(last), later ? 1 : 0);
        }
        a.split[a.split_by_head ? which : (int)blockIdx.x] = entry;
      }
      later = true;
    }
    stage = stage + 1 == S::kStages ? 0 : stage + 1;
    advance<kStep>(a, &now);
  }
}

// Joins the pieces of the heads that were split: a CTA for each entry of the table of the kernel above, row, and 32 features.  Every 16 bytes
// of a row are summed over the pieces by several threads, each with many loads in flight, on their way before the weights are known.  The table has an entry for each head where there are fewer heads than CTAs, else one for each CTA.
template <typename T, int D>
__global__ void __launch_bounds__(256) join_kernel(const __grid_constant__ AttendArgs a, int tile_rows) {
  constexpr int W = 32, kLanes = W / 4, kGroups = 256 / kLanes, kMost = 1024, kInFlight = 8;
  __shared__ float2 weights[kMost];  // of the first pieces: maximum and sum
  __shared__ float4 sums[256];
  __shared__ float totals[256], reduced[8];
  grid_wait();
  const int4 entry = a.split[blockIdx.x];
  if (entry.x < 0) return;
  const int block = entry.x % a.row_blocks, head = entry.x / a.row_blocks % a.cache.heads, e = entry.x / a.row_blocks / a.cache.heads;
  const int r = blockIdx.y, row = block * tile_rows + r, token = row / a.group, h = head * a.group + row - token * a.group;
  if (token >= a.N) return;
  const int pieces = entry.z - entry.y + 1;
  auto slot = [&](int i) { return (size_t)(2 * (entry.y + i) + (i == 0 ? entry.w : 0)) * tile_rows + r; };
  const int tid = threadIdx.x, lane = tid % kLanes, group = tid / kLanes;
  const float4* const rows = reinterpret_cast<const float4*>(a.part_o) + blockIdx.z * kLanes + lane;
  float4 x[kInFlight];
  auto load = [&](int i) {
#pragma unroll
    for (int j = 0; j < kInFlight; ++j)
      if (i + j * kGroups < pieces) x[j] = rows[slot(i + j * kGroups) * (D / 4)];
  };
  load(group);  // (on the way while the weights are found)
  float top = -CUDART_INF_F;
  for (int i = tid; i < pieces; i += 256) {
    const float2 ml = *reinterpret_cast<const float2*>(a.part_ml + 2 * slot(i));
    if (i < kMost) weights[i] = ml;
    top = fmaxf(top, ml.x);
  }
#pragma unroll
  for (int m = 16; m > 0; m >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, m));
  if ((tid & 31) == 0) reduced[tid >> 5] = top;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 8; ++i) top = fmaxf(top, reduced[i]);
  const float base = top == -CUDART_INF_F ? 0.0f : top;
  float4 acc = make_float4(0, 0, 0, 0);
  float total = 0.0f;
  for (int i = group; i < pieces; i += kGroups * kInFlight) {
#pragma unroll
    for (int j = 0; j < kInFlight; ++j) {
      const int n = i + j * kGroups;
      if (n >= pieces) break;
      const float2 ml = n < kMost ? weights[n] : *reinterpret_cast<const float2*>(a.part_ml + 2 * slot(n));
      const float weight = ex2(ml.x - base);
      total += weight * ml.y;
      acc.x += weight * x[j].x; acc.y += weight * x[j].y; acc.z += weight * x[j].z; acc.w += weight * x[j].w;
    }
    load(i + kGroups * kInFlight);
  }
  sums[tid] = acc;
  totals[tid] = total;
  __syncthreads();
  if (group != 0) return;
  for (int i = 1; i < min(kGroups, pieces); ++i) {
    const float4 y = sums[i * kLanes + lane];
    acc.x += y.x; acc.y += y.y; acc.z += y.z; acc.w += y.w;
    total += totals[i * kLanes + lane];
  }
  int len, count;
  sequence_of(a.cache, e, a.N, &len, &count);
  const float inverse = total > 0.0f ? 1.0f / total : 0.0f;
  if (!sees_keys(a, len, count, token)) acc = make_float4(0, 0, 0, 0);
  T* dst = reinterpret_cast<T*>(const_cast<void*>(a.out.ptr)) + e * a.out.se + h * a.out.sh + token * a.out.sn + blockIdx.z * W + lane * 4;
  *reinterpret_cast<uint2*>(dst) = make_uint2(sm100::pack2<T>(acc.x * inverse, acc.y * inverse), sm100::pack2<T>(acc.z * inverse, acc.w * inverse));
}

// The same where there are many rows: a warp for each row, without a word to the others.
template <typename T, int D>
__global__ void __launch_bounds__(256) join_rows_kernel(const __grid_constant__ AttendArgs a, int tile_rows, int rows, int entries, int stride) {
  constexpr int kRun = D / 32, kInFlight = 4;
  using Run = std::conditional_t<kRun == 4, float4, float2>;
  grid_wait();
  const int lane = threadIdx.x & 31, task = blockIdx.x * 8 + (threadIdx.x >> 5), at = task / rows, r = task - at * rows;
  if (at >= entries) return;
  const int4 entry = a.split[at];
  if (entry.x < 0) return;
  const int block = entry.x % a.row_blocks, unit = entry.x / a.row_blocks, e = unit / a.cache.heads, head = unit - e * a.cache.heads;
  const int row = block * tile_rows + r, token = row / a.group, h = head * a.group + row - token * a.group;
  if (token >= a.N) return;
  const int pieces = entry.z - entry.y + 1;
  auto slot = [&](int i) { return (size_t)(stride * (entry.y + i) + (i == 0 ? entry.w : 0)) * tile_rows + r; };
  float acc[kRun] = {}, total = 0.0f, top = -CUDART_INF_F;
  for (int i0 = 0; i0 < pieces; i0 += kInFlight) {
    float2 ml[kInFlight];
    Run x[kInFlight];
#pragma unroll
    for (int j = 0; j < kInFlight; ++j) {
      ml[j] = make_float2(-CUDART_INF_F, 0.0f);
      x[j] = Run{};
      if (i0 + j >= pieces) continue;
      ml[j] = *reinterpret_cast<const float2*>(a.part_ml + 2 * slot(i0 + j));
      x[j] = reinterpret_cast<const Run*>(a.part_o + slot(i0 + j) * D)[lane];
    }
    const float before = top;
#pragma unroll
    for (int j = 0; j < kInFlight; ++j) top = fmaxf(top, ml[j].x);
    const float base = top == -CUDART_INF_F ? 0.0f : top, shrink = ex2(before - base);
    total *= shrink;
#pragma unroll
    for (int f = 0; f < kRun; ++f) acc[f] *= shrink;
#pragma unroll
    for (int j = 0; j < kInFlight; ++j) {
      const float weight = ex2(ml[j].x - base);
      total += weight * ml[j].y;
      const float* y = reinterpret_cast<const float*>(&x[j]);
#pragma unroll
      for (int f = 0; f < kRun; ++f) acc[f] += weight * y[f];
    }
  }
  int len, count;
  sequence_of(a.cache, e, a.N, &len, &count);
  const float inverse = total > 0.0f ? 1.0f / total : 0.0f;
  if (!sees_keys(a, len, count, token)) {
#pragma unroll
    for (int f = 0; f < kRun; ++f) acc[f] = 0.0f;
  }
  T* dst = reinterpret_cast<T*>(const_cast<void*>(a.out.ptr)) + e * a.out.se + h * a.out.sh + token * a.out.sn + lane * kRun;
  if constexpr (kRun == 4)
    *reinterpret_cast<uint2*>(dst) = make_uint2(sm100::pack2<T>(acc[0] * inverse, acc[1] * inverse), sm100::pack2<T>(acc[2] * inverse, acc[3] * inverse));
  else
    *reinterpret_cast<uint32_t*>(dst) = sm100::pack2<T>(acc[0] * inverse, acc[1] * inverse);
}

// From as many rows on, the tcgen05 kernel.  us, it / this one, heads of 128 features: 64 sequences x 8 heads x 1024 tokens, 32 rows 96 / 74, 48 rows
// 97 / 122, 80 rows 99 / 177; 8 x 8 x 2048, 32 rows 28 / 25, 48 rows 29 / 35; 1 x 8 x 32768, 32 rows 44 / 42, 48 rows 45 / 59; 1 x 8 x 2048, 32 rows
// 18 / 16, 48 rows 19 / 16, 80 rows 20 / 20.
constexpr long long kPromptRows = 33;

// How a call is shared out.
struct Plan {
  int nt, warps;
  bool whole;       // heads are not split, and there is nothing to join
  long long grid;
};
Plan plan_of(int E, int N, int H, int kv_heads, int width, int window, long long longest) {
  const int rows = H / kv_heads * N;
  const long long looked_at = (long long)window + N + kScaleBlock;  // keys of a sequence, at most
  if (window > 0 && longest > looked_at) longest = looked_at;
  constexpr int kStep = Shape<128, 1, 4>::kStep;
  // Up to four tiles of 8 rows share a key's conversion; but three or four of them are a long chain for a warp, and where the steps are few
  // anyway, two blocks of rows that both read the keys are done sooner.  us, with as many tiles as there are rows / two: 16 sequences
  // of 20 rows x 4 heads, window 1024, 20.7 / 17.3, of 32 rows and up to 4096 tokens 38.3 / 34.6; 32 of 32 rows and up to 8000 82 / 86, one of
  // 20 rows and 131000 tokens 32 / 43.
  int nt = (rows + 7) / 8;
  if (nt > 2 && (long long)E * kv_heads * ((rows + 8 * nt - 1) / (8 * nt)) * ((longest + kStep - 1) / kStep) <= 16LL * sm_count()) nt = 2;
  const long long units = (long long)E * kv_heads * ((rows + 8 * nt - 1) / (8 * nt));
  // A head of a few steps stays with one CTA: a second kernel costs 3 to 4 us.  Where there are no more heads than SMs, each has a CTA of
  // twelve warps and steps of 384 tokens, 1.8 (64 features) to 3 us; the more of the SMs are busy that way, the longer it pays.
  // us, whole / split, 64 features: 12 heads of 600 tokens 8.0 / 9.5; 84 heads, 1400 11.4 / 13.5, 2000 14.7 / 14.8, 2800 18.8 / 17.7; 144 heads, 1400
  // 11.6 / 17.1, 4000 23.7 / 26.5; 128 features: 8 heads, 600 10.1 / 10.5, 800 12.6 / 10.4; 64 heads, 1400 15.9 / 18.6; 128 heads, 2800 26.2 / 27.7.
  if (nt <= 2 && units <= sm_count() && (longest <= 768 || longest * sm_count() <= 4352 * units)) return {nt, kWide, true, units};
  const bool whole = longest <= 4 * kStep;
  const long long steps = whole ? units : units * ((longest + kStep - 1) / kStep);
  // Rows of 64 features and one tile leave room for a fourth CTA of an SM, where it has some steps.  us, four / three: 32 sequences x 8 heads of 16384
  // tokens 117.6 / 122.3, of 8192 65.4 / 67.3, of 2048 24.6 / 25.3, of 1024 18.3 / 17.8; 2 heads of 131071 19.1 / 17.2.
  constexpr int kFour = Shape<64, 1, 4>::kCtas, kThree = Shape<128, 1, 4>::kCtas;
  const int per_sm = nt > 2 ? Shape<128, 4, 4>::kCtas : width == 64 && nt == 1 && steps >= 6LL * kFour * sm_count() ? kFour : kThree;
  const long long most = per_sm * (long long)sm_count();
  return {nt, 4, whole, steps < most ? steps : most};
}

template <typename T, int D, int NT, int W>
cudaError_t launch(AttendArgs& a, const Plan& plan, cudaStream_t stream) {
  const void* fn = (const void*)attend_kernel<T, D, NT, W>;
  constexpr size_t smem = Shape<D, NT, W>::kSmem;
  cudaError_t err = allow_dynamic_smem(fn, smem);
  if (err != cudaSuccess) return err;
  void* args[] = {(void*)&a};
  err = launch_kernel(fn, dim3((unsigned)plan.grid), dim3(W * 32), args, smem, stream);
  if (err != cudaSuccess || plan.whole) return err;
  int tile_rows = 8 * NT;
  void* join_args[] = {(void*)&a, (void*)&tile_rows};
  const unsigned rows = a.group * a.N < tile_rows ? a.group * a.N : tile_rows;
  const long long entries = a.split_by_head ? (long long)a.E * a.cache.heads * a.row_blocks : plan.grid;
  // Few heads have many pieces each: a CTA for 32 features of a row, else a warp for a row.  us of the call, the one / the other: a token of 2 heads of 131071
  // tokens 23 / 59, of 8 heads of 32768 23 / 31; 64 heads of 32768 (more rows than that) 101 / 99.
  if (entries * rows < 2 * sm_count()) return launch_kernel((const void*)join_kernel<T, D>, dim3((unsigned)entries, rows, D / 32), dim3(256), join_args, 0, stream);
  return launch_join(a, std::is_same<T, __half>::value ? MA_B200_F16 : MA_B200_BF16, D, tile_rows, (int)entries, 2, stream);
}
template <typename T, int D>
cudaError_t launch_rows(AttendArgs& a, const Plan& plan, cudaStream_t stream) {
  if (plan.warps == kWide) return plan.nt == 1 ? launch<T, D, 1, kWide>(a, plan, stream) : launch<T, D, 2, kWide>(a, plan, stream);
  return plan.nt == 1 ? launch<T, D, 1, 4>(a, plan, stream) : plan.nt == 2 ? launch<T, D, 2, 4>(a, plan, stream) :
         plan.nt == 3 ? launch<T, D, 3, 4>(a, plan, stream) : launch<T, D, 4, 4>(a, plan, stream);
}

}  // namespace

cudaError_t launch_join(const AttendArgs& a, int dtype, int width, int tile_rows, int entries, int stride, cudaStream_t stream) {
  int rows = a.group * a.N < tile_rows ? a.group * a.N : tile_rows;
  void* args[] = {(void*)&a, (void*)&tile_rows, (void*)&rows, (void*)&entries, (void*)&stride};
  const bool bf = dtype == MA_B200_BF16;
  const void* fn = width == 128 ? (bf ? (const void*)join_rows_kernel<__nv_bfloat16, 128> : (const void*)join_rows_kernel<__half, 128>)
                                : (bf ? (const void*)join_rows_kernel<__nv_bfloat16, 64> : (const void*)join_rows_kernel<__half, 64>);
  return launch_kernel(fn, dim3((unsigned)(((long long)entries * rows + 7) / 8)), dim3(256), args, 0, stream);
}

size_t attend_workspace(int E, int N, int H, int kv_heads, int width, int window, long long longest) {
  if (H / kv_heads * (long long)N >= kPromptRows) return prompt_workspace(E, N, H, kv_heads, width, longest);
  const Plan plan = plan_of(E, N, H, kv_heads, width, window, longest);
  if (plan.whole) return 256;
  const size_t entries = ((size_t)plan.grid * sizeof(int4) + 255) / 256 * 256;
  return entries + (size_t)plan.grid * 2 * 8 * plan.nt * (width + 2) * sizeof(float);
}

cudaError_t launch_attend(AttendArgs a, int dtype, int width, void* workspace, long long longest, int* wait_status, bool wait_expiry, cudaStream_t stream) {
  const long long strides[6] = {a.cache.k_sp, a.cache.k_sh, a.cache.k_st, a.cache.v_sp, a.cache.v_sh, a.cache.v_st};
  for (int i = 0; i < 6; ++i) (i < 3 ? a.k16[i] : a.v16[i - 3]) = (uint32_t)(strides[i] / 16);
  if (a.group * (long long)a.N >= kPromptRows) return launch_prompt(a, dtype, width, workspace, longest, wait_status, wait_expiry, stream);
  const Plan plan = plan_of(a.E, a.N, a.H, a.cache.heads, width, a.window, longest);
  const int tile_rows = 8 * plan.nt;
  a.row_blocks = (a.group * a.N + tile_rows - 1) / tile_rows;
  char* at = reinterpret_cast<char*>(workspace);
  a.split = reinterpret_cast<int4*>(at);
  a.part_o = reinterpret_cast<float*>(at + ((size_t)plan.grid * sizeof(int4) + 255) / 256 * 256);
  a.part_ml = a.part_o + (size_t)plan.grid * 2 * tile_rows * width;
  a.whole_heads = plan.whole;
  a.split_by_head = (long long)a.E * a.cache.heads * a.row_blocks <= plan.grid;
  const bool bf = dtype == MA_B200_BF16;
  if (width == 128) return bf ? launch_rows<__nv_bfloat16, 128>(a, plan, stream) : launch_rows<__half, 128>(a, plan, stream);
  return bf ? launch_rows<__nv_bfloat16, 64>(a, plan, stream) : launch_rows<__half, 64>(a, plan, stream);
}

}  // namespace ma
