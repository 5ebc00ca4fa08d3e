// Attention over the cache: the pieces of split heads are joined here, and a call goes to the kernel for few rows (ma_cache_attend.inc) or
// the one for many (ma_cache_prompt.cu).
#include "ma_cache_attend.inc"

namespace ma {
namespace {

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

// The second kernel of a call whose heads were split.
template <typename T, int D>
cudaError_t join(const AttendArgs& a, const Plan& plan, cudaStream_t stream) {
  int tile_rows = 8 * plan.nt;
  void* join_args[] = {(void*)&a, (void*)&tile_rows};
  const unsigned rows = a.group * a.N < tile_rows ? a.group * a.N : tile_rows;
  const long long entries = a.split_by_head ? (long long)a.E * a.cache.heads * a.row_blocks : plan.grid;
  // Few heads have many pieces each: a CTA for 32 features of a row, else a warp for a row.  us of the call, the one / the other: a token of 2 heads of 131071
  // tokens 23 / 59, of 8 heads of 32768 23 / 31; 64 heads of 32768 (more rows than that) 101 / 99.
  if (entries * rows < 2 * sm_count()) return launch_kernel((const void*)join_kernel<T, D>, dim3((unsigned)entries, rows, D / 32), dim3(256), join_args, 0, stream);
  return launch_join(a, std::is_same<T, __half>::value ? MA_B200_F16 : MA_B200_BF16, D, tile_rows, (int)entries, 2, stream);
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

size_t attend_tree_workspace(int E, int N, int H, int kv_heads, int width, int window, long long longest) {
  return H / kv_heads * (long long)N >= kPromptRows ? prompt_tree_workspace(E, N, H, kv_heads, width, longest) : attend_workspace(E, N, H, kv_heads, width, window, longest);
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
  const cudaError_t err = a.parents != nullptr ? launch_few_tree(a, dtype, width, plan.nt, plan.warps, plan.grid, stream)
                                               : launch_few_of<false>(a, dtype, width, plan.nt, plan.warps, plan.grid, stream);
  if (err != cudaSuccess || plan.whole) return err;
  const bool bf = dtype == MA_B200_BF16;
  if (width == 128) return bf ? join<__nv_bfloat16, 128>(a, plan, stream) : join<__half, 128>(a, plan, stream);
  return bf ? join<__nv_bfloat16, 64>(a, plan, stream) : join<__half, 64>(a, plan, stream);
}

}  // namespace ma
