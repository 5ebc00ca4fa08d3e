// C ABI of the rotary positions, the paged cache and the attention over it: argument checks and launches.
#include <math.h>

#include <string>

#include "ma_cache.cuh"

namespace ma {
int fail_with(int code, const std::string& msg);  // ma_api.cu: the calling thread's last error
}

namespace {

using ma::fail_with;

int invalid(const std::string& msg) { return fail_with(MA_B200_INVALID_ARGUMENT, msg); }

ma::View4 view(const ma_b200_tensor& t) { return ma::View4{t.ptr, t.stride_e, t.stride_h, t.stride_n}; }

// A tensor whose rows start on boundaries of `bytes` (of elements of `size`).
int check_tensor(const ma_b200_tensor& t, const char* name, size_t size, size_t bytes) {
  if (t.ptr == nullptr) return invalid(std::string(name) + " is NULL");
  if (t.stride_e < 0 || t.stride_h < 0 || t.stride_n < 0) return invalid(std::string(name) + ": negative stride");
  const long long per = (long long)(bytes / size);
  if (reinterpret_cast<uintptr_t>(t.ptr) % bytes != 0 || t.stride_e % per != 0 || t.stride_h % per != 0 || t.stride_n % per != 0)
    return invalid(std::string(name) + ": rows must start on " + std::to_string(bytes) + "-byte boundaries");
  return MA_B200_OK;
}

int check_cache(const ma_b200_cache& c, const ma_b200_sequences& s, int E, int H, int N, int dtype, ma::CacheArgs* out) {
  if (E <= 0 || N <= 0 || H < 0) return invalid("E, N must be positive and H must not be negative");
  if (dtype != MA_B200_BF16 && dtype != MA_B200_F16) return invalid("dtype must be bf16 or f16");
  if (c.width != 64 && c.width != 128) return fail_with(MA_B200_UNSUPPORTED, "the cache's head width must be 64 or 128");
  if (c.pages <= 0 || c.heads <= 0) return invalid("cache: pages and heads must be positive");
  if (c.page_size < ma::kScaleBlock || (c.page_size & (c.page_size - 1)) != 0) return invalid("cache: page_size must be a power of two from 16 on");
  if (c.k == nullptr || c.v == nullptr || c.k_scale == nullptr || c.v_scale == nullptr) return invalid("cache: a tensor is NULL");
  if (reinterpret_cast<uintptr_t>(c.k) % 16 != 0 || reinterpret_cast<uintptr_t>(c.v) % 16 != 0 || reinterpret_cast<uintptr_t>(c.k_scale) % 4 != 0 ||
      reinterpret_cast<uintptr_t>(c.v_scale) % 4 != 0)
    return invalid("cache: k and v must be 16-byte, the scales 4-byte aligned");
  for (int64_t st : {c.k_stride_page, c.k_stride_head, c.k_stride_token, c.v_stride_page, c.v_stride_head, c.v_stride_token})
    if (st < 0 || st % 16 != 0 || st / 16 > 0xffffffffLL) return invalid("cache: strides of k and v must be multiples of 16, below 2^36 and not negative");
  for (int64_t st : {c.ks_stride_page, c.ks_stride_head, c.vs_stride_page, c.vs_stride_head})
    if (st < 0) return invalid("cache: negative stride of the scales");
  if (s.page_table == nullptr || s.lengths == nullptr) return invalid("page_table and lengths must not be NULL");
  if (s.table_pages <= 0 || s.table_stride < 0) return invalid("page_table must have a column and no negative stride");
  int shift = 0;
  while ((1 << shift) < c.page_size) ++shift;
  int dev = 0;
  const cudaError_t ce = cudaGetDevice(&dev);
  if (ce != cudaSuccess) return fail_with(MA_B200_CUDA_ERROR, std::string("cudaGetDevice: ") + cudaGetErrorString(ce));
  *out = ma::CacheArgs{static_cast<uint8_t*>(c.k), static_cast<uint8_t*>(c.v), c.k_scale, c.v_scale,
                       c.k_stride_page, c.k_stride_head, c.k_stride_token, c.v_stride_page, c.v_stride_head, c.v_stride_token,
                       c.ks_stride_page, c.ks_stride_head, c.vs_stride_page, c.vs_stride_head,
                       c.pages, c.heads, shift, s.page_table, s.table_stride, s.table_pages, s.lengths, s.counts, ma::host_status_word(dev, 1)};
  return MA_B200_OK;
}

// Tokens that a sequence can have by its row of the page table.
long long longest(const ma_b200_sequences& s, int page_size) {
  const long long n = (long long)s.table_pages * page_size;
  return n < 0x7fffff00LL ? n : 0x7fffff00LL;
}

int check_attend_shape(const ma_b200_attend* p) {
  if (p == nullptr) return invalid("problem is NULL");
  if (p->abi_version != MA_B200_ABI_VERSION) return invalid("abi_version mismatch: got " + std::to_string(p->abi_version));
  if (p->E <= 0 || p->H <= 0 || p->N <= 0 || p->cache.heads <= 0 || p->cache.page_size <= 0 || p->sequences.table_pages <= 0)
    return invalid("E, H, N, the cache's heads and page size and the table's columns must be positive");
  if (p->H % p->cache.heads != 0) return invalid("H must be a multiple of the cache's heads");
  const long long rows = (long long)p->H / p->cache.heads * p->N;
  if (rows > (1 << 28) || (rows + 7) / 8 * p->cache.heads * p->E > 0x7fffffffLL) return invalid("too many query rows");
  return MA_B200_OK;
}

int launched(cudaError_t ce, const char* what) {
  if (ce != cudaSuccess) return fail_with(MA_B200_CUDA_ERROR, std::string(what) + ": " + cudaGetErrorString(ce));
  return MA_B200_OK;
}

int attend(const ma_b200_attend* p, void* workspace, size_t workspace_bytes, void* stream, bool wait_expiry) {
  int rc = check_attend_shape(p);
  if (rc != MA_B200_OK) return rc;
  if (p->window < 0 || (p->window > 0 && !p->causal)) return invalid("window must not be negative, and needs causal");
  if (!isfinite(p->scale) || !(p->softcap == 0.0f || (p->softcap >= 1e-20f && p->softcap <= 1e30f)))
    return invalid("scale must be finite, softcap 0 (none) or from 1e-20 to 1e30");
  ma::AttendArgs a{};
  if ((rc = check_cache(p->cache, p->sequences, p->E, p->H, p->N, p->dtype, &a.cache)) != MA_B200_OK) return rc;
  if ((rc = check_tensor(p->q, "q", 2, 16)) != MA_B200_OK || (rc = check_tensor(p->out, "out", 2, 16)) != MA_B200_OK) return rc;
  const long long most = longest(p->sequences, p->cache.page_size);
  const size_t need = ma::attend_workspace(p->E, p->N, p->H, p->cache.heads, p->cache.width, p->window, most);
  if (workspace == nullptr || reinterpret_cast<uintptr_t>(workspace) % 256 != 0) return invalid("workspace is NULL or not 256-byte aligned");
  if (workspace_bytes < need)
    return fail_with(MA_B200_WORKSPACE_TOO_SMALL, "workspace has " + std::to_string(workspace_bytes) + " bytes, need " + std::to_string(need));
  int dev = 0;
  (void)cudaGetDevice(&dev);
  int* const wait_status = ma::host_status_word(dev, 0);
  a.q = view(p->q); a.out = view(p->out);
  a.E = p->E; a.N = p->N; a.H = p->H; a.group = p->H / p->cache.heads;
  a.causal = p->causal != 0; a.window = p->window; a.scale = p->scale; a.softcap = p->softcap;
  return launched(ma::launch_attend(a, p->dtype, p->cache.width, workspace, most, wait_status, wait_expiry, reinterpret_cast<cudaStream_t>(stream)), "attention over the cache");
}

}  // namespace

extern "C" {

int ma_b200_rotary_apply(const ma_b200_rotation* p, void* stream) {
  if (p == nullptr) return invalid("problem is NULL");
  if (p->abi_version != MA_B200_ABI_VERSION) return invalid("abi_version mismatch: got " + std::to_string(p->abi_version));
  if (p->E <= 0 || p->N <= 0 || p->D <= 0 || p->H < 0 || p->Hk < 0 || p->H + p->Hk == 0) return invalid("E, N, D and the number of heads must be positive");
  if (p->dtype != MA_B200_F32 && p->dtype != MA_B200_BF16 && p->dtype != MA_B200_F16) return invalid("unknown dtype");
  const size_t size = p->dtype == MA_B200_F32 ? 4 : 2;
  int rc = MA_B200_OK;
  if (p->H > 0 && ((rc = check_tensor(p->q, "q", size, size)) != MA_B200_OK || (rc = check_tensor(p->q_out, "q_out", size, size)) != MA_B200_OK)) return rc;
  if (p->Hk > 0 && ((rc = check_tensor(p->k, "k", size, size)) != MA_B200_OK || (rc = check_tensor(p->k_out, "k_out", size, size)) != MA_B200_OK)) return rc;
  ma::RotaryArgs rotary;
  if (const char* why = ma::rotary_args(&p->rotary, p->D, &rotary)) return invalid(why);
  if (p->inverse) rotary.sign = -1.0f;
  if ((long long)p->E * p->N > 0x7fffffffLL || p->H + p->Hk > 65535 || p->D > 1 << 16) return invalid("too many tokens, heads or features");
  return launched(ma::launch_rotary(p, rotary, reinterpret_cast<cudaStream_t>(stream)), "rotary");
}

int ma_b200_cache_append(const ma_b200_append* p, void* stream) {
  if (p == nullptr) return invalid("problem is NULL");
  if (p->abi_version != MA_B200_ABI_VERSION) return invalid("abi_version mismatch: got " + std::to_string(p->abi_version));
  if (longest(p->sequences, p->cache.page_size) + p->N + ma::kScaleBlock > 0x7fffffffLL) return invalid("positions would pass 2^31");
  ma::AppendArgs a{};
  int rc = check_cache(p->cache, p->sequences, p->E, p->H, p->N, p->dtype, &a.cache);
  if (rc != MA_B200_OK) return rc;
  const size_t lane = 16;  // bytes that a lane reads at once
  if ((rc = check_tensor(p->k, "k", 2, lane)) != MA_B200_OK || (rc = check_tensor(p->v, "v", 2, lane)) != MA_B200_OK) return rc;
  if (p->H > 0 && ((rc = check_tensor(p->q, "q", 2, lane)) != MA_B200_OK || (rc = check_tensor(p->q_out, "q_out", 2, lane)) != MA_B200_OK)) return rc;
  if (const char* why = ma::rotary_args(p->rotary, p->cache.width, &a.rotary)) return invalid(why);
  if (p->rotary != nullptr && p->rotary->dim % 16 != 0) return fail_with(MA_B200_UNSUPPORTED, "rotary: dim must be a multiple of 16 here");
  if ((long long)p->E * ((p->N + 14) / 16 + 1) > 0x7fffffffLL || (long long)2 * p->cache.heads + p->H > (1 << 18)) return invalid("too many tokens or heads");
  a.k = view(p->k); a.v = view(p->v); a.q = view(p->q); a.q_out = view(p->q_out);
  a.E = p->E; a.N = p->N; a.H = p->H;
  return launched(ma::launch_append(a, p->dtype, p->cache.width, reinterpret_cast<cudaStream_t>(stream)), "append");
}

size_t ma_b200_cache_attend_workspace_bytes(const ma_b200_attend* p) {
  if (check_attend_shape(p) != MA_B200_OK) return 0;
  return ma::attend_workspace(p->E, p->N, p->H, p->cache.heads, p->cache.width, p->window, longest(p->sequences, p->cache.page_size));
}

int ma_b200_cache_attend(const ma_b200_attend* p, void* workspace, size_t workspace_bytes, void* stream) {
  return attend(p, workspace, workspace_bytes, stream, false);
}

int ma_b200_selftest_attend_wait_expiry(const ma_b200_attend* p, void* workspace, size_t workspace_bytes, void* stream) {
  if (p != nullptr && p->dtype != MA_B200_BF16) return fail_with(MA_B200_UNSUPPORTED, "the self-test is of bf16");
  return attend(p, workspace, workspace_bytes, stream, true);
}

int ma_b200_poll_cache_status(int device) {
  const int code = ma::fused_poll_status(device, 1);
  if (code == 0) return MA_B200_OK;
  return fail_with(MA_B200_DEVICE_BAD_SEQUENCE, "device " + std::to_string(device) + ": an earlier call met a " +
                                                    (code == ma::kBadPage ? "page outside the cache" : "length or count outside its range") +
                                                    "; what it concerns was left out");
}

}  // extern "C"
