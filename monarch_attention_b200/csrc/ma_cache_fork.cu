// Sequences that go on from others, end, or get room: the page table, the pages' counts of uses, and the copies of half-filled pages.
//
// Row e takes what row source[e] held: its full pages are shared (a use more each), the rest belongs to one row, the keeper: the row itself where it goes on from
// itself, else the first that goes on from it.  The keeper keeps the pages behind the full ones, as far as no other row has them too; others get a page of
// their own and, where tokens are in it, a copy.  Pages for length + room tokens are given out, the lowest free ones in the order of rows and places: whole
// numbers, so that the same call has the same result whatever the order of the atomics.
//
// The bookkeeping is one cluster of CTAs with its barriers between the steps (a launch for each would cost more than the steps):
//   1  a row's pages: those in front of its first entry that names none; a minimum over the entries
//   2  keepers, lengths, how many pages a row keeps and how many it wants: a warp a row
//   3  uses: one less for each page of the rows as they were, one more for each that a row keeps; kept entries of other rows into the workspace, since
//      all rows change at once; where a row's wanted pages stand among all: a prefix sum
//   4  free pages of each CTA's part of the pool
//   5  the free pages that are wanted, the lowest first, into a list; from there into the rows
// The pages' contents are copied by a second kernel, all layers at once, a warp taking the keys and values of 16 tokens of a head.  Pages that are read there are not given
// out in the same call.
// The first is bound by latency: some 15 reads one after another and six barriers.  Measured in a graph, the first alone / both: 4 rows of 33 pages, 12 layers 9.4 / 11.6 us,
// 128 rows of 17, 16 layers 14.2 / 36.2, 8 rows of 3752, 2 layers 16.4 / 18.7 (5 more with rows' numbers from global memory in each step and atomics for pages that stay).  Eight SMs do it whatever the
// table's size: 64 rows of 8192 entries, 524288 pages 68 (exchanged 89, shared anew by four 145).  The second by memory: 70 half pages of 16 layers, 8 heads of 128 features, 127 MB in 20.5 us, 6.2 TB/s.
#include <cooperative_groups.h>

#include "ma_cache.cuh"

namespace ma {
namespace {

constexpr int kThreads = 1024, kWarps = kThreads / 32, kMostCtas = 8;
constexpr int kCached = 1024;  // rows whose numbers each CTA keeps in shared memory

// Parts of the workspace, in ints.
struct ForkLayout {
  long long held, keeper, plan, first, staged, free_list, copies, total;
  __host__ __device__ ForkLayout(long long E, long long P, long long pages) {
    const long long rows = (E + 3) / 4 * 4;
    long long at = 8 + kMostCtas;  // [0] copies, [8 ..] free pages of each CTA's part
    held = at; at += rows;
    keeper = at; at += rows;
    plan = at; at += 4 * rows;     // length, entries kept, entries wanted in all, page that is copied (-1: none)
    first = at; at += rows;        // the number of a row's first new page
    copies = at; at += 4 * rows;   // from, to, tokens
    staged = at; at += E * P;
    free_list = at; at += pages;
    total = at;
  }
};

// Of a row: where it goes on from, pages that it held, that it keeps, that it ends with, and the number of its first new one.
struct Row {
  int source, held, kept, need, first;
};

__device__ __forceinline__ int page_in(const CacheArgs& c, int entry) { return entry >= 0 && entry < c.pages ? entry : -1; }

static_assert(kWarps == 32, "a lane has a warp's sum");
// The sum of x over the threads in front of this one, and (in *all) over all; every thread takes part.
__device__ __forceinline__ int sum_before(int x, int* scratch, int* all) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  int upto = x;
#pragma unroll
  for (int m = 1; m < 32; m <<= 1) {
    const int o = __shfl_up_sync(0xffffffffu, upto, m);
    if (lane >= m) upto += o;
  }
  __syncthreads();  // (the scratch of a call before this one has been read)
  if (lane == 31) scratch[w] = upto;
  __syncthreads();
  int warps = scratch[lane];
#pragma unroll
  for (int m = 1; m < 32; m <<= 1) {
    const int o = __shfl_up_sync(0xffffffffu, warps, m);
    if (lane >= m) warps += o;
  }
  *all = __shfl_sync(0xffffffffu, warps, 31);
  const int before = __shfl_sync(0xffffffffu, warps, max(w - 1, 0));
  return (w > 0 ? before : 0) + upto - x;
}

__global__ void __launch_bounds__(kThreads, 1) fork_kernel(const __grid_constant__ ForkArgs a) {
  __shared__ int scratch[kWarps];
  namespace cg = cooperative_groups;
  const cg::cluster_group cluster = cg::this_cluster();
  const CacheArgs& c = a.cache;
  const int E = a.E, P = c.table_pages, tid = threadIdx.x, lane = tid & 31, rank = blockIdx.x, ctas = gridDim.x;  // (one cluster is the grid)
  const int me = rank * kThreads + tid, all = ctas * kThreads, page_size = 1 << c.page_shift;
  const ForkLayout at(E, P, c.pages);
  int* const ws = a.workspace;
  int *const held = ws + at.held, *const keeper = ws + at.keeper, *const first = ws + at.first, *const staged = ws + at.staged, *const free_list = ws + at.free_list;
  int4 *const plan = reinterpret_cast<int4*>(ws + at.plan), *const copies = reinterpret_cast<int4*>(ws + at.copies);
  const unsigned entries = (unsigned)E * (unsigned)P;  // (under 2^31)
  auto source_of = [&](int e) { const int s = a.source != nullptr ? a.source[e] : e; return s >= -1 && s < E ? s : e; };
  grid_wait();
  for (int e = me; e < E; e += all) {
    held[e] = P;
    keeper[e] = 0x7fffffff;
    if (a.source != nullptr && (a.source[e] < -1 || a.source[e] >= E)) report(c.status, kBadSource);
  }
  if (me == 0) ws[0] = 0;
  cluster.sync();

  // --- 1
  constexpr int kInFlight = 4;
  for (unsigned i0 = me; i0 < entries; i0 += all * kInFlight) {
    int now[kInFlight], before[kInFlight], e[kInFlight], j[kInFlight];
#pragma unroll
    for (int k = 0; k < kInFlight; ++k) {
      const unsigned i = i0 + k * all;
      e[k] = -1;
      if (i >= entries) continue;
      e[k] = (int)(i / (unsigned)P);
      j[k] = (int)(i - (unsigned)e[k] * P);
      const int* row = a.table + e[k] * c.table_se;
      now[k] = row[j[k]];
      before[k] = j[k] > 0 ? row[j[k] - 1] : 0;
    }
#pragma unroll
    for (int k = 0; k < kInFlight; ++k)  // (only where a run of pages ends: the rest of a row says the same)
      if (e[k] >= 0 && page_in(c, now[k]) < 0 && page_in(c, before[k]) >= 0) atomicMin(&held[e[k]], j[k]);
  }
  for (int e = me; e < E; e += all) {
    const int s = source_of(e);
    if (s >= 0) atomicMin(&keeper[s], s == e ? -1 : e);
  }
  cluster.sync();

  // --- 2
  for (int e = me >> 5; e < E; e += all >> 5) {
    const int s = source_of(e);
    int length = 0, kept = 0, behind = 0;
    if (s >= 0) {
      const int l = a.lengths[s], has = __ldcg(held + s);
      length = (int)min((long long)max(l, 0), (long long)has << c.page_shift);
      if (l != length && lane == 0) report(c.status, kBadLength);
      kept = length >> c.page_shift;
      behind = __ldcg(keeper + s) == (s == e ? -1 : e) ? has : 0;
    }
    const int room = a.room != nullptr ? a.room[e] : a.room_all;
    long long wants = ((long long)length + max(room, 0) + page_size - 1) >> c.page_shift;
    if ((room < 0 || wants > P) && lane == 0) report(c.status, kBadLength);
    const int full = kept, need = (int)min(wants, (long long)P);
    // pages behind the full ones that no other row has
    for (int j0 = full, end = min(behind, need); j0 < end; j0 += 32) {
      const int j = j0 + lane, page = j < end ? a.table[s * c.table_se + j] : -1;
      const unsigned mine = __ballot_sync(0xffffffffu, page >= 0 && a.uses[page] == 1);
      const int run = mine == 0xffffffffu ? 32 : __ffs(~mine) - 1;
      kept += run;
      if (run < 32) break;
    }
    if (lane == 0) {
      const bool copied = (length & (page_size - 1)) != 0 && kept == full;
      plan[e] = make_int4(length, kept, need, copied ? a.table[s * c.table_se + full] : -1);
    }
  }
  cluster.sync();

  // --- 3
  // What the last steps need of a row, in each CTA's shared memory (of the first kCached): reads that depend on one another are what these steps consist of.
  __shared__ Row rows[kCached];
  int wanted = 0;
  for (int e0 = 0; e0 < E; e0 += kThreads) {
    const int e = e0 + tid;
    int wants = 0, part;
    Row r{};
    if (e < E) {
      const int4 p = __ldcg(plan + e);
      r = Row{source_of(e), __ldcg(held + e), p.y, p.z, 0};
      wants = max(p.z - p.y, 0);
    }
    r.first = wanted + sum_before(wants, scratch, &part);
    if (e < kCached && e < E) rows[e] = r;
    else if (e < E) first[e] = r.first;  // (each CTA the same)
    wanted += part;
  }
  __syncthreads();
  auto row = [&](int e) {
    if (e < kCached) return rows[e];
    const int4 p = __ldcg(plan + e);
    return Row{source_of(e), __ldcg(held + e), p.y, p.z, first[e]};
  };
  for (unsigned i0 = me; i0 < entries; i0 += all * kInFlight) {
    int mine[kInFlight], theirs[kInFlight];  // pages given up and taken, -1: none
#pragma unroll
    for (int k = 0; k < kInFlight; ++k) {
      const unsigned i = i0 + k * all;
      mine[k] = theirs[k] = -1;
      if (i >= entries) continue;
      const int e = (int)(i / (unsigned)P), j = (int)(i - (unsigned)e * P);
      const Row r = row(e);
      const bool keeps = j < r.kept;
      if (r.source == e && keeps) continue;
      if (j < r.held) mine[k] = a.table[e * c.table_se + j];
      if (keeps) theirs[k] = a.table[r.source * c.table_se + j];
    }
#pragma unroll
    for (int k = 0; k < kInFlight; ++k) {
      if (theirs[k] >= 0) staged[i0 + k * all] = theirs[k];
      if (mine[k] == theirs[k]) continue;  // (as where a row goes on again from one that it shares its pages with)
      if (mine[k] >= 0) atomicSub(&a.uses[mine[k]], 1);
      if (theirs[k] >= 0) atomicAdd(&a.uses[theirs[k]], 1);
    }
  }
  for (int e = me; e < E; e += all) {  // (a page that is copied is not given out)
    const int page = __ldcg(&plan[e].w), end = row(e).held;
    if (page >= 0) atomicAdd(&a.uses[page], 1);
    if (end < P && a.table[e * c.table_se + end] >= 0) report(c.status, kBadPage);  // (what is behind a row's end may be anything)
  }
  cluster.sync();

  // --- 4: a CTA's part of the pool, of which a thread has a run
  const int run = (int)(((long long)c.pages + all - 1) / all);
  const long long page0 = (long long)me * run, page1 = min(page0 + run, (long long)c.pages);
  int part, mine = 0, free_pages = 0;
  unsigned unused = 0;  // of the run's first 32, a bit each
  if (wanted > 0) {
    int n = 0;
#pragma unroll 4
    for (long long p = page0; p < page1; ++p) {
      const bool is = __ldcg(a.uses + p) == 0;
      n += is;
      if (is && p - page0 < 32) unused |= 1u << (p - page0);
    }
    mine = sum_before(n, scratch, &part);
    if (tid == 0) ws[8 + rank] = part;
  }
  cluster.sync();

  // --- 5
  if (wanted > 0) {
#pragma unroll
    for (int i = 0; i < kMostCtas; ++i) {
      const int n = i < ctas ? __ldcg(ws + 8 + i) : 0;
      if (i < rank) mine += n;
      free_pages += n;
    }
    if (wanted > free_pages && me == 0) report(c.status, kNoPage);
    auto give = [&](long long p) {
      if (mine >= wanted) return;
      free_list[mine++] = (int)p;
      a.uses[p] = 1;
    };
    for (unsigned bits = unused; bits != 0; bits &= bits - 1) give(page0 + __ffs(bits) - 1);
    for (long long p = page0 + 32; p < page1 && mine < wanted; ++p)
      if (__ldcg(a.uses + p) == 0) give(p);
  }
  cluster.sync();
  for (unsigned i0 = me; i0 < entries; i0 += all * kInFlight) {
    int page[kInFlight];
    int* at_entry[kInFlight];
#pragma unroll
    for (int k = 0; k < kInFlight; ++k) {
      const unsigned i = i0 + k * all;
      at_entry[k] = nullptr;
      page[k] = -1;
      if (i >= entries) continue;
      const int e = (int)(i / (unsigned)P), j = (int)(i - (unsigned)e * P);
      const Row r = row(e);
      if (j < r.kept) {
        if (r.source == e) continue;
        page[k] = staged[i];
      } else if (j < r.need) {
        const int n = r.first + j - r.kept;
        if (n < free_pages) page[k] = __ldcg(free_list + n);
      }
      at_entry[k] = a.table + e * c.table_se + j;
    }
#pragma unroll
    for (int k = 0; k < kInFlight; ++k)
      if (at_entry[k] != nullptr) *at_entry[k] = page[k];
  }
  for (int e = me; e < E; e += all) {
    const int4 p = __ldcg(plan + e);
    const int new_page = row(e).first;
    // (where the pages did not suffice, a row ends with the last that it has)
    const int got = min(max(free_pages - new_page, 0), max(p.z - p.y, 0));
    a.lengths[e] = (int)min((long long)p.x, (long long)(p.y + got) << c.page_shift);
    if (p.w < 0) continue;
    atomicSub(&a.uses[p.w], 1);
    if (got > 0) copies[atomicAdd(ws, 1)] = make_int4(p.w, __ldcg(free_list + new_page), p.x & (page_size - 1), 0);
  }
}

template <int D>
__global__ void __launch_bounds__(256) copy_kernel(const __grid_constant__ ForkArgs a) {
  constexpr int kLanes = D / 16, kRows = 32 / kLanes, kPasses = kScaleBlock / kRows;
  const CacheArgs& c = a.cache;
  const int lane = threadIdx.x & 31, lane_row = lane / kLanes, piece = lane % kLanes;
  grid_wait();
  const ForkLayout at(a.E, c.table_pages, c.pages);
  const int copies = a.workspace[0], blocks = 1 << c.page_shift >> 4;
  const int4* const list = reinterpret_cast<const int4*>(a.workspace + at.copies);
  const long long tasks = (long long)copies * a.layers * c.heads * blocks;
  for (long long task = blockIdx.x * 8 + (threadIdx.x >> 5); task < tasks; task += gridDim.x * 8) {
    const int block = (int)(task & (blocks - 1));
    const long long unit = task >> (c.page_shift - 4);
    const int head = (int)(unit % c.heads), layer = (int)(unit / c.heads % a.layers);
    const int4 copy = list[unit / c.heads / a.layers];
    if (block * kScaleBlock >= copy.z) continue;
    const LayerPointers& l = a.layer[layer];
    const long long from = copy.x, to = copy.y, row = block * kScaleBlock + lane_row;
    const uint8_t* const k = l.k + from * c.k_sp + head * c.k_sh + row * c.k_st + piece * 16;
    const uint8_t* const v = l.v + from * c.v_sp + head * c.v_sh + row * c.v_st + piece * 16;
    uint4 x[2][kPasses];
#pragma unroll
    for (int p = 0; p < kPasses; ++p) {
      x[0][p] = *reinterpret_cast<const uint4*>(k + p * kRows * c.k_st);
      x[1][p] = *reinterpret_cast<const uint4*>(v + p * kRows * c.v_st);
    }
    float scale = 0.0f;
    if (lane < 2) scale = (lane ? l.v_scale + from * c.vs_sp + head * c.vs_sh : l.k_scale + from * c.ks_sp + head * c.ks_sh)[block];
#pragma unroll
    for (int p = 0; p < kPasses; ++p) {
      *reinterpret_cast<uint4*>(l.k + to * c.k_sp + head * c.k_sh + (row + p * kRows) * c.k_st + piece * 16) = x[0][p];
      *reinterpret_cast<uint4*>(l.v + to * c.v_sp + head * c.v_sh + (row + p * kRows) * c.v_st + piece * 16) = x[1][p];
    }
    if (lane < 2) (lane ? l.v_scale + to * c.vs_sp + head * c.vs_sh : l.k_scale + to * c.ks_sp + head * c.ks_sh)[block] = scale;
  }
}

}  // namespace

size_t fork_workspace(int E, int table_pages, int pages) { return (size_t)ForkLayout(E, table_pages, pages).total * sizeof(int); }

cudaError_t launch_fork_copies(const ForkArgs& a, int width, cudaStream_t stream) {
  void* args[] = {(void*)&a};
  // a CTA for 8 blocks of 16 tokens of a head, up to eight of an SM
  const long long most = (long long)a.E * a.layers * a.cache.heads << (a.cache.page_shift - 4), grid = (most + 7) / 8, places = 8 * sm_count();
  return launch_kernel(width == 128 ? (const void*)copy_kernel<128> : (const void*)copy_kernel<64>, dim3((unsigned)(grid < places ? grid : places)), dim3(256), args, 0, stream);
}

cudaError_t launch_fork(const ForkArgs& a, int width, cudaStream_t stream) {
  void* args[] = {(void*)&a};
  // Few entries and pages: one CTA, whose barriers are its own.  us of the call in a graph, one / eight, each row going on from itself: 4 rows of 36 entries and 200 pages 7.0 / 9.8, 16 x 100 and
  // 1600 8.6 / 10.4, 32 x 64 and 2000 8.7 / 10.4, 64 x 40 and 2600 11.0 / 11.2, 128 x 17 and 2183 14.0 / 11.3, 32 x 128 and 4000 10.3 / 10.5, 8 x 1000 and 8000 13.5 / 10.1, 256 x 32 and 8000 26 / 11.5.
  const long long work = (long long)a.E * a.cache.table_pages + a.cache.pages;
  const int ctas = work <= 4 * kThreads ? 1 : kMostCtas;
  const cudaError_t err = launch_kernel((const void*)fork_kernel, dim3(ctas), dim3(kThreads), args, 0, stream, ctas);
  if (err != cudaSuccess) return err;
  return launch_fork_copies(a, width, stream);
}

}  // namespace ma
