// What a step needs to know of its requests, made on the device: states and pages that follow the beams of a search, and the description of a step from the requests' lengths.
// The reference keeps block tables on the host and hands none to its kernels (runtime/blocks.py:31-111); a search's parents are known on the device first.
//
// Reordering.  Beam i of a search goes on from beam parents[i].  A parent's first child keeps the parent's state slot and the page the parent is writing; every
// other child takes those of a beam that has no child, in order (there are as many), and only these are copied: 2 x (rows of state + written entries of a page) bytes are
// read and written, which is what bounds it.  Whole pages are never written again, so a child's table names its parent's.  What is copied to had no child and what is copied from keeps
// its place: no row is both, and the copies need no order among themselves.  Every block works out who takes whose place for itself (a warp a search, votes); the copying is dealt over the blocks in
// units.  Measured, us (what is copied, read and written once, at the measured copy rate): 16 rows of 16.8 MB of state 86 (82); a page of two beams in 24 layers 4.9 (0.04); pages of 32 beams in 28 layers of a 7B
// model, 23.8 MB in pieces of 3 KB, 18 (7.3): a unit's look-ups of slots and pages are two dependent loads before its first copy.
//
// Step tables.  Request s brings q_lens[s] tokens behind have[s]; starts are sums over the requests before it, which every block that works for s adds up itself
// (a thousand lengths are four a thread; a launch of its own for them would cost more).  Measured, us: 8 decoded tokens 2.7, 48 requests with 4,099 tokens in two groups and new pages 6.6, 512 requests
// with 32,768 tokens and tables of 2,100 columns 7.0 (1.0 for its bytes): the sums and the look-ups, one after the other, bound it.
//
// Attention kernels read lengths and block tables before they wait for the kernel before, so the launch behind either operator is a plain one (`launch_kernel_describing`).
#include "common.cuh"

namespace sllm {

constexpr int REORDER_THREADS = 256, REORDER_STATES = 64, REORDER_PAGED = 8, REORDER_ROWS = 2048;

struct StateTable {
  unsigned char* base;
  long long row_bytes;
  int slots, width;            // width: bytes a lane moves at a time (16, 8, 4, 2 or 1)
};
struct PagedTable {
  unsigned char* base;
  const int* table;
  int* new_table;
  long long entry_bytes;       // of one head: head size x element size
  int outer, heads, pages, page_size, stride, columns, width;      // outer: runs x (keys, values)
};
struct ReorderPlan {
  StateTable states[REORDER_STATES];
  PagedTable paged[REORDER_PAGED];
  int num_states, num_paged;
  long long unit;              // bytes a block copies at a time
};

constexpr int REORDER_LOADS = 4;                // a thread's copies in flight

// `n` pieces of V, the block's threads side by side
template <typename V>
__device__ __forceinline__ void copy_run(unsigned char* dst, const unsigned char* src, int n) {
  V* d = reinterpret_cast<V*>(dst);
  const V* s = reinterpret_cast<const V*>(src);
  for (int i = threadIdx.x; i < n; i += REORDER_LOADS * REORDER_THREADS) {
    V v[REORDER_LOADS];
#pragma unroll
    for (int u = 0; u < REORDER_LOADS; ++u)
      if (i + u * REORDER_THREADS < n) v[u] = s[i + u * REORDER_THREADS];
#pragma unroll
    for (int u = 0; u < REORDER_LOADS; ++u)
      if (i + u * REORDER_THREADS < n) d[i + u * REORDER_THREADS] = v[u];
  }
}

// Pieces [from, from + n) of the written entries of a page: `per` pieces of every head of every outer copy, one after the other.
template <typename V>
__device__ __forceinline__ void copy_page(const PagedTable& t, int dst_page, int src_page, unsigned per, unsigned long long from, int n) {
  const size_t head_bytes = (size_t)t.page_size * t.entry_bytes, page_bytes = head_bytes * t.heads, outer_bytes = page_bytes * t.pages;
  // the unit's first segment once, then 32-bit steps from it
  const unsigned seg0 = (unsigned)(from / per), at0 = (unsigned)(from - (unsigned long long)seg0 * per);
  const long long move = ((long long)dst_page - src_page) * (long long)page_bytes;
  unsigned char* base = t.base + (size_t)src_page * page_bytes;
  for (int i0 = threadIdx.x; i0 < n; i0 += REORDER_LOADS * REORDER_THREADS) {
    V v[REORDER_LOADS];
    unsigned char* p[REORDER_LOADS];
#pragma unroll
    for (int u = 0; u < REORDER_LOADS; ++u) {
      const int i = i0 + u * REORDER_THREADS;
      p[u] = nullptr;
      if (i < n) {
        const unsigned k = at0 + (unsigned)i, seg = seg0 + k / per, at = k % per, o = seg / (unsigned)t.heads, h = seg % (unsigned)t.heads;
        p[u] = base + (size_t)o * outer_bytes + (size_t)h * head_bytes + (size_t)at * sizeof(V);
        v[u] = *reinterpret_cast<const V*>(p[u]);
      }
    }
#pragma unroll
    for (int u = 0; u < REORDER_LOADS; ++u)
      if (p[u]) *reinterpret_cast<V*>(p[u] + move) = v[u];
  }
}

__global__ void __launch_bounds__(REORDER_THREADS, 4) beam_reorder_kernel(const int* parents, const int* slots, const int* lens, int len_step, int* new_slots, int G, int B, const ReorderPlan plan) {
  extern __shared__ int reorder_smem[];
  const int S = G * B;
  int* source = reorder_smem;                   // [S] the row a row goes on from
  int* takes = source + S;                      // [S] the row whose slot and page it has then
  int* first_unit = takes + S;                  // [S + 1] units of copying before the row's
  __shared__ int spare[REORDER_THREADS / 32][32];
  __shared__ int warp_units[REORDER_THREADS / 32 + 1];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  pdl_wait();
  int state_units = 0;
  for (int k = 0; k < plan.num_states; ++k) state_units += (int)((plan.states[k].row_bytes + plan.unit - 1) / plan.unit);
  // a warp a search, a lane a beam
  for (int g = warp; g < G; g += REORDER_THREADS / 32) {
    const bool in = lane < B;
    int p = in ? parents[g * B + lane] : -1;
    if (p < 0 || p >= B) p = -1;
    const unsigned same = __match_any_sync(0xffffffffu, p);
    const bool keeps = p >= 0 && __ffs(same) - 1 == lane;
    const unsigned parent_of = __reduce_or_sync(0xffffffffu, p >= 0 ? 1u << p : 0u);
    const unsigned childless = ~parent_of & (B == 32 ? 0xffffffffu : (1u << B) - 1);
    const unsigned below = (1u << lane) - 1;
    if (in && (childless >> lane & 1)) spare[warp][__popc(childless & below)] = lane;
    const unsigned takers = __ballot_sync(0xffffffffu, in && !keeps);
    __syncwarp();
    if (in) {
      const int t = keeps ? p : spare[warp][__popc(takers & below)];
      const bool copies = !keeps && p >= 0;
      source[g * B + lane] = g * B + (p >= 0 ? p : t);
      takes[g * B + lane] = g * B + t;
      int units = 0;
      if (copies) {
        units = state_units;
        for (int k = 0; k < plan.num_paged; ++k) {
          const PagedTable& t = plan.paged[k];
          const long long written = max(lens[g * len_step], 0) / t.stride % t.page_size;
          if (written > 0) units += (int)((written * t.entry_bytes * t.heads * t.outer + plan.unit - 1) / plan.unit);
        }
      }
      first_unit[g * B + lane] = units;
    }
    __syncwarp();
  }
  __syncthreads();
  // units before each row
  {
    const int per = (S + REORDER_THREADS - 1) / REORDER_THREADS, r0 = threadIdx.x * per, r1 = min(r0 + per, S);
    int sum = 0;
    for (int r = r0; r < r1; ++r) sum += first_unit[r];
    int incl = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    if (lane == 31) warp_units[warp] = incl;
    __syncthreads();
    int before = incl - sum;
    for (int w = 0; w < warp; ++w) before += warp_units[w];
    for (int r = r0; r < r1; ++r) {
      const int u = first_unit[r];
      first_unit[r] = before;
      before += u;
    }
    if (threadIdx.x == REORDER_THREADS - 1) first_unit[S] = before;
  }
  __syncthreads();
  // slots
  if (new_slots != nullptr && blockIdx.x == 0)
    for (int r = threadIdx.x; r < S; r += REORDER_THREADS) new_slots[r] = slots[takes[r]];
  // the copies
  const int all = first_unit[S];
  for (int u = blockIdx.x; u < all; u += gridDim.x) {
    int lo = 0, hi = S;                         // the last row whose units begin at or before u
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (first_unit[mid] <= u) lo = mid;
      else hi = mid;
    }
    const int r = lo;
    int at = u - first_unit[r];
    if (at < state_units) {
      const int dst = slots[takes[r]], src = slots[source[r]];
      for (int k = 0; k < plan.num_states; ++k) {
        const StateTable& t = plan.states[k];
        const int n = (int)((t.row_bytes + plan.unit - 1) / plan.unit);
        if (at >= n) {
          at -= n;
          continue;
        }
        if (dst >= 0 && dst < t.slots && src >= 0 && src < t.slots) {
          const long long b0 = at * plan.unit;
          const int bytes = (int)min(plan.unit, t.row_bytes - b0);
          unsigned char* d = t.base + (size_t)dst * t.row_bytes + b0;
          const unsigned char* s = t.base + (size_t)src * t.row_bytes + b0;
          if (t.width == 16) copy_run<uint4>(d, s, bytes / 16);
          else if (t.width == 4) copy_run<uint32_t>(d, s, bytes / 4);
          else copy_run<unsigned char>(d, s, bytes);
        }
        break;
      }
      continue;
    }
    at -= state_units;
    for (int k = 0; k < plan.num_paged; ++k) {
      const PagedTable& t = plan.paged[k];
      const int entries = max(lens[r / B * len_step], 0) / t.stride, written = entries % t.page_size, column = entries / t.page_size;
      if (written == 0) continue;
      const long long bytes = (long long)written * t.entry_bytes * t.heads * t.outer;
      const int n = (int)((bytes + plan.unit - 1) / plan.unit);
      if (at >= n) {
        at -= n;
        continue;
      }
      if (column < t.columns) {
        const int src = t.table[(size_t)source[r] * t.columns + column], dst = t.table[(size_t)takes[r] * t.columns + column];
        if (src >= 0 && src < t.pages && dst >= 0 && dst < t.pages) {
          const long long b0 = at * plan.unit;
          const int n_bytes = (int)min(plan.unit, bytes - b0);
          const unsigned per = (unsigned)(written * t.entry_bytes / t.width);
          if (t.width == 16) copy_page<uint4>(t, dst, src, per, b0 / 16, n_bytes / 16);
          else if (t.width == 4) copy_page<uint32_t>(t, dst, src, per, b0 / 4, n_bytes / 4);
          else copy_page<unsigned short>(t, dst, src, per, b0 / 2, n_bytes / 2);
        }
      }
      break;
    }
  }
  // the tables: rows over the blocks
  for (int k = 0; k < plan.num_paged; ++k) {
    const PagedTable& t = plan.paged[k];
    for (int r = blockIdx.x; r < S; r += gridDim.x) {
      const int entries = max(lens[r / B * len_step], 0) / t.stride, at = entries / t.page_size;
      const bool begun = entries % t.page_size > 0;
      const int *own = t.table + (size_t)r * t.columns, *from = t.table + (size_t)source[r] * t.columns, *taken = t.table + (size_t)takes[r] * t.columns;
      for (int c = threadIdx.x; c < t.columns; c += REORDER_THREADS) t.new_table[(size_t)r * t.columns + c] = c < at ? from[c] : (c == at && begun) ? taken[c] : own[c];
    }
  }
  pdl_launch_dependents();
}

// ---- a step's description ---------------------------------------------------------------------------------------------------

constexpr int TABLES_THREADS = 256, TABLES_GROUPS = 8;

struct TableGroup {
  int* pages;                  // [rows, columns] every live request's pages
  const int* free;             // pages that requests take as they grow, in order; or null
  int* block_table;            // [S, out_columns]
  int* slot_mapping;           // [T]
  int columns, out_columns, free_count, stride;
};
struct TableGroups {
  TableGroup g[TABLES_GROUPS];
  int n;
};

// lengths within what sums of two and their pages keep in 32 bits
__device__ __forceinline__ int length_of(int n) { return min(max(n, 0), (1 << 30) - 1); }
__device__ __forceinline__ int pages_of(int entries, int page_size) { return entries / page_size + (entries % page_size > 0); }

// blockIdx.x: the request; the blocks of blockIdx.y share its tokens and its table's columns
__global__ void __launch_bounds__(TABLES_THREADS) step_tables_kernel(const int* q_lens, const int* have_lens, const int* rows, int S, int N, int T, int page_size, int* q_start, int* ctx_len, int* positions,
                                                                     int* seq_of_token, const TableGroups groups) {
  __shared__ int sums[TABLES_GROUPS][TABLES_THREADS / 32];
  __shared__ long long token_sums[TABLES_THREADS / 32];
  pdl_launch_dependents();
  pdl_wait();
  const int s = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  // tokens, and new pages of each group, of the requests before this one
  int before[TABLES_GROUPS] = {};
  long long tokens = 0;
  for (int r = threadIdx.x; r < s; r += TABLES_THREADS) {
    const int q = length_of(q_lens[r]), have = length_of(have_lens[r]);
    tokens += q;
#pragma unroll
    for (int k = 0; k < TABLES_GROUPS; ++k)
      if (k < groups.n && groups.g[k].free != nullptr) before[k] += pages_of((have + q) / groups.g[k].stride, page_size) - pages_of(have / groups.g[k].stride, page_size);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) tokens += __shfl_xor_sync(0xffffffffu, tokens, o);
  if (lane == 0) token_sums[warp] = tokens;
#pragma unroll
  for (int k = 0; k < TABLES_GROUPS; ++k) {
    if (k >= groups.n || groups.g[k].free == nullptr) continue;
    int v = before[k];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (lane == 0) sums[k][warp] = v;
  }
  __syncthreads();
  auto total = [&](int k) {
    int v = 0;
#pragma unroll
    for (int w = 0; w < TABLES_THREADS / 32; ++w) v += sums[k][w];
    return v;
  };
  tokens = 0;
#pragma unroll
  for (int w = 0; w < TABLES_THREADS / 32; ++w) tokens += token_sums[w];
  // (tokens beyond T are left out)
  const int start = (int)min(tokens, (long long)T), q = min(length_of(q_lens[s]), T - start), have = length_of(have_lens[s]), ctx = have + length_of(q_lens[s]);
  const int step = gridDim.y * TABLES_THREADS, first = blockIdx.y * TABLES_THREADS + threadIdx.x;
  if (first == 0) {
    q_start[s] = start;
    ctx_len[s] = ctx;
    if (s == S - 1) q_start[S] = start + q;
  }
  for (int i = first; i < q; i += step) {
    positions[start + i] = have + i;
    seq_of_token[start + i] = s;
  }
  if (s == S - 1)                                 // rows behind the last token
    for (int t = start + q + first; t < T; t += step) {
      positions[t] = 0;
      seq_of_token[t] = 0;
    }
  const int row = rows != nullptr ? rows[s] : s;
  const bool known = row >= 0 && row < N;
  for (int k = 0; k < groups.n; ++k) {
    const TableGroup& g = groups.g[k];
    const int had = pages_of(have / g.stride, page_size), needs = pages_of(ctx / g.stride, page_size);
    const int fresh = g.free != nullptr ? total(k) : 0;
    int* mine = g.pages + (size_t)(known ? row : 0) * g.columns;
    // the page of a column; new ones from the list, -1 where there is none
    auto page = [&](int c) {
      if (!known || c >= g.columns) return -1;       // (c >= 0: lengths are)
      if (g.free == nullptr || c < had) return mine[c];
      const int f = fresh + (c - had);
      return f >= 0 && f < g.free_count ? g.free[f] : -1;
    };
    for (int c = first; c < g.out_columns; c += step) g.block_table[(size_t)s * g.out_columns + c] = c < needs ? page(c) : -1;
    for (int i = first; i < q; i += step) {
      const int p = have + i;
      int slot = -1;
      if (g.stride == 1 || (p + 1) % g.stride == 0) {
        const int entry = g.stride == 1 ? p : (p + 1) / g.stride - 1;
        const int id = page(entry / page_size);
        if (id >= 0) slot = id * page_size + entry % page_size;
      }
      g.slot_mapping[start + i] = slot;
    }
    if (s == S - 1)
      for (int t = start + q + first; t < T; t += step) g.slot_mapping[t] = -1;
    // (columns from `had` on, which no block reads)
    if (g.free != nullptr && known)
      for (int c = had + first; c < needs && c < g.columns; c += step) mine[c] = page(c);
  }
}

}  // namespace sllm

using namespace sllm;

// `states` (on the host): base, bytes a row, rows of each table; `paged` (on the host), 10 numbers each: base, table, new table, bytes of an entry of one head, outer, heads, pages,
// page size, stride, columns.  lens[g * len_step] tokens are in search g's caches.  new_slots may be null.
SLLM_EXPORT int sllm_beam_reorder(const int* parents, const int* slots, const int* lens, int len_step, int* new_slots, int G, int B, const long long* states, int num_states,
                                  const long long* paged, int num_paged, cudaStream_t stream) {
  SLLM_REQUIRE(G >= 0 && B >= 1 && B <= 32 && (long long)G * B <= REORDER_ROWS, "beam_reorder: %d searches of %d beams (at most 32, %d in all)", G, B, REORDER_ROWS);
  SLLM_REQUIRE(num_states >= 0 && num_states <= REORDER_STATES && num_paged >= 0 && num_paged <= REORDER_PAGED, "beam_reorder: %d states, %d paged caches", num_states, num_paged);
  if (G == 0) return SLLM_OK;
  ReorderPlan plan = {};
  plan.num_states = num_states;
  plan.num_paged = num_paged;
  long long bytes = 0, units = 0, cells = 0;     // at most, a row
  for (int k = 0; k < num_states; ++k) bytes += states[3 * k + 1];
  for (int k = 0; k < num_paged; ++k) bytes += paged[10 * k + 3] * paged[10 * k + 4] * paged[10 * k + 5] * paged[10 * k + 7];
  // A unit is a load a thread where little can be copied at all, so that it spreads over the SMs, else four.  (Pages of two beams over 24 layers, 0.1 MB: 4.9 us against 6.0 with four; of
  // twelve beams over 28 layers of a 7B model, 4.5 MB: 9.6 against 7.4.)
  plan.unit = bytes * G * B <= 16384ll * num_sms() ? REORDER_THREADS * 16 : REORDER_THREADS * 16 * REORDER_LOADS;
  for (int k = 0; k < num_states; ++k) {
    const long long* s = states + 3 * k;
    SLLM_REQUIRE(s[1] > 0 && s[1] < (1ll << 40) && s[2] > 0 && s[2] < (1ll << 31), "beam_reorder: state %d: %lld rows of %lld bytes", k, s[2], s[1]);
    const long long low = s[0] | s[1];
    plan.states[k] = StateTable{reinterpret_cast<unsigned char*>(s[0]), s[1], (int)s[2], low % 16 == 0 ? 16 : low % 4 == 0 ? 4 : 1};
    units += (s[1] + plan.unit - 1) / plan.unit;
  }
  for (int k = 0; k < num_paged; ++k) {
    const long long* p = paged + 10 * k;
    for (int i = 3; i < 10; ++i) SLLM_REQUIRE(p[i] > 0 && p[i] < (1ll << 31), "beam_reorder: paged cache %d: size %lld", k, p[i]);
    const long long low = p[0] | p[3];
    SLLM_REQUIRE(low % 2 == 0, "beam_reorder: paged cache %d: entries of %lld bytes", k, p[3]);
    plan.paged[k] = PagedTable{reinterpret_cast<unsigned char*>(p[0]), reinterpret_cast<const int*>(p[1]), reinterpret_cast<int*>(p[2]), p[3], (int)p[4], (int)p[5], (int)p[6],
                               (int)p[7], (int)p[8], (int)p[9], low % 16 == 0 ? 16 : low % 4 == 0 ? 4 : 2};
    const long long page = p[3] * p[4] * p[5] * p[7];
    SLLM_REQUIRE(page < (1ll << 40) && p[3] * p[7] < (1ll << 31), "beam_reorder: paged cache %d: a page of %lld bytes", k, page);
    units += (page + plan.unit - 1) / plan.unit;
    cells += p[9];
  }
  SLLM_REQUIRE(units * G * B < (1ll << 30), "beam_reorder: %lld bytes a beam", units * plan.unit);
  const long long work = units * G * B + (cells * G * B + 1023) / 1024, most = (long long)num_sms() * 4;
  const int grid = (int)(work < 1 ? 1 : work < most ? work : most);
  launch_kernel_describing(beam_reorder_kernel, grid, REORDER_THREADS, (size_t)(3 * G * B + 1) * sizeof(int), stream, parents, slots, lens, len_step, new_slots, G, B, plan);
  return launch_status("beam_reorder");
}

// `groups` (on the host), 8 numbers each: pages, free (or 0), block table, slot mapping, columns, columns of the block table, free pages, stride
SLLM_EXPORT int sllm_step_tables(const int* q_lens, const int* have, const int* rows, int S, int N, int T, int page_size, int* q_start, int* ctx_len, int* positions, int* seq_of_token,
                                 const long long* groups, int num_groups, cudaStream_t stream) {
  SLLM_REQUIRE(S >= 1 && N >= 1 && T >= 0 && page_size >= 1 && num_groups >= 0 && num_groups <= TABLES_GROUPS, "step_tables: %d requests, %d rows, %d tokens, pages of %d, %d groups", S, N, T, page_size,
               num_groups);
  TableGroups gs = {};
  gs.n = num_groups;
  long long most = T;
  for (int k = 0; k < num_groups; ++k) {
    const long long* p = groups + 8 * k;
    SLLM_REQUIRE(p[4] >= 0 && p[5] >= 0 && p[6] >= 0 && p[7] >= 1 && p[4] < (1ll << 31) && p[5] < (1ll << 31) && p[6] < (1ll << 31) && p[7] < (1ll << 31), "step_tables: group %d: %lld columns, %lld free pages, stride %lld", k, p[4],
                 p[6], p[7]);
    gs.g[k] = TableGroup{reinterpret_cast<int*>(p[0]), reinterpret_cast<const int*>(p[1]), reinterpret_cast<int*>(p[2]), reinterpret_cast<int*>(p[3]), (int)p[4], (int)p[5], (int)p[6], (int)p[7]};
    most = most > p[5] ? most : p[5];
  }
  long long y = (most + TABLES_THREADS - 1) / TABLES_THREADS, room = 8ll * num_sms() / S;
  y = y < room ? y : room;
  launch_kernel_describing(step_tables_kernel, dim3((unsigned)S, (unsigned)(y < 1 ? 1 : y)), TABLES_THREADS, 0, stream, q_lens, have, rows, S, N, T, page_size, q_start, ctx_len, positions, seq_of_token, gs);
  return launch_status("step_tables");
}
