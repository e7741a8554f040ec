// A step's tables from request lengths, on the device: where every row of a packed batch lies and which pages its sequence
// has, with pages for what does not fit a sequence's last page taken from a stack of free ones.
//
// State: lengths[slot] tokens a sequence holds, table[slot][i] its i-th page, free[0 ... n_free - 1] pages nobody holds.
// A slot holds ceil(length / page) pages.  Request i brings new[i] tokens of the sequence in slots[i]:
//   have_i = ceil(length / page), total_i = ceil((length + new) / page); the sums of new, total and total - have over the
//   requests before i are its first row, its first place in page_ids and how many free pages were taken before it;
//   the k-th page taken is free[n_free - 1 - k].
// sb_page_tables changes neither lengths nor n_free, so it can be called again; sb_page_advance records the step,
// sb_page_release gives sequences' pages back.
//
// All of it is latency: a launch, one gather of the lengths, three sums over the requests.  Every block works the sums out
// for itself (they fit its shared memory) and then fills its stretches of the rows and of the page list, so the blocks
// need not wait for one another.  Every block also finds the same status; where it is not 0 the tables describe no rows.
#include "common.cuh"

namespace {

constexpr int TB = 512;                          // threads
constexpr int CHUNK = 2 * TB;                    // rows or pages that a block fills in one go
constexpr int MAX_SEQS = 8192;                   // five numbers of every request in shared memory
constexpr int MAX_SLOTS = 1 << 18;               // a bit of every slot in shared memory
constexpr int MAX_COUNT = 1 << 21;               // rows, pages of a slot: sums of a tile of requests stay inside 32 bits

struct Sums {
  int rows, total, taken;
};
__device__ __forceinline__ Sums add(Sums a, Sums b) { return {a.rows + b.rows, a.total + b.total, a.taken + b.taken}; }
__device__ __forceinline__ Sums up(Sums v, int o) {
  return {__shfl_up_sync(0xffffffffu, v.rows, o), __shfl_up_sync(0xffffffffu, v.total, o), __shfl_up_sync(0xffffffffu, v.taken, o)};
}

// Pages of so many tokens, up to the largest int; none of fewer than 0.
__device__ __forceinline__ int pages_of(int tokens, int page_size) {
  return (int)(((unsigned)max(tokens, 0) + (unsigned)page_size - 1u) / (unsigned)page_size);
}

// The last i with at[i] <= v, of n + 1 ascending numbers with at[0] <= v < at[n].
__device__ __forceinline__ int owner_of(const int* at, int n, int v) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (at[mid] <= v) lo = mid;
    else hi = mid;
  }
  return lo;
}

__global__ void __launch_bounds__(TB) page_tables_kernel(const SbPageTables a) {
  extern __shared__ __align__(16) int smem[];
  __shared__ Sums warp_sums[TB / 32];
  __shared__ int found;
  int* row0 = smem;                              // [n + 1]
  int* off = row0 + a.n_seqs + 1;                // [n + 1]
  int* taken = off + a.n_seqs + 1;               // [n]
  int* length = taken + a.n_seqs;                // [n]
  int* slot_of = length + a.n_seqs;              // [n]
  unsigned* seen = reinterpret_cast<unsigned*>(slot_of + a.n_seqs);     // a bit of every slot
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  for (int i = tid; i < (a.n_slots + 31) / 32; i += TB) seen[i] = 0;
  if (tid == 0) found = 0;
  sb_pdl_wait();
  const int n_free = a.n_free[0];
  __syncthreads();
  long long rows = 0, pages = 0, needed = 0;     // of the tiles before this one
  for (int first = 0; first < a.n_seqs; first += TB) {
    const int i = first + tid;
    Sums v = {0, 0, 0};
    int bad = 0;
    if (i < a.n_seqs) {
      const int slot = a.slots[i];
      int fresh = a.fresh[i], held = 0;
      if (slot < 0 || slot >= a.n_slots || fresh < 0) {
        bad = SB_TABLES_BAD_REQUEST;
      } else if (atomicOr(&seen[slot >> 5], 1u << (slot & 31)) >> (slot & 31) & 1) {
        bad = SB_TABLES_BAD_REQUEST;             // the same sequence twice
      } else {
        held = a.lengths[slot];
        const long long len = (long long)held + fresh;
        if (held < 0 || fresh > a.max_new || len > a.max_len || len > (long long)a.width * a.page_size) bad = SB_TABLES_TOO_LONG;
      }
      if (bad) fresh = held = 0;
      const int have = pages_of(held, a.page_size), total = pages_of(held + fresh, a.page_size);
      v = {min(fresh, a.max_rows + 1), total, total - have};
      length[i] = held;
      slot_of[i] = bad ? 0 : slot;
    }
    if (bad) atomicOr(&found, bad);
    Sums mine = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const Sums w = up(mine, o);
      if (lane >= o) mine = add(mine, w);
    }
    if (lane == 31) warp_sums[warp] = mine;
    __syncthreads();
    Sums before = {0, 0, 0}, tile = {0, 0, 0};
#pragma unroll
    for (int w = 0; w < TB / 32; ++w) {
      if (w == warp) before = tile;
      tile = add(tile, warp_sums[w]);
    }
    if (i < a.n_seqs) {                          // sums past what fits are not used: the status says so below
      row0[i] = (int)rows + before.rows + mine.rows - v.rows;
      off[i] = (int)pages + before.total + mine.total - v.total;
      taken[i] = (int)needed + before.taken + mine.taken - v.taken;
    }
    rows += tile.rows; pages += tile.total; needed += tile.taken;
    __syncthreads();
  }
  int status = found;
  if (rows > a.max_rows) status |= SB_TABLES_ROWS;
  if (pages > a.max_pages) status |= SB_TABLES_PAGE_LIST;
  if (needed > 0 && (needed > n_free || n_free > a.n_pages)) status |= SB_TABLES_NO_PAGES;
  if (tid == 0) {
    row0[a.n_seqs] = status ? 0 : (int)rows;
    off[a.n_seqs] = status ? 0 : (int)pages;
  }
  __syncthreads();
  if (blockIdx.x == 0) {
    for (int i = tid; i <= a.n_seqs; i += TB) {
      a.seq_row0[i] = status ? 0 : row0[i];
      a.page_off[i] = status ? 0 : off[i];
      if (i < a.n_seqs) a.seq_pos0[i] = status ? 0 : length[i];
    }
    if (tid == 0) a.status[0] = status;
  }
  const int n_rows = row0[a.n_seqs], n_list = off[a.n_seqs];
  // page i of a request: held, or the next one of the stack
  auto page_of = [&](int s, int i) {
    const int have = pages_of(length[s], a.page_size);
    return i < have ? a.table[(size_t)slot_of[s] * a.width + i] : a.free[n_free - 1 - (taken[s] + i - have)];
  };
  const int row_chunks = (a.max_rows + CHUNK - 1) / CHUNK, chunks = row_chunks + (n_list + CHUNK - 1) / CHUNK;
  for (int c = blockIdx.x; c < chunks; c += gridDim.x) {
    if (c < row_chunks) {
      const int end = min((c + 1) * CHUNK, a.max_rows);
      for (int r = c * CHUNK + tid; r < end; r += TB) {
        int s = 0, pos = -1, where = -1;
        if (r < n_rows) {
          s = owner_of(row0, a.n_seqs, r);
          pos = length[s] + r - row0[s];
          const int nth = (int)((unsigned)pos / (unsigned)a.page_size);
          where = page_of(s, nth) * a.page_size + pos - nth * a.page_size;
        }
        a.row_seq[r] = s;
        a.row_pos[r] = pos;
        a.row_slot[r] = where;
      }
    } else {
      const int end = min((c - row_chunks + 1) * CHUNK, n_list);
      for (int k = (c - row_chunks) * CHUNK + tid; k < end; k += TB) {
        const int s = owner_of(off, a.n_seqs, k), i = k - off[s], page = page_of(s, i);
        a.page_ids[k] = page;
        if (i >= pages_of(length[s], a.page_size)) a.table[(size_t)slot_of[s] * a.width + i] = page;
      }
    }
  }
}

// Nothing: see sb_page_tables_settle.
__global__ void settle_kernel() {}

// One block: the sequences' new lengths and what is left of the stack.  A step whose tables have a status records nothing.
__global__ void __launch_bounds__(TB) page_advance_kernel(const int32_t* slots, const int32_t* fresh, int n_seqs, int32_t* lengths,
                                                          int n_slots, int32_t* n_free, int page_size, const int32_t* status) {
  __shared__ int taken;
  if (threadIdx.x == 0) taken = 0;
  sb_pdl_wait();
  if (status[0]) return;
  __syncthreads();
  int mine = 0;
  for (int i = threadIdx.x; i < n_seqs; i += TB) {
    const int slot = slots[i];
    if (slot < 0 || slot >= n_slots) continue;
    const int held = lengths[slot], len = held + fresh[i];
    mine += pages_of(len, page_size) - pages_of(held, page_size);
    lengths[slot] = len;
  }
  if (mine) atomicAdd(&taken, mine);             // whole numbers: the order does not matter
  __syncthreads();
  if (threadIdx.x == 0) n_free[0] -= taken;
}

// One block: the sequences' pages go back on the stack, a slot named twice where it is named first, one that does not exist not
// at all.
__global__ void __launch_bounds__(TB) page_release_kernel(const int32_t* slots, int n_seqs, int n_slots, int32_t* lengths, int32_t* table,
                                                          int width, int32_t* free, int n_pages, int32_t* n_free, int page_size) {
  extern __shared__ __align__(16) unsigned released[];          // a bit of every slot
  __shared__ int warp_sums[TB / 32], twice;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  for (int i = tid; i < (n_slots + 31) / 32; i += TB) released[i] = 0;
  if (tid == 0) twice = 0;
  sb_pdl_wait();
  __syncthreads();
  for (int i = tid; i < n_seqs; i += TB) {
    const int slot = slots[i];
    if (slot >= 0 && slot < n_slots && atomicOr(&released[slot >> 5], 1u << (slot & 31)) >> (slot & 31) & 1) twice = 1;
  }
  __syncthreads();
  int top = min(max(n_free[0], 0), n_pages);     // at most n_pages at all times, whatever lengths say
  for (int first = 0; first < n_seqs; first += TB) {
    const int i = first + tid;
    int slot = -1, count = 0;
    if (i < n_seqs) {
      slot = slots[i];
      if (slot < 0 || slot >= n_slots) slot = -1;
      if (twice)                                 // some slot is: who is named before looks for itself
        for (int j = 0; j < i; ++j)
          if (slots[j] == slot) slot = -1;
      if (slot >= 0) count = min(pages_of(lengths[slot], page_size), width);
    }
    int mine = count;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int w = __shfl_up_sync(0xffffffffu, mine, o);
      if (lane >= o) mine += w;
    }
    if (lane == 31) warp_sums[warp] = mine;
    __syncthreads();
    int before = 0, tile = 0;
#pragma unroll
    for (int w = 0; w < TB / 32; ++w) {
      if (w == warp) before = tile;
      tile += warp_sums[w];
    }
    // a warp takes its sequences one after another, so that a long one's pages move together
    const int at = (int)min((long long)top + before + mine - count, (long long)n_pages);
    for (int l = 0; l < 32; ++l) {
      const int s = __shfl_sync(0xffffffffu, slot, l), n = __shfl_sync(0xffffffffu, count, l), to = __shfl_sync(0xffffffffu, at, l);
      if (s < 0) continue;
      for (int k = lane; k < n; k += 32) {
        const size_t from = (size_t)s * width + k;
        if (k < n_pages - to) free[to + k] = table[from];
        table[from] = -1;
      }
      if (lane == 0) lengths[s] = 0;
    }
    top = (int)min((long long)top + tile, (long long)n_pages);
    __syncthreads();
  }
  if (tid == 0) n_free[0] = top;
}

int check_pool(const char* who, const void* slots, const void* lengths, const void* n_free, int n_seqs, int n_slots, int page_size) {
  if (!slots || !lengths || !n_free) SB_FAIL(SB_ERR_ARG, "%s: slots, lengths or n_free missing", who);
  if (n_seqs <= 0 || n_slots <= 0 || page_size <= 0)
    SB_FAIL(SB_ERR_ARG, "%s: %d requests, %d slots, pages of %d tokens", who, n_seqs, n_slots, page_size);
  if (n_seqs > MAX_SEQS || n_slots > MAX_SLOTS)
    SB_FAIL(SB_ERR_UNSUPPORTED, "%s: %d requests (at most %d), %d slots (at most %d)", who, n_seqs, MAX_SEQS, n_slots, MAX_SLOTS);
  return SB_OK;
}

}  // namespace

extern "C" int sb_page_tables(const SbPageTables* args, cudaStream_t stream) {
  const char* who = "sb_page_tables";
  if (!args) SB_FAIL(SB_ERR_ARG, "%s: no arguments", who);
  const SbPageTables a = *args;
  if (int rc = check_pool(who, a.slots, a.lengths, a.n_free, a.n_seqs, a.n_slots, a.page_size)) return rc;
  if (!a.fresh || !a.table || !a.free || !a.seq_row0 || !a.seq_pos0 || !a.row_seq || !a.row_pos || !a.row_slot || !a.page_off || !a.page_ids ||
      !a.status)
    SB_FAIL(SB_ERR_ARG, "%s: an array is missing", who);
  if (a.width <= 0 || a.n_pages <= 0 || a.max_rows <= 0 || a.max_pages <= 0 || a.max_new <= 0 || a.max_len <= 0)
    SB_FAIL(SB_ERR_ARG, "%s: %d pages a slot, %d pages, room for %d rows and %d pages, max_new %d, max_len %d", who, a.width, a.n_pages,
            a.max_rows, a.max_pages, a.max_new, a.max_len);
  if (a.width > MAX_COUNT || a.max_rows > MAX_COUNT || (long)a.n_pages * a.page_size > 2147483647L)
    SB_FAIL(SB_ERR_UNSUPPORTED, "%s: %d pages a slot, %d rows (at most %d), %d pages of %d tokens (places are 32-bit numbers)", who, a.width,
            a.max_rows, MAX_COUNT, a.n_pages, a.page_size);
  constexpr int MOST_SMEM = ((5 * MAX_SEQS + 2) + MAX_SLOTS / 32) * 4;
  static_assert(MOST_SMEM <= 226 * 1024, "the requests' numbers fit a block's shared memory");
  if (cudaError_t e = sb_allow_shared<page_tables_kernel>(MOST_SMEM))
    SB_FAIL(SB_ERR_CUDA, "%s: shared memory opt-in failed: %s", who, cudaGetErrorString(e));
  const size_t smem = ((size_t)5 * a.n_seqs + 2 + (a.n_slots + 31) / 32) * 4;
  const long chunks = (a.max_rows + CHUNK - 1) / CHUNK + ((long)a.max_pages + CHUNK - 1) / CHUNK;
  sb_launch<SB_K_OTHER>(page_tables_kernel, dim3((unsigned)(chunks < 256 ? chunks : 256)), dim3(TB), smem, stream, a);
  SB_CHECK_LAUNCH(who);
  return SB_OK;
}

extern "C" int sb_page_tables_settle(cudaStream_t stream) {
  sb_launch<0>(settle_kernel, dim3(1), dim3(32), 0, stream);
  SB_CHECK_LAUNCH("sb_page_tables_settle");
  return SB_OK;
}

extern "C" int sb_page_advance(const int32_t* slots, const int32_t* fresh, int n_seqs, int32_t* lengths, int n_slots, int32_t* n_free,
                               int page_size, const int32_t* status, cudaStream_t stream) {
  const char* who = "sb_page_advance";
  if (int rc = check_pool(who, slots, lengths, n_free, n_seqs, n_slots, page_size)) return rc;
  if (!fresh || !status) SB_FAIL(SB_ERR_ARG, "%s: an array is missing", who);
  sb_launch<SB_K_OTHER>(page_advance_kernel, dim3(1), dim3(TB), 0, stream, slots, fresh, n_seqs, lengths, n_slots, n_free, page_size,
                        status);
  SB_CHECK_LAUNCH(who);
  return SB_OK;
}

extern "C" int sb_page_release(const int32_t* slots, int n_seqs, int32_t* lengths, int32_t* table, int n_slots, int width, int32_t* free,
                               int n_pages, int32_t* n_free, int page_size, cudaStream_t stream) {
  const char* who = "sb_page_release";
  if (int rc = check_pool(who, slots, lengths, n_free, n_seqs, n_slots, page_size)) return rc;
  if (!table || !free || width <= 0 || n_pages <= 0) SB_FAIL(SB_ERR_ARG, "%s: %d pages a slot, %d pages, or an array is missing", who, width, n_pages);
  if (width > MAX_COUNT) SB_FAIL(SB_ERR_UNSUPPORTED, "%s: %d pages a slot (at most %d)", who, width, MAX_COUNT);
  sb_launch<SB_K_OTHER>(page_release_kernel, dim3(1), dim3(TB), (size_t)((n_slots + 31) / 32) * 4, stream, slots, n_seqs, n_slots, lengths,
                        table, width, free, n_pages, n_free, page_size);
  SB_CHECK_LAUNCH(who);
  return SB_OK;
}
