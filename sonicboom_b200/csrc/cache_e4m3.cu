// The paged key/value cache in 8 bits: the write that ends a q|k|v product's work, and attention that reads it in its plainest
// form.  Layout [page][k|v][head][position in page][head size] of e4m3 numbers (e4m3.cuh), scales float32 [page][k|v][head].
#include "common.cuh"
#include "e4m3.cuh"

int sb_check_attention_args(const char* who, int n_rows, int n_q_heads, int n_kv_heads, int hd, int window, int page_size);

namespace {

// The sequence's page i, or -1 where it has none: beyond its list, given back, or no page of this cache.
__device__ __forceinline__ int own_page(const int32_t* page_off, const int32_t* page_ids, int seq, int i, int n_pages) {
  const int first = page_off[seq];
  if (i < 0 || i >= page_off[seq + 1] - first) return -1;
  const int page = page_ids[first + i];
  return page < n_pages ? page : -1;
}

// -------------------------------------------------------------------------------------- store
// One block: the new rows of one sequence that lie in one page, of one head (query heads, then k, then v heads).  So the page's
// scale is decided where all its new values are at hand, with no order between blocks.
// Rotation of the pair (a, b): a c - b s, a s + b c, each product and sum rounded on its own, as everywhere in this library.
constexpr int STORE_THREADS = 128;
constexpr int STORE_FEW = 8;                      // new rows a sequence up to which a warp takes a head

template <typename TQ>
__global__ void __launch_bounds__(STORE_THREADS) store_kernel(const SbStoreE4m3 a) {
  __shared__ float warp_most[STORE_THREADS / 32];
  sb_pdl_launch();
  sb_pdl_wait();
  const int seq = blockIdx.z, head = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int row0 = a.seq_row0[seq], n_new = a.seq_row0[seq + 1] - row0, pos0 = a.seq_pos0[seq];
  if (n_new <= 0 || pos0 < 0) return;
  const int nth = pos0 / a.page_size + blockIdx.x, start = nth * a.page_size;
  const int lo = max(pos0, start), hi = min(pos0 + n_new, start + a.page_size);       // positions
  if (lo >= hi) return;
  const int width = (a.n_q_heads + 2 * a.n_kv_heads) * a.hd, half = a.rot >> 1;
  const bool is_v = head >= a.n_q_heads + a.n_kv_heads;
  auto value = [&](int pos, int e) {
    const int row = row0 + pos - pos0;
    const float* x = a.qkv + (size_t)row * width + (size_t)head * a.hd;
    if (is_v || e >= a.rot) return x[e];
    const float* turn = a.angles + (size_t)row * a.rot;
    return e < half ? sb_rot_lo(x[e], x[e + half], turn[e], turn[half + e]) : sb_rot_hi(x[e - half], x[e], turn[e - half], turn[e]);
  };
  if (head < a.n_q_heads) {
    for (int pos = lo + warp; pos < hi; pos += STORE_THREADS / 32)
      for (int e = lane; e < a.hd; e += 32)
        ((TQ*)a.q_out)[((size_t)(row0 + pos - pos0) * a.n_q_heads + head) * a.hd + e] = sb_from_f32<TQ>(value(pos, e));
    return;
  }
  const int page = own_page(a.page_off, a.page_ids, seq, nth, a.n_pages);
  if (page < 0) return;                          // no page of its own there: nothing is written
  float most = 0.0f;
  for (int pos = lo + warp; pos < hi; pos += STORE_THREADS / 32)
    for (int e = lane; e < a.hd; e += 32) most = fmaxf(most, e4m3_size(value(pos, e)));
  most = sb_warp_max(most);
  if (lane == 0) warp_most[warp] = most;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < STORE_THREADS / 32; ++w) most = fmaxf(most, warp_most[w]);
  const size_t block = (size_t)page * 2 * a.n_kv_heads + (head - a.n_q_heads);
  uint8_t* dst = (uint8_t*)a.cache + block * a.page_size * a.hd;
  int e2 = e4m3_exponent(most);
  if (lo > start) {                              // the page holds tokens of earlier steps
    const int before = exponent_of(a.scales[block]);
    if (e2 > before) {
      const float shrink = exp2_int(max(before - e2, -126));     // 2^-126 and less: nothing of a number is left
      for (int i = 2 * tid; i < (lo - start) * a.hd; i += 2 * STORE_THREADS) {
        const float2 v = e4m3x2_to_float2(*reinterpret_cast<const uint16_t*>(dst + i));
        *reinterpret_cast<uint16_t*>(dst + i) = (uint16_t)to_e4m3x2(v.x, v.y, shrink);
      }
    } else {
      e2 = before;
    }
  }
  __syncthreads();                               // everybody has read the scale
  if (tid == 0) a.scales[block] = exp2_int(e2);
  const float inverse = exp2_int(-e2);
  for (int pos = lo + warp; pos < hi; pos += STORE_THREADS / 32)
    for (int e = 2 * lane; e < a.hd; e += 64)
      *reinterpret_cast<uint16_t*>(dst + (size_t)(pos - start) * a.hd + e) = (uint16_t)to_e4m3x2(value(pos, e), value(pos, e + 1), inverse);
}

// The same for head sizes and rotated parts that are multiples of 8: a thread keeps eight values of up to P rows in registers (four
// pairs four and four, or eight of the part beyond the rotation), so a value is read once, 16 bytes at a time, between the rotation,
// the page's largest and the rounding.  Stretches of rows: 256 threads, as many heads a block as leave every SM the two blocks that
// its registers hold; the heads share the rows' angles in shared memory, and the next head's values are asked for before this
// one's are written.  2,048 rows of 28/4 heads of 128 take 13.1 us, 8.5 at the memory's pace (47 with a warp a row and every value
// read twice; 15 with values kept in shared memory for four blocks an SM).  Up to STORE_FEW rows: a warp a head.
constexpr int MANY_THREADS = 256;
constexpr int MANY_SMEM = 64 * 1024;              // the angles of a page of 64 tokens at rotated parts up to 256

template <typename TQ>
__device__ __forceinline__ void store_four(TQ* dst, const float* v);
template <>
__device__ __forceinline__ void store_four<float>(float* dst, const float* v) {
  *reinterpret_cast<float4*>(dst) = make_float4(v[0], v[1], v[2], v[3]);
}
template <>
__device__ __forceinline__ void store_four<__nv_bfloat16>(__nv_bfloat16* dst, const float* v) {
  const __nv_bfloat162 x = __floats2bfloat162_rn(v[0], v[1]), y = __floats2bfloat162_rn(v[2], v[3]);
  *reinterpret_cast<uint2*>(dst) = make_uint2(*reinterpret_cast<const uint32_t*>(&x), *reinterpret_cast<const uint32_t*>(&y));
}
__device__ __forceinline__ void load_four(float* v, const float* src) {
  const float4 x = *reinterpret_cast<const float4*>(src);
  v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
}

template <int THREADS, int P, typename TQ>
__global__ void __launch_bounds__(THREADS) store_many_kernel(const SbStoreE4m3 a, int heads_per_block) {
  extern __shared__ __align__(16) float turns[];               // [row][rot]: the rows' angles
  __shared__ float warp_most[2][THREADS / 32];
  sb_pdl_launch();
  sb_pdl_wait();
  const int seq = blockIdx.z, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int row0 = a.seq_row0[seq], n_new = a.seq_row0[seq + 1] - row0, pos0 = a.seq_pos0[seq];
  if (n_new <= 0 || pos0 < 0) return;
  const int nth = pos0 / a.page_size + blockIdx.x, start = nth * a.page_size;
  const int lo = max(pos0, start), hi = min(pos0 + n_new, start + a.page_size);       // positions
  if (lo >= hi) return;
  const int page = own_page(a.page_off, a.page_ids, seq, nth, a.n_pages);
  const int units = a.hd / 8, per_pass = THREADS / units, u = tid % units, r = tid / units, first = row0 + lo - pos0;
  const int half = a.rot >> 1, pairs = a.rot / 8, n_turned = a.n_q_heads + a.n_kv_heads, n_heads = n_turned + a.n_kv_heads;
  const int e1 = u < pairs ? 4 * u : a.rot + 8 * (u - pairs), e2 = u < pairs ? e1 + half : e1 + 4;
  const int head0 = blockIdx.y * heads_per_block, head1 = min(head0 + heads_per_block, n_heads);
  auto mine = [&](int p) { return r < per_pass && lo + r + p * per_pass < hi; };
  auto load = [&](float (&x)[P][8], int head) {
#pragma unroll
    for (int p = 0; p < P; ++p) {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[p][i] = 0.0f;
      if (mine(p)) {
        const float* src = a.qkv + ((size_t)(first + r + p * per_pass) * n_heads + head) * a.hd;
        load_four(x[p], src + e1);
        load_four(x[p] + 4, src + e2);
      }
    }
  };
  float x[P][8];
  load(x, head0);
  const float* my_turns = a.angles + (size_t)first * a.rot;
  if (THREADS > 32 && head0 < n_turned) {
    for (int i = 4 * tid; i < (hi - lo) * a.rot; i += 4 * THREADS)
      *reinterpret_cast<float4*>(turns + i) = *reinterpret_cast<const float4*>(my_turns + i);
    my_turns = turns;
    __syncthreads();
  }
  for (int head = head0; head < head1; ++head) {
    const bool is_q = head < a.n_q_heads;
    if (!is_q && page < 0) return;               // no page of its own there: nothing is written
    float next[P][8];                            // the next head's values are on their way while this one's are written
    if (THREADS > 32 && head + 1 < head1) load(next, head + 1);
    if (u < pairs && head < n_turned) {
#pragma unroll
      for (int p = 0; p < P; ++p)
        if (mine(p)) {
          float cs[4], sn[4];
          load_four(cs, my_turns + (size_t)(r + p * per_pass) * a.rot + 4 * u);
          load_four(sn, my_turns + (size_t)(r + p * per_pass) * a.rot + half + 4 * u);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float y = x[p][i], z = x[p][4 + i];
            x[p][i] = sb_rot_lo(y, z, cs[i], sn[i]);
            x[p][4 + i] = sb_rot_hi(y, z, cs[i], sn[i]);
          }
        }
    }
    if (is_q) {
#pragma unroll
      for (int p = 0; p < P; ++p)
        if (mine(p)) {
          TQ* dst = (TQ*)a.q_out + ((size_t)(first + r + p * per_pass) * a.n_q_heads + head) * a.hd;
          store_four<TQ>(dst + e1, x[p]);
          store_four<TQ>(dst + e2, x[p] + 4);
        }
    } else {
      const size_t block = (size_t)page * 2 * a.n_kv_heads + (head - a.n_q_heads);
      uint8_t* dst = (uint8_t*)a.cache + block * a.page_size * a.hd;
      const int before = lo > start ? exponent_of(a.scales[block]) : E4M3_LOWEST;      // of tokens of earlier steps
      float most = 0.0f;
#pragma unroll
      for (int p = 0; p < P; ++p)
#pragma unroll
        for (int i = 0; i < 8; ++i) most = fmaxf(most, e4m3_size(x[p][i]));
      most = sb_warp_max(most);
      float* shared = warp_most[head & 1];       // two of them: the next head's are written while these are read
      if (lane == 0) shared[warp] = most;
      __syncthreads();                           // and everybody has read the scale
#pragma unroll
      for (int w = 0; w < THREADS / 32; ++w) most = fmaxf(most, shared[w]);
      const int e = max(e4m3_exponent(most), before);
      if (lo > start && e > before) {
        const float shrink = exp2_int(max(before - e, -126));      // 2^-126 and less: nothing of a number is left
        for (int i = 4 * tid; i < (lo - start) * a.hd; i += 4 * THREADS) {
          const uint32_t v = *reinterpret_cast<const uint32_t*>(dst + i);
          const float2 y = e4m3x2_to_float2(v & 0xffffu), z = e4m3x2_to_float2(v >> 16);
          *reinterpret_cast<uint32_t*>(dst + i) = to_e4m3x2(y.x, y.y, shrink) | to_e4m3x2(z.x, z.y, shrink) << 16;
        }
      }
      if (tid == 0) a.scales[block] = exp2_int(e);
      const float inverse = exp2_int(-e);
#pragma unroll
      for (int p = 0; p < P; ++p)
        if (mine(p)) {
          uint8_t* row = dst + (size_t)(lo - start + r + p * per_pass) * a.hd;
          *reinterpret_cast<uint32_t*>(row + e1) = to_e4m3x2(x[p][0], x[p][1], inverse) | to_e4m3x2(x[p][2], x[p][3], inverse) << 16;
          *reinterpret_cast<uint32_t*>(row + e2) = to_e4m3x2(x[p][4], x[p][5], inverse) | to_e4m3x2(x[p][6], x[p][7], inverse) << 16;
        }
    }
    if (THREADS > 32) {
#pragma unroll
      for (int p = 0; p < P; ++p)
#pragma unroll
        for (int i = 0; i < 8; ++i) x[p][i] = next[p][i];
    }
  }
}

// -------------------------------------------------------------------------------------- values
// The pages of a step's sequences as values in bfloat16 or float32, one after another as the plan lists them: [place in
// page_ids][k|v][head][position][hd], with `numbers` for the page list that says so.  Exact (a number has four bits, the scale is a power of two) but for bfloat16 at
// scales below 2^-124, whose smallest numbers lie below bfloat16's smallest, 2^-133, and are rounded to it or to 0.  What no row of
// the step sees (positions behind a sequence's end, before its first row's window) becomes 0, whatever the page holds there; pages
// that lie wholly before the window are left out.  A sequence whose list ends before its last row gets rows of zeros in `out`, which
// the attention of bfloat16 rows behind this kernel leaves alone; that of float32 rows goes row by row, and finds that the pages
// there are have no number: their keys and values count as zeros.  One block a page and head, 16 bytes out a thread and step
// (8 bytes in for bfloat16: with 16 in and 32 out a thread, 16,512 tokens took 24 us instead of 10); bound by memory (1 byte in, 2 or
// 4 out a value) or, at few pages, by its start.  What attends to the values waits for this kernel before it reads any of them.
constexpr int VALUES_THREADS = 128;

// Numbers times a scale, 16 bytes of results: eight of bfloat16, four of float32 (or of bfloat16, 8 bytes).
__device__ __forceinline__ uint32_t bf16_pair(uint32_t v, float scale) {
  const float2 a = e4m3x2_to_float2(v);
  const __nv_bfloat162 x = __floats2bfloat162_rn(a.x * scale, a.y * scale);
  return *reinterpret_cast<const uint32_t*>(&x);
}
__device__ __forceinline__ void store_values(__nv_bfloat16* dst, const uint32_t (&v)[2], float scale) {
  *reinterpret_cast<uint4*>(dst) = make_uint4(bf16_pair(v[0] & 0xffffu, scale), bf16_pair(v[0] >> 16, scale),
                                              bf16_pair(v[1] & 0xffffu, scale), bf16_pair(v[1] >> 16, scale));
}
__device__ __forceinline__ void store_values(__nv_bfloat16* dst, const uint32_t (&v)[1], float scale) {
  *reinterpret_cast<uint2*>(dst) = make_uint2(bf16_pair(v[0] & 0xffffu, scale), bf16_pair(v[0] >> 16, scale));
}
__device__ __forceinline__ void store_values(float* dst, const uint32_t (&v)[1], float scale) {
  const float2 a = e4m3x2_to_float2(v[0] & 0xffffu), b = e4m3x2_to_float2(v[0] >> 16);
  *reinterpret_cast<float4*>(dst) = make_float4(a.x * scale, a.y * scale, b.x * scale, b.y * scale);
}

template <int WORDS, typename T>
__global__ void __launch_bounds__(VALUES_THREADS)
values_kernel(const int32_t* seq_row0, const int32_t* seq_pos0, const int32_t* page_off, const int32_t* page_ids, int n_list, int page_size,
              const uint8_t* cache, const float* scales, int n_pages, int n_kv_heads, int hd, int window, T* values,
              int32_t* numbers, T* out, int out_width) {
  sb_pdl_wait();
  const int i = blockIdx.x, head = blockIdx.y, seq = blockIdx.z, tid = threadIdx.x;
  const int row0 = seq_row0[seq], n_new = seq_row0[seq + 1] - row0, pos0 = seq_pos0[seq];
  const int first = page_off[seq], n_own = page_off[seq + 1] - first, len = pos0 + n_new;
  if (n_new <= 0) return;
  if (pos0 < 0 || (len - 1) / page_size >= n_own) {
    for (size_t at = ((size_t)i * gridDim.y + head) * VALUES_THREADS + tid; at < (size_t)n_new * out_width;
         at += (size_t)gridDim.x * gridDim.y * VALUES_THREADS)
      out[(size_t)row0 * out_width + at] = sb_from_f32<T>(0.0f);
    if (i < n_own && first + i < n_list && head == 0 && tid == 0) numbers[first + i] = -1;
    return;
  }
  const int start = i * page_size, low = window > 0 ? max(0, pos0 - window + 1) : 0;
  if (start >= len || first + i >= n_list) return;
  if (head == 0 && tid == 0) numbers[first + i] = first + i;
  if (start + page_size <= low) return;
  const int page = min(max(page_ids[first + i], 0), n_pages - 1);
  const size_t block = (size_t)page * gridDim.y + head;
  const uint32_t* src = reinterpret_cast<const uint32_t*>(cache + block * page_size * hd);
  T* dst = values + ((size_t)(first + i) * gridDim.y + head) * page_size * hd;
  const float scale = scales[block];
  constexpr int STEPS = 8;                       // steps whose loads are issued together
  for (int w0 = tid; w0 < page_size * hd / (4 * WORDS); w0 += STEPS * VALUES_THREADS) {
    uint32_t v[STEPS][WORDS];
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
      const int w = w0 + i * VALUES_THREADS, pos = start + 4 * WORDS * w / hd;
#pragma unroll
      for (int j = 0; j < WORDS; ++j) v[i][j] = 0;
      if (w >= page_size * hd / (4 * WORDS) || pos < low || pos >= len) continue;
      if constexpr (WORDS == 2) {
        const uint2 x = *reinterpret_cast<const uint2*>(src + 2 * (size_t)w);
        v[i][0] = x.x; v[i][1] = x.y;
      } else {
        v[i][0] = src[w];
      }
    }
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
      const int w = w0 + i * VALUES_THREADS;
      if (w >= page_size * hd / (4 * WORDS)) break;
      store_values(dst + 4 * WORDS * (size_t)w, v[i], scale);
    }
  }
}

// -------------------------------------------------------------------------------------- plain attention
// One block per (row, query head), float32 arithmetic; chunks of 256 keys at absolute positions, merged in ascending order.
constexpr int PLAIN_THREADS = 128, PLAIN_CHUNK = 256, PLAIN_MAX_HD = 1024;

template <typename TQ>
__global__ void __launch_bounds__(PLAIN_THREADS)
attention_kernel(const TQ* q, TQ* out, const int32_t* row_seq, const int32_t* row_pos, const int32_t* page_off, const int32_t* page_ids,
                 int page_size, const uint8_t* cache, const float* scales, int n_pages, int n_q_heads, int n_kv_heads, int hd, int window,
                 float scale, int n_rows) {
  __shared__ float qs[PLAIN_MAX_HD], scores[PLAIN_CHUNK], shared[4];
  sb_pdl_launch();
  sb_pdl_wait();
  const int t = blockIdx.x, h = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int kvh = h / (n_q_heads / n_kv_heads), pos = row_pos[t], seq = row_seq[t];
  TQ* dst = out + ((size_t)t * n_q_heads + h) * hd;
  if (pos < 0) return;                           // a row behind the last sequence: left as it is
  // The sequence's last row: its rows follow one another, with another sequence's or rows of none behind them.
  int last = t, end = n_rows;
  while (end - last > 1) {
    const int mid = (last + end) >> 1;
    if (row_seq[mid] == seq && row_pos[mid] > pos) last = mid;
    else end = mid;
  }
  const int n_own = page_off[seq + 1] - page_off[seq];
  if (row_pos[last] / page_size >= n_own) {      // the list ends before that one: zeros, nothing is read
    for (int d = tid; d < hd; d += PLAIN_THREADS) dst[d] = sb_from_f32<TQ>(0.0f);
    return;
  }
  auto block_of = [&](int key, int v) -> size_t {
    const int page = min(max(page_ids[page_off[seq] + key / page_size], 0), n_pages - 1);
    return ((size_t)page * 2 + v) * n_kv_heads + kvh;
  };
  for (int d = tid; d < hd; d += PLAIN_THREADS) qs[d] = sb_to_f32<TQ>(q[((size_t)t * n_q_heads + h) * hd + d]);
  __syncthreads();
  const int lo = window > 0 ? max(0, pos - window + 1) : 0;
  float m = -INFINITY, l = 0.0f, acc[PLAIN_MAX_HD / PLAIN_THREADS] = {};
  for (int first = lo / PLAIN_CHUNK * PLAIN_CHUNK; first <= pos; first += PLAIN_CHUNK) {
    for (int j = first + warp; j < first + PLAIN_CHUNK; j += PLAIN_THREADS / 32) {
      float s = -INFINITY;
      if (j >= lo && j <= pos) {
        const size_t b = block_of(j, 0);
        const uint8_t* k = cache + (b * page_size + j % page_size) * hd;
        float dot = 0.0f;
        for (int d = lane; d < hd; d += 32) dot = fmaf(qs[d], e4m3x2_to_float2(k[d]).x, dot);
        s = sb_warp_sum(dot) * scales[b] * scale;
      }
      if (lane == 0) scores[j - first] = s;
    }
    __syncthreads();
    if (warp == 0) {
      float cm = -INFINITY;
      for (int i = lane; i < PLAIN_CHUNK; i += 32) cm = fmaxf(cm, scores[i]);
      const float m_new = fmaxf(m, sb_warp_max(cm)), base = m_new == -INFINITY ? 0.0f : m_new;
      float sum = 0.0f;
      for (int i = lane; i < PLAIN_CHUNK; i += 32) {
        const float p = expf(scores[i] - base);
        scores[i] = p;
        sum += p;
      }
      sum = sb_warp_sum(sum);
      if (lane == 0) {
        shared[0] = expf(m - base);
        shared[1] = sum;
      }
      m = m_new;
    }
    __syncthreads();
    const float alpha = shared[0];
    l = l * alpha + shared[1];
#pragma unroll
    for (int i = 0; i < PLAIN_MAX_HD / PLAIN_THREADS; ++i) acc[i] *= alpha;
    for (int j = max(first, lo); j <= min(first + PLAIN_CHUNK - 1, pos); ++j) {
      const size_t b = block_of(j, 1);
      const uint8_t* v = cache + (b * page_size + j % page_size) * hd;
      const float p = scores[j - first] * scales[b];
#pragma unroll
      for (int i = 0; i < PLAIN_MAX_HD / PLAIN_THREADS; ++i) {
        const int d = tid + i * PLAIN_THREADS;
        if (d < hd) acc[i] = fmaf(p, e4m3x2_to_float2(v[d]).x, acc[i]);
      }
    }
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < PLAIN_MAX_HD / PLAIN_THREADS; ++i) {
    const int d = tid + i * PLAIN_THREADS;
    if (d < hd) dst[d] = sb_from_f32<TQ>(acc[i] / l);
  }
}

}  // namespace

extern "C" int sb_rope_store_e4m3(const SbStoreE4m3* args, cudaStream_t stream) {
  const char* who = "sb_rope_store_e4m3";
  if (!args) SB_FAIL(SB_ERR_ARG, "%s: no arguments", who);
  const SbStoreE4m3 a = *args;
  const int max_new = a.max_new, n_q_heads = a.n_q_heads, n_kv_heads = a.n_kv_heads, hd = a.hd, rot = a.rot, page_size = a.page_size;
  if (!a.qkv || !a.seq_row0 || !a.seq_pos0 || !a.page_off || !a.page_ids || !a.cache || !a.scales || !a.q_out)
    SB_FAIL(SB_ERR_ARG, "%s: an array is missing", who);
  if (a.n_rows <= 0 || a.n_seqs <= 0 || max_new <= 0 || n_q_heads <= 0 || n_kv_heads <= 0 || page_size <= 0 || a.n_pages <= 0)
    SB_FAIL(SB_ERR_ARG, "%s: rows=%d seqs=%d max_new=%d heads=%d/%d page=%d pages=%d", who, a.n_rows, a.n_seqs, max_new, n_q_heads, n_kv_heads,
            page_size, a.n_pages);
  if (hd <= 0 || (hd & 1) || rot < 0 || rot > hd || (rot & 1))
    SB_FAIL(SB_ERR_ARG, "%s: rotary dims %d of head dim %d (both even, rotary dims at most the head dim)", who, rot, hd);
  if (rot > 0 && !a.angles) SB_FAIL(SB_ERR_ARG, "%s: %d rotary dims without angles", who, rot);
  if (!sb_valid_dtype(a.q_dtype)) SB_FAIL(SB_ERR_ARG, "%s: dtype code %d", who, a.q_dtype);
  if (a.n_seqs > 65535 || (long)n_q_heads + 2L * n_kv_heads > 65535)
    SB_FAIL(SB_ERR_UNSUPPORTED, "%s: %d sequences, %d/%d heads", who, a.n_seqs, n_q_heads, n_kv_heads);
  const int n_seqs = a.n_seqs, n_sms = a.n_sms, q_dtype = a.q_dtype;
  const int n_heads = n_q_heads + 2 * n_kv_heads;
  dim3 grid((unsigned)(((long)max_new + 2 * page_size - 2) / page_size), n_heads, n_seqs);
  if (hd % 8 == 0 && rot % 8 == 0 && hd <= 8 * MANY_THREADS &&
      (((uintptr_t)a.qkv | (uintptr_t)a.angles | (uintptr_t)a.q_out) & 15) == 0 && ((uintptr_t)a.cache & 3) == 0) {
    const bool few = max_new <= STORE_FEW && hd <= 256;
    const int per_pass = (few ? 32 : MANY_THREADS) / (hd / 8), rows = few ? max_new : page_size, passes = (rows + per_pass - 1) / per_pass;
    const long blocks = (long)grid.x * n_heads * n_seqs, fill = blocks / (2L * (n_sms > 0 ? n_sms : 1));
    const int per_block = few ? 1 : (int)(fill < 1 ? 1 : fill > 8 ? 8 : fill);
    if (passes <= 8 && (few || (long)page_size * rot * 4 <= MANY_SMEM)) {
      if (!few) {
        cudaError_t e = cudaSuccess;
        SB_DISPATCH_DTYPE(q_dtype, TQ, {
          e = passes <= 2 ? sb_allow_shared<store_many_kernel<MANY_THREADS, 2, TQ>>(MANY_SMEM)
                          : passes <= 4 ? sb_allow_shared<store_many_kernel<MANY_THREADS, 4, TQ>>(MANY_SMEM)
                                        : sb_allow_shared<store_many_kernel<MANY_THREADS, 8, TQ>>(MANY_SMEM);
        });
        if (e != cudaSuccess) SB_FAIL(SB_ERR_CUDA, "%s: shared memory opt-in failed: %s", who, cudaGetErrorString(e));
      }
      grid.y = (n_heads + per_block - 1) / per_block;
      SB_DISPATCH_DTYPE(q_dtype, TQ, {
        auto kernel = few ? (passes <= 1 ? store_many_kernel<32, 1, TQ> : passes <= 4 ? store_many_kernel<32, 4, TQ> : store_many_kernel<32, 8, TQ>)
                          : passes <= 2 ? store_many_kernel<MANY_THREADS, 2, TQ>
                                        : passes <= 4 ? store_many_kernel<MANY_THREADS, 4, TQ> : store_many_kernel<MANY_THREADS, 8, TQ>;
        sb_launch<SB_K_ELEMENTWISE>(kernel, grid, dim3(few ? 32 : MANY_THREADS), few ? 0 : (size_t)page_size * rot * sizeof(float), stream, a,
                                    per_block);
      });
      SB_CHECK_LAUNCH(who);
      return SB_OK;
    }
  }
  SB_DISPATCH_DTYPE(q_dtype, TQ, { sb_launch<SB_K_ELEMENTWISE>(store_kernel<TQ>, grid, dim3(STORE_THREADS), 0, stream, a); });
  SB_CHECK_LAUNCH(who);
  return SB_OK;
}

extern "C" int sb_cache_e4m3_values(const int32_t* seq_row0, const int32_t* seq_pos0, int n_seqs, int max_len, const int32_t* page_off,
                                    const int32_t* page_ids, int n_list, int page_size, const void* cache, const float* scales, int n_pages,
                                    int n_q_heads, int n_kv_heads, int hd, int window, void* values, int dtype,
                                    int32_t* numbers, void* out, cudaStream_t stream) {
  const char* who = "sb_cache_e4m3_values";
  if (!seq_row0 || !seq_pos0 || !page_off || !page_ids || !cache || !scales || !values || !numbers || !out)
    SB_FAIL(SB_ERR_ARG, "%s: an array is missing", who);
  if (n_seqs <= 0 || max_len <= 0 || n_list <= 0 || page_size <= 0 || n_pages <= 0 || n_q_heads <= 0 || n_kv_heads <= 0 || window < 0)
    SB_FAIL(SB_ERR_ARG, "%s: seqs=%d max_len=%d list=%d page=%d pages=%d heads=%d/%d window=%d", who, n_seqs, max_len, n_list, page_size,
            n_pages, n_q_heads, n_kv_heads, window);
  if (hd <= 0 || hd % 4 || (((uintptr_t)cache | (uintptr_t)values) & 15))
    SB_FAIL(SB_ERR_UNSUPPORTED, "%s: head size %d (a multiple of 4), or unaligned pages", who, hd);
  if (!sb_valid_dtype(dtype)) SB_FAIL(SB_ERR_ARG, "%s: dtype code %d", who, dtype);
  if (n_seqs > 65535 || n_kv_heads > 32767) SB_FAIL(SB_ERR_UNSUPPORTED, "%s: %d sequences, %d key/value heads", who, n_seqs, n_kv_heads);
  const dim3 grid((max_len + page_size - 1) / page_size, 2 * n_kv_heads, n_seqs);
  SB_DISPATCH_DTYPE(dtype, T, {
    auto kernel = values_kernel<1, T>;
    if constexpr (sizeof(T) == 2) {
      if (hd % 8 == 0) kernel = values_kernel<2, T>;
    }
    sb_launch<SB_K_ELEMENTWISE>(kernel, grid, dim3(VALUES_THREADS), 0, stream, seq_row0, seq_pos0, page_off, page_ids, n_list,
                                page_size, (const uint8_t*)cache, scales, n_pages, n_kv_heads, hd, window, (T*)values, numbers, (T*)out,
                                n_q_heads * hd);
  });
  SB_CHECK_LAUNCH(who);
  return SB_OK;
}

extern "C" int sb_attention_e4m3_plain(const void* q, void* out, int act_dtype, int n_rows, const int32_t* row_seq, const int32_t* row_pos,
                                       const int32_t* page_off, const int32_t* page_ids, int page_size, const void* cache,
                                       const float* scales, int n_pages, int n_q_heads, int n_kv_heads, int hd, int window, float scale,
                                       cudaStream_t stream) {
  const char* who = "sb_attention_e4m3_plain";
  if (int rc = sb_check_attention_args(who, n_rows, n_q_heads, n_kv_heads, hd, window, page_size)) return rc;
  if (!q || !out || !row_seq || !row_pos || !page_off || !page_ids || !cache || !scales || n_pages <= 0)
    SB_FAIL(SB_ERR_ARG, "%s: %d pages, or an array is missing", who, n_pages);
  if (hd > PLAIN_MAX_HD) SB_FAIL(SB_ERR_UNSUPPORTED, "%s: head dim %d is above %d", who, hd, PLAIN_MAX_HD);
  if (!sb_valid_dtype(act_dtype)) SB_FAIL(SB_ERR_ARG, "%s: dtype code %d", who, act_dtype);
  if (n_q_heads > 65535) SB_FAIL(SB_ERR_UNSUPPORTED, "%s: %d heads", who, n_q_heads);
  SB_DISPATCH_DTYPE(act_dtype, TQ, {
    sb_launch<SB_K_OTHER>(attention_kernel<TQ>, dim3(n_rows, n_q_heads), dim3(PLAIN_THREADS), 0, stream, (const TQ*)q, (TQ*)out, row_seq,
                          row_pos, page_off, page_ids, page_size, (const uint8_t*)cache, scales, n_pages, n_q_heads, n_kv_heads, hd, window,
                          scale, n_rows);
  });
  SB_CHECK_LAUNCH(who);
  return SB_OK;
}
