// Causal grouped-query attention over the paged cache in 8 bits (e4m3.cuh), for few rows a sequence: compiled once per head
// size (-DSB_HD), beside attn_mma.cu.
//
//   out_i = sum_j exp2(s_ij - m) v_j / sum_j exp2(s_ij - m),   s_ij = scale log2(e) (q_i . k_j)
//
// over the keys j that row i sees.  What bounds it is reading every key and value byte once, so both go from global memory
// straight into registers and through the tensor cores with the keys (and the value's dimensions) as the long side of the tile:
//   S^T [16 keys x 8 rows] = K Q^T,   O^T [16 dims x 8 rows] += V^T P^T        (mma.sync m16n8k16, halves in, float32 out)
// A tile's k index is a sum's order and nothing more, so a thread takes what lies together: 16 bytes of a key's row for four
// k-steps of S, 16 bytes of each of four values' rows for eight tiles of O.  No shared memory, no barrier: a warp walks its
// pages alone, with RING steps of 16 keys in flight.  e4m3 to half is exact.  q is brought to halves with a power of two for each
// row: a bfloat16's 8 bits stay.  Weights are rounded to halves (2^-11) after they were summed in float32, times 2^15 so that
// small ones stay normal numbers.  For float32 rows q and the weights are two halves each, the second what the first left over
// (together within 2^-24 of a row's largest value, 2^-22 of a weight), and every product two.
//
// Scales.  A page's key scale joins the score.  Its value scale 2^e joins the weight: with m the largest score so far and n the
// largest of score + e, weights are exp2(s - m) in the sum and exp2(s + e - n) in the product with V, each at most 1, and
// the two references meet when the partial results are merged.  So pages of very unequal scale lose nothing.
//
// A sequence's keys are cut into splits of whole pages by its own length alone, so a result depends on neither the batch nor
// the pages' places: a block takes one split of one key/value head, warp w its pages w, w + 4, ..., merged in warp order; splits
// are merged in ascending order by a second kernel.
#include "common.cuh"
#include "e4m3.cuh"

#ifndef SB_HD
#define SB_HD 128
#endif

namespace {

typedef __nv_bfloat16 bf16;
constexpr int HD = SB_HD;
constexpr int PAGE = 64;
constexpr int WARPS = 4;
constexpr int RING = HD > 128 ? 2 : 4;           // steps of 16 keys (or values) in flight a warp
constexpr int PART = HD + 4;                     // floats of a split's partial row: o, m, l
constexpr float LOG2E = 1.4426950408889634f;
// values of a thread: stretches of 128, 64, 32, 16 dims with 16, 8, 4, 2 bytes a lane, as head size has them
constexpr int N128 = HD / 128, N64 = HD / 64 & 1, N32 = HD / 32 & 1, N16 = HD / 16 & 1;
constexpr int K_WORDS = HD / 16;                 // words of a thread of one key's row: a quarter of it
constexpr int V_WORDS = 4 * N128 + 2 * N64 + N32 + N16;       // words of a thread of one value's row
constexpr int STEP_WORDS = 2 * K_WORDS > 4 * V_WORDS ? 2 * K_WORDS : 4 * V_WORDS;

static_assert(HD % 16 == 0 && HD >= 16 && HD <= 256, "head size in steps of 16, at most 256");

struct Args {
  const void* q;                                 // [rows, n_q_heads, HD]
  void* out;
  const int32_t *seq_row0, *seq_pos0, *page_off, *page_ids;
  const uint8_t* cache;                          // [page][k|v][kv head][PAGE][HD]
  const float* scales;                           // [page][k|v][kv head]
  float* scratch;                                // [row][q head][split][PART]
  int n_q_heads, n_kv_heads, n_pages, window, n_splits;
  float scale_log2;
};

// Pages of a split of a sequence of this length.
__host__ __device__ constexpr int split_pages(int len) { return len <= 2048 ? 4 : len <= 8192 ? 8 : 16; }
int most_splits(int max_len) {
  int most = 1;
  for (int len : {2048, 8192, max_len})
    if (len <= max_len) {
      const int keys = split_pages(len) * PAGE, n = (len + keys - 1) / keys;
      if (n > most) most = n;
    }
  return most;
}

// What every kernel works out for a sequence, the same way.
struct Seq {
  int row0, n_new, pos0, last, low, sp, split_lo, split_hi;
  bool reads;                                    // its new positions lie in its own pages
};
__device__ __forceinline__ Seq sequence(const Args& a, int b) {
  Seq s;
  s.row0 = a.seq_row0[b];
  s.n_new = a.seq_row0[b + 1] - s.row0;
  s.pos0 = a.seq_pos0[b];
  s.last = s.pos0 + s.n_new - 1;
  s.low = a.window > 0 ? max(0, s.pos0 - a.window + 1) : 0;
  s.sp = split_pages(s.last + 1);
  s.split_lo = s.low / (s.sp * PAGE);
  s.split_hi = max(s.last, 0) / (s.sp * PAGE);
  s.reads = s.pos0 >= 0 && s.last / PAGE < a.page_off[b + 1] - a.page_off[b] && s.split_hi < a.n_splits;
  return s;
}

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_half(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(r) : "r"(v));
  return r;
}

template <int BYTES>
__device__ __forceinline__ void load_bytes(uint32_t* dst, const uint8_t* src) {
  if constexpr (BYTES == 16) {
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];\n" : "=r"(dst[0]), "=r"(dst[1]), "=r"(dst[2]), "=r"(dst[3]) : "l"(src));
  } else if constexpr (BYTES == 8) {
    asm volatile("ld.global.L1::no_allocate.v2.u32 {%0,%1}, [%2];\n" : "=r"(dst[0]), "=r"(dst[1]) : "l"(src));
  } else if constexpr (BYTES == 4) {
    asm volatile("ld.global.L1::no_allocate.u32 %0, [%1];\n" : "=r"(dst[0]) : "l"(src));
  } else {
    uint16_t v;
    asm volatile("ld.global.L1::no_allocate.u16 %0, [%1];\n" : "=h"(v) : "l"(src));
    dst[0] = v;
  }
}

// Keys 16 sub + g and 16 sub + g + 8 of a page: thread t of a quad has bytes 16 t ... of every 64, 8 t ... of 32, 4 t ... of 16.
__device__ __forceinline__ void load_keys(uint32_t (&w)[STEP_WORDS], const uint8_t* page, int sub, int g, int t) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const uint8_t* row = page + (size_t)(16 * sub + 8 * h + g) * HD;
    uint32_t* dst = w + h * K_WORDS;
    int n = 0;
#pragma unroll
    for (int c = 0; c < HD / 64; ++c, n += 4) load_bytes<16>(dst + n, row + 64 * c + 16 * t);
    if constexpr (N32) load_bytes<8>(dst + HD / 64 * 4, row + HD / 64 * 64 + 8 * t);
    if constexpr (N16) load_bytes<4>(dst + HD / 64 * 4 + 2 * N32, row + HD / 64 * 64 + 32 * N32 + 4 * t);
  }
}
// Values 16 sub + 2 t + {0, 1, 8, 9} of a page: lane g has bytes 16 g ... of every 128, 8 g ... of 64, and so on.
__device__ __forceinline__ void load_values(uint32_t (&w)[STEP_WORDS], const uint8_t* page, int sub, int g, int t) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint8_t* row = page + (size_t)(16 * sub + 2 * t + (j & 1) + 8 * (j >> 1)) * HD;
    uint32_t* dst = w + j * V_WORDS;
#pragma unroll
    for (int c = 0; c < N128; ++c) load_bytes<16>(dst + 4 * c, row + 128 * c + 16 * g);
    if constexpr (N64) load_bytes<8>(dst + 4 * N128, row + 128 * N128 + 8 * g);
    if constexpr (N32) load_bytes<4>(dst + 4 * N128 + 2 * N64, row + 128 * N128 + 64 * N64 + 4 * g);
    if constexpr (N16) load_bytes<2>(dst + 4 * N128 + 2 * N64 + N32, row + HD - 16 + 2 * g);
  }
}
// The dim of a thread's accumulator d, half h (rows g and g + 8 of tile d of O^T).
__device__ __forceinline__ int dim_of(int d, int h, int g) {
  if (d < 8 * N128) return d / 8 * 128 + 16 * g + 2 * (d % 8) + h;
  int base = 128 * N128;
  d -= 8 * N128;
  if (N64) {
    if (d < 4) return base + 8 * g + 2 * d + h;
    d -= 4;
    base += 64;
  }
  if (N32) {
    if (d < 2) return base + 4 * g + 2 * d + h;
    d -= 2;
    base += 32;
  }
  return base + 2 * g + h;
}

// A value as PARTS halves: itself rounded, then what that left over.
template <int PARTS>
__device__ __forceinline__ void to_halves(uint32_t (&f)[PARTS], float lo, float hi) {
  f[0] = pack_half(lo, hi);
  if constexpr (PARTS == 2) {
    const float2 first = __half22float2(*reinterpret_cast<const __half2*>(&f[0]));
    f[1] = pack_half(lo - first.x, hi - first.y);
  }
}

// A row of q as the B operand of S^T, in the keys' order of k, over 2^x; returns 2^x, the row's largest exponent.
template <typename T, int PARTS>
__device__ __forceinline__ float load_query(uint32_t (&f)[HD / 16][2][PARTS], const T* row, bool valid, int t) {
  float v[HD / 4];
  float most = 0.0f;
#pragma unroll
  for (int i = 0; i < HD / 16; ++i) {            // four dims of k-step i
    const int c = i / 4, rest = HD / 64 * 4;
    const int dim = i < rest ? 64 * c + 16 * t + 4 * (i % 4)
                    : N32 && i < rest + 2 ? HD / 64 * 64 + 8 * t + 4 * (i - rest) : HD - 16 + 4 * t;
    if constexpr (sizeof(T) == 2) {
      uint2 raw = make_uint2(0u, 0u);
      if (valid) raw = *reinterpret_cast<const uint2*>(row + dim);
      v[4 * i] = __uint_as_float(raw.x << 16);
      v[4 * i + 1] = __uint_as_float(raw.x & 0xffff0000u);
      v[4 * i + 2] = __uint_as_float(raw.y << 16);
      v[4 * i + 3] = __uint_as_float(raw.y & 0xffff0000u);
    } else {
      float4 raw = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (valid) raw = *reinterpret_cast<const float4*>(row + dim);
      v[4 * i] = raw.x; v[4 * i + 1] = raw.y; v[4 * i + 2] = raw.z; v[4 * i + 3] = raw.w;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) most = fmaxf(most, fabsf(v[4 * i + j]));
  }
  most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
  most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
  const int x = min(max(exponent_of(most), -126), 126);
  const float inverse = exp2_int(-x);
#pragma unroll
  for (int i = 0; i < HD / 16; ++i) {
    to_halves<PARTS>(f[i][0], v[4 * i] * inverse, v[4 * i + 1] * inverse);
    to_halves<PARTS>(f[i][1], v[4 * i + 2] * inverse, v[4 * i + 3] * inverse);
  }
  return exp2_int(x);
}

// A NaN (0x7f in any byte's low bits) among four e4m3 numbers: a mask of the bytes.
__device__ __forceinline__ uint32_t nan_bytes(uint32_t v) { return __vcmpeq4(v & 0x7f7f7f7fu, 0x7f7f7f7fu); }

// O^T += V^T P^T of 16 keys.
template <int NT, int PARTS>
__device__ __forceinline__ void values_step(float (&o)[NT][HD / 16][4], const uint32_t (&w)[STEP_WORDS], const uint32_t (&p)[NT][2][PARTS]) {
  auto tile = [&](int d, uint32_t a01, uint32_t a23) {       // keys 2t, 2t+1 and 2t+8, 2t+9 of two dims, bytes in pairs
    const uint32_t a0 = e4m3x2_to_half2(a01 & 0xffffu), a1 = e4m3x2_to_half2(a01 >> 16);
    const uint32_t a2 = e4m3x2_to_half2(a23 & 0xffffu), a3 = e4m3x2_to_half2(a23 >> 16);
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int j = 0; j < PARTS; ++j) mma_f16(o[n][d], a0, a1, a2, a3, p[n][0][j], p[n][1][j]);
  };
#pragma unroll
  for (int i = 0; i < V_WORDS; ++i) {
    const uint32_t x = w[i], y = w[V_WORDS + i], z = w[2 * V_WORDS + i], u = w[3 * V_WORDS + i];
    tile(2 * i, __byte_perm(x, y, 0x5140), __byte_perm(z, u, 0x5140));
    if (!(N16 && i == V_WORDS - 1)) tile(2 * i + 1, __byte_perm(x, y, 0x7362), __byte_perm(z, u, 0x7362));
  }
}

__device__ __forceinline__ void store_row(bf16* dst, float4 v) {
  const __nv_bfloat162 lo = __floats2bfloat162_rn(v.x, v.y), hi = __floats2bfloat162_rn(v.z, v.w);
  *reinterpret_cast<uint2*>(dst) = make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
}
__device__ __forceinline__ void store_row(float* dst, float4 v) { *reinterpret_cast<float4*>(dst) = v; }

constexpr float WEIGHT_BITS = 15.0f;             // weights as halves are at most 2^15

template <int NT, typename T>
__global__ void __launch_bounds__(WARPS * 32, HD <= 128 && NT == 1 && sizeof(T) == 2 ? 3 : 2) attn_e4m3_kernel(const Args a) {
  constexpr int ROWS = 8 * NT, PARTS = sizeof(T) / 2;
  const T* const q = (const T*)a.q;
  T* const out = (T*)a.out;
  __shared__ __align__(16) float part[WARPS][ROWS][PART];
  __shared__ float stat_m[WARPS][ROWS], stat_l[WARPS][ROWS], stat_n[WARPS][ROWS];
  sb_pdl_wait();
  sb_pdl_launch();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int split = blockIdx.x, kvh = blockIdx.y % a.n_kv_heads, row_base = blockIdx.y / a.n_kv_heads * ROWS, b = blockIdx.z;
  const int G = a.n_q_heads / a.n_kv_heads;
  const Seq sq = sequence(a, b);
  const int R = sq.n_new * G;                    // rows of this sequence and head: (new token r / G, query head r % G of the group)
  if (row_base >= R) return;
  auto row_at = [&](int r) { return (size_t)(sq.row0 + r / G) * a.n_q_heads + kvh * G + r % G; };
  if (!sq.reads) {                               // zeros; no page is read
    if (split == 0)
      for (int i = tid; i < min(ROWS, R - row_base) * (HD / 4); i += WARPS * 32)
        store_row(out + row_at(row_base + i / (HD / 4)) * HD + 4 * (i % (HD / 4)), make_float4(0.0f, 0.0f, 0.0f, 0.0f));
    return;
  }
  if (split < sq.split_lo || split > sq.split_hi) return;
  // the rows' positions and what they see; the last row's lowest key and the first row's position bound the pages that all rows
  // see whole
  const int first_pos = sq.pos0 + row_base / G, last_pos = sq.pos0 + (min(row_base + ROWS, R) - 1) / G;
  auto low_of = [&](int pos) { return a.window > 0 ? max(0, pos - a.window + 1) : 0; };
  const int low = low_of(first_pos), high_low = low_of(last_pos);
  const int tile_lo = max(split * sq.sp, low / PAGE), tile_hi = min(split * sq.sp + sq.sp - 1, last_pos / PAGE);
  const int32_t* pages = a.page_ids + a.page_off[b];

  uint32_t qf[NT][HD / 16][2][PARTS];
  float fac[NT][2];                              // of rows 2t, 2t + 1: 2^x scale log2(e)
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int r = row_base + 8 * n + g;
    const float f = load_query<T, PARTS>(qf[n], q + row_at(min(r, R - 1)) * HD, r < R, t) * a.scale_log2;
    fac[n][0] = __shfl_sync(0xffffffffu, f, 8 * t);
    fac[n][1] = __shfl_sync(0xffffffffu, f, 8 * t + 4);
  }
  float m[NT][2], l[NT][2], ref[NT][2], o[NT][HD / 16][4];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
#pragma unroll
    for (int r = 0; r < 2; ++r) m[n][r] = ref[n][r] = -INFINITY, l[n][r] = 0.0f;
#pragma unroll
    for (int d = 0; d < HD / 16; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i) o[n][d][i] = 0.0f;
  }

  const size_t kind = (size_t)a.n_kv_heads * PAGE * HD;
  auto page_at = [&](int tile) { return min(max(pages[tile], 0), a.n_pages - 1); };
  auto bytes_of = [&](int page) { return a.cache + ((size_t)page * 2 * a.n_kv_heads + kvh) * (PAGE * HD); };
  uint32_t ring[RING][STEP_WORDS];
  // step s = 0 ... 7 of a page: its keys in four steps, then its values
  auto issue = [&](uint32_t (&w)[STEP_WORDS], const uint8_t* page, int s) {
    if (s < 4) load_keys(w, page, s, g, t);
    else load_values(w, page + kind, s - 4, g, t);
  };
  int tile = tile_lo + warp;
  if (tile <= tile_hi) {
    int page = page_at(tile);
    const uint8_t* bytes = bytes_of(page);
#pragma unroll
    for (int s = 0; s < RING; ++s) issue(ring[s], bytes, s);
    while (true) {
      const float k_scale = a.scales[(size_t)page * 2 * a.n_kv_heads + kvh];
      const int e = exponent_of(a.scales[((size_t)page * 2 + 1) * a.n_kv_heads + kvh]);
      const bool more = tile + WARPS <= tile_hi;
      const int next_page = more ? page_at(tile + WARPS) : page;
      const uint8_t* next_bytes = bytes_of(next_page);
      float s[NT][4][4];
#pragma unroll
      for (int sub = 0; sub < 4; ++sub) {
        const uint32_t(&w)[STEP_WORDS] = ring[sub % RING];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) s[n][sub][i] = 0.0f;
#pragma unroll
        for (int i = 0; i < HD / 16; ++i) {
          const uint32_t x = w[i], y = w[K_WORDS + i];
          const uint32_t a0 = e4m3x2_to_half2(x & 0xffffu), a1 = e4m3x2_to_half2(y & 0xffffu);
          const uint32_t a2 = e4m3x2_to_half2(x >> 16), a3 = e4m3x2_to_half2(y >> 16);
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int j = 0; j < PARTS; ++j) mma_f16(s[n][sub], a0, a1, a2, a3, qf[n][i][0][j], qf[n][i][1][j]);
        }
        if (sub + RING < 8) issue(ring[sub % RING], bytes, sub + RING);
        else if (more) issue(ring[sub % RING], next_bytes, sub + RING - 8);
      }
      const int key0 = tile * PAGE;
      const bool whole = key0 + PAGE - 1 <= first_pos && key0 >= high_low;      // every row sees every key
      uint32_t p[4][NT][2][PARTS];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float most[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const float f = fac[n][r] * k_scale;
          const int row = row_base + 8 * n + 2 * t + r, pos = row < R ? sq.pos0 + row / G : -1, lo = low_of(pos);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            float& v = s[n][i >> 1][2 * (i & 1) + r];
            const int key = key0 + 8 * i + g;
            v = whole || (key <= pos && key >= lo) ? v * f : -INFINITY;
            most[r] = fmaxf(most[r], v);
          }
        }
        float shrink[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
#pragma unroll
          for (int x = 4; x < 32; x <<= 1) most[r] = fmaxf(most[r], __shfl_xor_sync(0xffffffffu, most[r], x));
          const float m_new = fmaxf(m[n][r], most[r]), ref_new = fmaxf(ref[n][r], most[r] + (float)e);
          const float m_at = m_new == -INFINITY ? 0.0f : m_new, ref_at = ref_new == -INFINITY ? 0.0f : ref_new;   // nothing seen: weights 0
          l[n][r] *= exp2f(m[n][r] - m_at);
          shrink[r] = exp2f(ref[n][r] - ref_at);
          const float shift = (float)e - ref_at + WEIGHT_BITS;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            float& v = s[n][i >> 1][2 * (i & 1) + r];
            l[n][r] += exp2f(v - m_at);
            v = exp2f(v + shift);
          }
          m[n][r] = m_new;
          ref[n][r] = ref_new;
        }
        // most pages leave every row's reference where it was: the factors are exactly 1 then
        if (__any_sync(0xffffffffu, shrink[0] != 1.0f || shrink[1] != 1.0f)) {
#pragma unroll
          for (int d = 0; d < HD / 16; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[n][d][i] *= shrink[i & 1];
        }
#pragma unroll
        for (int sub = 0; sub < 4; ++sub) {
          to_halves<PARTS>(p[sub][n][0], s[n][sub][0], s[n][sub][1]);
          to_halves<PARTS>(p[sub][n][1], s[n][sub][2], s[n][sub][3]);
#pragma unroll
          for (int j = 0; j < PARTS; ++j) {
            p[sub][n][0][j] = transpose8x8(p[sub][n][0][j]);
            p[sub][n][1][j] = transpose8x8(p[sub][n][1][j]);
          }
        }
      }
#pragma unroll
      for (int sub = 0; sub < 4; ++sub) {
        uint32_t(&w)[STEP_WORDS] = ring[(sub + 4) % RING];
        if (!whole) {
          // Values that no row sees may hold anything, and 0 * NaN is NaN: they become 0.  A NaN that some rows see and others do
          // not goes to those that see it: it becomes 0 too, and a product of "is NaN" with "is seen" finds its rows.
          uint32_t nans = 0;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int key = key0 + 16 * sub + 2 * t + (j & 1) + 8 * (j >> 1);
            const bool seen = key <= last_pos && key >= low;
#pragma unroll
            for (int i = 0; i < V_WORDS; ++i) {
              uint32_t& v = w[j * V_WORDS + i];
              if (!seen) v = 0;
              nans |= nan_bytes(v);
            }
          }
          if (__any_sync(0xffffffffu, nans)) {
            uint32_t is_nan[STEP_WORDS], sees[NT][2][1];
#pragma unroll
            for (int i = 0; i < 4 * V_WORDS; ++i) {
              const uint32_t f = nan_bytes(w[i]);
              is_nan[i] = f & 0x38383838u;       // 1 as e4m3
              w[i] &= ~f;
            }
            float count[NT][HD / 16][4] = {};
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              const int row = row_base + 8 * n + g, pos = row < R ? sq.pos0 + row / G : -1, lo = low_of(pos);
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const int key = key0 + 16 * sub + 2 * t + 8 * h;
                sees[n][h][0] = (key <= pos && key >= lo ? 0x3c00u : 0u) | (key + 1 <= pos && key + 1 >= lo ? 0x3c000000u : 0u);
              }
            }
            values_step<NT, 1>(count, is_nan, sees);
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int d = 0; d < HD / 16; ++d)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                  if (count[n][d][i] > 0.0f) o[n][d][i] = NAN;
          }
        }
        values_step<NT, PARTS>(o, w, p[sub]);
        if (sub + 4 + RING < 8) issue(w, bytes, sub + 4 + RING);
        else if (more) issue(w, next_bytes, sub + 4 + RING - 8);
      }
      if (!more) break;
      tile += WARPS;
      page = next_page;
      bytes = next_bytes;
    }
  }

  // the warps' partial results
#pragma unroll
  for (int n = 0; n < NT; ++n) {
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int row = 8 * n + 2 * t + r;
#pragma unroll
      for (int x = 4; x < 32; x <<= 1) l[n][r] += __shfl_xor_sync(0xffffffffu, l[n][r], x);
#pragma unroll
      for (int d = 0; d < HD / 16; ++d)
        *reinterpret_cast<float2*>(&part[warp][row][dim_of(d, 0, g)]) = make_float2(o[n][d][r], o[n][d][2 + r]);
      if (g == 0) {
        stat_m[warp][row] = m[n][r];
        stat_l[warp][row] = l[n][r];
        stat_n[warp][row] = ref[n][r] - WEIGHT_BITS;
      }
    }
  }
  __syncthreads();
  const bool single = sq.split_lo == sq.split_hi;
  for (int i = tid; i < min(ROWS, R - row_base) * (HD / 4); i += WARPS * 32) {
    const int row = i / (HD / 4), c = 4 * (i % (HD / 4));
    float mm = -INFINITY;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) mm = fmaxf(mm, stat_m[w][row]);
    const float at = mm == -INFINITY ? 0.0f : mm;
    float sum = 0.0f;
    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      sum += stat_l[w][row] * exp2f(stat_m[w][row] - at);
      const float f = exp2f(stat_n[w][row] - at);
      const float4 v = *reinterpret_cast<const float4*>(&part[w][row][c]);
      acc.x += v.x * f; acc.y += v.y * f; acc.z += v.z * f; acc.w += v.w * f;
    }
    const size_t at_row = row_at(row_base + row);
    if (single) {
      const float inv = 1.0f / sum;
      store_row(out + at_row * HD + c, make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv));
    } else {
      float* dst = a.scratch + (at_row * a.n_splits + split) * PART;
      *reinterpret_cast<float4*>(dst + c) = acc;
      if (c == 0) *reinterpret_cast<float2*>(dst + HD) = make_float2(mm, sum);
    }
  }
}

// Merges the splits of one row: weights from every split's maximum, then four groups of threads add a stretch of splits each in
// ascending order, eight loads at a time, and the groups' sums are added in their order.  How the splits are shared out depends
// on their number alone.
constexpr int GROUPS = 4;
constexpr int MERGE_THREADS = (HD / 4) * GROUPS;
template <typename T>
__global__ void __launch_bounds__(MERGE_THREADS) attn_e4m3_merge_kernel(const Args a) {
  extern __shared__ __align__(16) float weights[];                  // [n_splits]
  __shared__ __align__(16) float sums[GROUPS][HD];
  __shared__ float den[MERGE_THREADS];
  sb_pdl_wait();
  sb_pdl_launch();
  const int tid = threadIdx.x, head = blockIdx.x, b = blockIdx.y, row = blockIdx.z;
  const Seq sq = sequence(a, b);
  if (row >= sq.n_new || !sq.reads || sq.split_lo == sq.split_hi) return;
  const int ns = sq.split_hi - sq.split_lo + 1;
  const size_t at_row = (size_t)(sq.row0 + row) * a.n_q_heads + head;
  const float* src = a.scratch + (at_row * a.n_splits + sq.split_lo) * PART;
  float mm = -INFINITY;
  for (int i = tid; i < ns; i += MERGE_THREADS) {
    const float v = __ldcg(src + (size_t)i * PART + HD);
    weights[i] = v;
    mm = fmaxf(mm, v);
  }
  den[tid] = mm;
  __syncthreads();
  for (int i = 0; i < MERGE_THREADS && i < ns; ++i) mm = fmaxf(mm, den[i]);
  const float at = mm == -INFINITY ? 0.0f : mm;
  __syncthreads();
  for (int i = tid; i < ns; i += MERGE_THREADS) weights[i] = exp2f(weights[i] - at);
  __syncthreads();
  const int c = 4 * (tid % (HD / 4)), group = tid / (HD / 4), per = (ns + GROUPS - 1) / GROUPS;
  float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  float sum = 0.0f;
  for (int k = group * per; k < min(ns, (group + 1) * per); ++k) {
    const float f = weights[k];
    const float4 v = __ldcg(reinterpret_cast<const float4*>(src + (size_t)k * PART + c));
    acc.x = fmaf(v.x, f, acc.x); acc.y = fmaf(v.y, f, acc.y); acc.z = fmaf(v.z, f, acc.z); acc.w = fmaf(v.w, f, acc.w);
    sum = fmaf(__ldcg(src + (size_t)k * PART + HD + 1), f, sum);
  }
  *reinterpret_cast<float4*>(&sums[group][c]) = acc;
  if (c == 0) den[group] = sum;
  __syncthreads();
  if (group) return;
#pragma unroll
  for (int i = 1; i < GROUPS; ++i) {
    const float4 v = *reinterpret_cast<const float4*>(&sums[i][c]);
    acc.x += v.x; acc.y += v.y; acc.z += v.z; acc.w += v.w;
  }
  const float inv = 1.0f / (((den[0] + den[1]) + den[2]) + den[3]);
  store_row((T*)a.out + at_row * HD + c, make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv));
}

}  // namespace

extern "C" size_t sb_attention_e4m3_scratch_bytes(int n_rows, int n_q_heads, int max_len) {
  const int n = most_splits(max_len);
  return n <= 1 || n_rows <= 0 || n_q_heads <= 0 ? 0 : (size_t)n_rows * n_q_heads * n * PART * sizeof(float);
}

extern "C" int sb_attention_e4m3(const void* q, void* out, int dtype, int n_rows, int n_seqs, int max_new, int max_len, const int32_t* seq_row0,
                                 const int32_t* seq_pos0, const int32_t* page_off, const int32_t* page_ids, int page_size,
                                 const void* cache, const float* scales, int n_pages, int n_q_heads, int n_kv_heads, int hd, int window,
                                 float scale, void* scratch, size_t scratch_bytes, cudaStream_t stream) {
  const char* who = "sb_attention_e4m3";
  if (hd != HD) SB_FAIL(SB_ERR_ARG, "%s: built for head size %d, called with %d", who, HD, hd);
  if (page_size != PAGE) SB_FAIL(SB_ERR_UNSUPPORTED, "%s: cache pages of %d keys (needs %d)", who, page_size, PAGE);
  if (!q || !out || !seq_row0 || !seq_pos0 || !page_off || !page_ids || !cache || !scales) SB_FAIL(SB_ERR_ARG, "%s: an array is missing", who);
  if (n_rows <= 0 || n_seqs <= 0 || max_new <= 0 || max_len <= 0 || n_q_heads <= 0 || n_kv_heads <= 0 || n_pages <= 0)
    SB_FAIL(SB_ERR_ARG, "%s: rows=%d seqs=%d max_new=%d max_len=%d heads=%d/%d pages=%d", who, n_rows, n_seqs, max_new, max_len, n_q_heads,
            n_kv_heads, n_pages);
  if (n_q_heads % n_kv_heads)
    SB_FAIL(SB_ERR_ARG, "%s: %d query heads are not a multiple of %d key/value heads", who, n_q_heads, n_kv_heads);
  if (window < 0) SB_FAIL(SB_ERR_ARG, "%s: window %d (0: none)", who, window);
  if ((((uintptr_t)q | (uintptr_t)cache | (uintptr_t)scratch) & 15) || ((uintptr_t)out & 15)) SB_FAIL(SB_ERR_ARG, "%s: unaligned operands", who);
  if (!sb_valid_dtype(dtype)) SB_FAIL(SB_ERR_ARG, "%s: dtype code %d", who, dtype);
  const int G = n_q_heads / n_kv_heads, n_splits = most_splits(max_len);
  const long rows = (long)max_new * G;
  const bool two = HD <= 128 && dtype == SB_BF16 && rows > 8;     // sixteen rows a block: the pages are read once for them
  const long groups = (rows + (two ? 15 : 7)) / (two ? 16 : 8);
  if (groups * n_kv_heads > 65535 || n_seqs > 65535 || max_new > 65535 || n_splits > 8192)
    SB_FAIL(SB_ERR_UNSUPPORTED, "%s: %d new rows of %d/%d heads, %d sequences, max_len %d", who, max_new, n_q_heads, n_kv_heads, n_seqs, max_len);
  const size_t need = sb_attention_e4m3_scratch_bytes(n_rows, n_q_heads, max_len);
  if (need > scratch_bytes || (need && !scratch)) SB_FAIL(SB_ERR_ARG, "%s: %zu bytes of scratch needed, %zu given", who, need, scratch_bytes);
  const Args a = {q, out, seq_row0, seq_pos0, page_off, page_ids, (const uint8_t*)cache, scales, (float*)scratch,
                  n_q_heads, n_kv_heads, n_pages, window, n_splits, scale * LOG2E};
  const dim3 grid(n_splits, (unsigned)(groups * n_kv_heads), n_seqs);
#if SB_HD <= 128
  if (two) sb_launch<SB_K_ATTENTION>(attn_e4m3_kernel<2, bf16>, grid, dim3(WARPS * 32), 0, stream, a);
#endif
  if (!two) SB_DISPATCH_DTYPE(dtype, T, { sb_launch<SB_K_ATTENTION>(attn_e4m3_kernel<1, T>, grid, dim3(WARPS * 32), 0, stream, a); });
  SB_CHECK_LAUNCH(who);
  if (n_splits > 1) {
    SB_DISPATCH_DTYPE(dtype, T, {
      sb_launch<SB_K_ATTENTION>(attn_e4m3_merge_kernel<T>, dim3(n_q_heads, n_seqs, max_new), dim3(MERGE_THREADS), n_splits * sizeof(float), stream, a);
    });
    SB_CHECK_LAUNCH(who);
  }
  return SB_OK;
}
