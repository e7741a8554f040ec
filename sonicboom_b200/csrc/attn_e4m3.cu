// Causal grouped-query attention over the paged cache in 8 bits (e4m3.cuh), for few rows a sequence: compiled once per head
// size (-DSB_HD), beside attn_mma.cu.
//
//   out_i = sum_j exp2(s_ij - m) v_j / sum_j exp2(s_ij - m),   s_ij = scale log2(e) (q_i . k_j)
//
// over the keys j that row i sees.  What bounds it is reading every key and value byte once; both go through the tensor cores with
// the keys (and the value's dimensions) as the long side of the tile:
//   S^T [16 keys x 8 rows] = K Q^T,   O^T [16 dims x 8 rows] += V^T P^T        (mma.sync m16n8k16, halves in, float32 out)
// A tile's k index is a sum's order and nothing more, so a thread takes what lies together: 16 bytes of a key's row for four
// k-steps of S, 16 bytes of each of four values' rows for eight tiles of O.  A warp walks its pages alone: one bulk copy brings a
// page's keys of the head, another its values, into the warp's own shared memory, and the next page's are asked for as soon as
// the tile has been read.  (Copies of 16 bytes a lane, into registers or shared memory, kept the memory at 4.4 of the 6.1 TB/s
// that bulk copies of the same pages reach: 64 sequences of 512 to 8,192 keys 78 to 80 us when bulk copies took 65.)
// e4m3 to half is exact.  q is brought to halves with a power of two for each row: a bfloat16's 8 bits stay down to 2^-17 of the
// row's largest number, smaller ones are off by at most 2^-25 of it.  Weights are rounded to halves (2^-11 of a weight) after they
// were summed in float32, times 2^15 so that those down to 2^-29 of the largest are normal numbers; smaller ones are off by at most
// 2^-40 of it.  For float32 rows q and the weights are two halves each, the second what the first left over (together within 2^-24 of
// a row's largest number, 2^-22 of a weight or 2^-40 of the largest), and every product two.
//
// Scales.  A page's key scale joins the score.  Its value scale 2^e joins the weight: with m the largest score so far and n the
// largest of score + e, weights are exp2(s - m) in the sum and exp2(s + e - n) in the product with V, each at most 1, and
// the two references meet when the partial results are merged.  "Largest" above is of the weights times their pages' scales that
// a warp has met: a page whose share is 2^29 below another's loses bits, one 2^40 below counts as 0, also in a channel where the
// other page holds zeros.  (The kernels over values and the plain one multiply in float32's or bfloat16's range.)
//
// A sequence's keys are cut into splits of whole pages by its own length alone, so this kernel's result depends on neither the batch
// nor the pages' places: a block takes one split of one key/value head, warp w its pages w, w + 4, ..., merged in warp order; splits
// are merged in ascending order by a second kernel.  (The block that is done last, by an arrival counter, took 3 us more than the
// kernel's 2 at one sequence and as much more at 64; a cluster of the splits' blocks held shared memory for sequences with fewer
// splits, 89 us when this took 65.)
#include "common.cuh"
#include "e4m3.cuh"
#include "tc5.cuh"

#ifndef SB_HD
#define SB_HD 128
#endif

namespace {

typedef __nv_bfloat16 bf16;
constexpr int HD = SB_HD;
constexpr int PAGE = 64;
constexpr int WARPS = 4;
constexpr int TILE = PAGE * HD;                  // bytes of a page's keys, or values, of one head
// Step `sub` of a tile takes sixteen of its keys: slot m (row m of S^T, k = m of O^T) is key key_of(m) + sub STEP_KEYS for m < 8, slot
// m + 8 the key HALF_KEYS behind slot m.  Where rows are 128 or 256 bytes, keys that lie as in memory begin at the same bank, and the
// 16-byte reads of eight lanes meet twice (keys) and four times (values).  There a tile lies in four quarters of sixteen rows, each a
// copy of its own, that start eight banks on from one another, and a step takes four keys of every quarter: the eight lanes read two
// quarters two apart, or all four, and none meet (64 sequences of 512 to 8,192 keys, size 128: 65.2 to 61.2 us; size 256, 12,000 keys
// each: 373 to 345).  At other sizes three more copies cost more than they save (80: 97 to 104 us; 64: 96.5 to 99.4), and a tile is
// one copy with its keys in order.
constexpr bool QUARTERS = HD % 128 == 0;
constexpr int PIECES = QUARTERS ? 4 : 1, PIECE = TILE / PIECES, PIECE_SMEM = PIECE + (QUARTERS ? 32 : 0), TILE_SMEM = PIECES * PIECE_SMEM;
constexpr int STEP_KEYS = QUARTERS ? 4 : 16, HALF_KEYS = QUARTERS ? 1 : 8;
__device__ __forceinline__ int key_of(int m) { return QUARTERS ? 16 * (((m >> 1) + 2 * (m & 1)) & 3) + 2 * (m & 1) : m; }
__device__ __forceinline__ int bytes_at(int key) { return key * HD + (QUARTERS ? (key >> 4) * 32 : 0); }
constexpr int AHEAD = HD > 64 ? 1 : HD > 32 ? 2 : 4;         // pages whose tiles a warp has room for
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
  int n_q_heads, n_kv_heads, group, n_pages, window, n_splits;    // group = n_q_heads / n_kv_heads
  uint32_t by_group;                             // ceil(2^32 / group), or 0
  float scale_log2;
};

// Pages of a split of a sequence of this length.  Shorter splits give few sequences enough blocks, longer ones cost many sequences
// less (a block's start and its partial rows).  Four, eight and sixteen pages at 28/4 heads of 128, us with the merge: one sequence of
// 1,500 keys 7.4, 9.2, 12.5 and 64 of them 31.8, 27.4, 29.1; of 6,000 keys 7.3, 9.2, 12.9 and 88.9, 72.8, 71.2; one of 30,000
// 17.2, 13.8, 14.4 and four of them 34.3, 27.7, 26.3.
__host__ __device__ constexpr int split_shift(int len) { return len <= 2048 ? 2 : len <= 16384 ? 3 : len <= 131072 ? 4 : len <= 524288 ? 6 : 8; }
constexpr int STRETCH = 8;                       // splits that are added up together
long most_splits(int max_len) {
  long most = 1;
  for (long len : {2048L, 16384L, 131072L, 524288L, (long)max_len})
    if (len <= max_len) {
      const long keys = (long)PAGE << split_shift((int)len), n = (len + keys - 1) / keys;
      if (n > most) most = n;
    }
  return most;
}

// What every kernel works out for a sequence, the same way.
struct Seq {
  int row0, n_new, pos0, last, low, sp, split_lo, split_hi;
  bool reads;                                    // its new positions lie in its own pages
};
static_assert(PAGE == 1 << 6, "pages and splits by shifts");
__device__ __forceinline__ Seq sequence(const Args& a, int b) {
  Seq s;
  s.row0 = a.seq_row0[b];
  s.n_new = a.seq_row0[b + 1] - s.row0;
  s.pos0 = a.seq_pos0[b];
  s.last = s.pos0 + s.n_new - 1;
  s.low = a.window > 0 ? max(0, s.pos0 - a.window + 1) : 0;
  const int shift = split_shift(s.last + 1), last_page = max(s.last, 0) >> 6;
  s.sp = 1 << shift;
  s.split_lo = s.low >> (6 + shift);
  s.split_hi = last_page >> shift;
  s.reads = s.pos0 >= 0 && last_page < a.page_off[b + 1] - a.page_off[b] && s.split_hi < a.n_splits;
  return s;
}

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm(
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
__device__ __forceinline__ void read_bytes(uint32_t* dst, const unsigned char* src) {
  if constexpr (BYTES == 16) {
    const uint4 v = *reinterpret_cast<const uint4*>(src);
    dst[0] = v.x; dst[1] = v.y; dst[2] = v.z; dst[3] = v.w;
  } else if constexpr (BYTES == 8) {
    const uint2 v = *reinterpret_cast<const uint2*>(src);
    dst[0] = v.x; dst[1] = v.y;
  } else if constexpr (BYTES == 4) {
    dst[0] = *reinterpret_cast<const uint32_t*>(src);
  } else {
    dst[0] = *reinterpret_cast<const uint16_t*>(src);
  }
}

// The keys of slots g and g + 8 of step `sub`, whose slot g is at `mine` in step 0: thread t of a quad has bytes 16 t ...
// of every 64, 8 t ... of 32, 4 t ... of 16.
__device__ __forceinline__ void read_keys(uint32_t (&w)[STEP_WORDS], const unsigned char* mine, int sub, int t) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const unsigned char* row = mine + (STEP_KEYS * sub + HALF_KEYS * h) * HD;
    uint32_t* dst = w + h * K_WORDS;
#pragma unroll
    for (int c = 0; c < HD / 64; ++c) read_bytes<16>(dst + 4 * c, row + 64 * c + 16 * t);
    if constexpr (N32) read_bytes<8>(dst + HD / 64 * 4, row + HD / 64 * 64 + 8 * t);
    if constexpr (N16) read_bytes<4>(dst + HD / 64 * 4 + 2 * N32, row + HD / 64 * 64 + 32 * N32 + 4 * t);
  }
}
// The values of slots 2 t + {0, 1, 8, 9}, the first two at `even` and `odd` in step 0: lane g has bytes 16 g ... of every 128, 8 g ...
// of 64, and so on.
__device__ __forceinline__ void read_values(uint32_t (&w)[STEP_WORDS], const unsigned char* even, const unsigned char* odd, int sub, int g) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const unsigned char* row = (j & 1 ? odd : even) + (STEP_KEYS * sub + HALF_KEYS * (j >> 1)) * HD;
    uint32_t* dst = w + j * V_WORDS;
#pragma unroll
    for (int c = 0; c < N128; ++c) read_bytes<16>(dst + 4 * c, row + 128 * c + 16 * g);
    if constexpr (N64) read_bytes<8>(dst + 4 * N128, row + 128 * N128 + 8 * g);
    if constexpr (N32) read_bytes<4>(dst + 4 * N128 + 2 * N64, row + 128 * N128 + 64 * N64 + 4 * g);
    if constexpr (N16) read_bytes<2>(dst + 4 * N128 + 2 * N64 + N32, row + HD - 16 + 2 * g);
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

__device__ __forceinline__ float exp2_approx(float x) {      // relative error 2^-22; 0 below 2^-126
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
}

constexpr float WEIGHT_BITS = 15.0f;             // weights as halves are at most 2^15

template <int NT, typename T>
__global__ void __launch_bounds__(WARPS * 32, HD <= 128 && NT == 1 && sizeof(T) == 2 ? 3 : 2) attn_e4m3_kernel(const Args a) {
  constexpr int ROWS = 8 * NT, PARTS = sizeof(T) / 2;
  const T* const q = (const T*)a.q;
  T* const out = (T*)a.out;
  extern __shared__ __align__(128) unsigned char tiles[];           // [warp][AHEAD][k|v][TILE_SMEM], then the warps' partial results
  float(*part)[ROWS][PART] = reinterpret_cast<float(*)[ROWS][PART]>(tiles);
  __shared__ float stat_m[WARPS][ROWS], stat_l[WARPS][ROWS], stat_n[WARPS][ROWS];
  __shared__ __align__(8) uint64_t landed[WARPS][2 * AHEAD];
  __shared__ int stopped[WARPS];                 // what each warp gave up at, or 0
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const unsigned char* const my_tiles = tiles + warp * (2 * AHEAD * TILE_SMEM);
  const uint32_t ring = (uint32_t)__cvta_generic_to_shared(my_tiles);
  const uint32_t bars = (uint32_t)__cvta_generic_to_shared(landed[warp]);
  if (lane == 0) {                               // barriers and tiles of a warp's own
#pragma unroll
    for (int i = 0; i < 2 * AHEAD; ++i) mbar_init(bars + 8 * i, 1);
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
  }
  __syncwarp();
  sb_pdl_wait();
  sb_pdl_launch();
  const int split = blockIdx.x, kvh = blockIdx.y % a.n_kv_heads, row_base = blockIdx.y / a.n_kv_heads * ROWS, b = blockIdx.z;
  const int G = a.group;
  // r / G: by_group is too large by less than G / 2^32, exact while r G < 2^32 (the host sees to that)
  auto token_of = [&](int r) { return a.by_group ? (int)__umulhi((uint32_t)r, a.by_group) : r / G; };
  const Seq sq = sequence(a, b);
  const int R = sq.n_new * G;                    // rows of this sequence and head: (new token r / G, query head r % G of the group)
  if (row_base >= R) return;
  auto row_at = [&](int r) {
    const int token = token_of(r);
    return (size_t)(sq.row0 + token) * a.n_q_heads + kvh * G + r - token * G;
  };
  if (!sq.reads) {                               // zeros; no page is read
    if (split == 0)
      for (int i = tid; i < min(ROWS, R - row_base) * (HD / 4); i += WARPS * 32)
        store_row(out + row_at(row_base + i / (HD / 4)) * HD + 4 * (i % (HD / 4)), make_float4(0.0f, 0.0f, 0.0f, 0.0f));
    return;
  }
  if (split < sq.split_lo || split > sq.split_hi) return;
  const bool single = sq.split_lo == sq.split_hi;
  // the rows' positions and what they see; the last row's lowest key and the first row's position bound the pages that all rows
  // see whole
  const int first_pos = sq.pos0 + token_of(row_base), last_pos = sq.pos0 + token_of(min(row_base + ROWS, R) - 1);
  auto low_of = [&](int pos) { return a.window > 0 ? max(0, pos - a.window + 1) : 0; };
  const int low = low_of(first_pos), high_low = low_of(last_pos);
  const int tile_lo = max(split * sq.sp, low >> 6), tile_hi = min(split * sq.sp + sq.sp - 1, last_pos >> 6);
  const int32_t* pages = a.page_ids + a.page_off[b];
  // Page i of this warp's (i from 0) goes to places 2 (i mod AHEAD) and the next; lane 0 asks for its tiles, every lane waits for them.
  const int n_tiles = (tile_hi - tile_lo - warp + WARPS) / WARPS;   // none or less: no page is this warp's
  const size_t kind = (size_t)a.n_kv_heads * TILE;
  auto page_at = [&](int i) { return min(max(pages[tile_lo + warp + i * WARPS], 0), a.n_pages - 1); };
  auto ask = [&](int i, int page, int v) {
    const uint32_t at = 2 * (i % AHEAD) + v;
    const uint8_t* src = a.cache + ((size_t)page * 2 * a.n_kv_heads + kvh) * TILE + v * kind;
    mbar_expect_tx(bars + 8 * at, TILE);
#pragma unroll
    for (int c = 0; c < PIECES; ++c)
      asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];\n" ::"r"(
                       ring + at * TILE_SMEM + c * PIECE_SMEM), "l"(src + c * PIECE), "n"(PIECE), "r"(bars + 8 * at) : "memory");
  };
  const size_t scale_stride = 2 * (size_t)a.n_kv_heads;
  int page = n_tiles > 0 ? page_at(0) : 0;
  if (lane == 0) {
#pragma unroll
    for (int i = 0; i < AHEAD; ++i)
      if (i < n_tiles) {
        const int p = i == 0 ? page : page_at(i);
        ask(i, p, 0);
        ask(i, p, 1);
      }
  }
  const int own_key = key_of(g), even_key = key_of(2 * t), odd_key = key_of(2 * t + 1);
  float k_scale = a.scales[page * scale_stride + kvh], v_scale = a.scales[page * scale_stride + a.n_kv_heads + kvh];

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

  // the rows' positions and first keys (a padding row sees nothing)
  int row_pos[NT][2], row_low[NT][2];
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int row = row_base + 8 * n + 2 * t + r;
      row_pos[n][r] = row < R ? sq.pos0 + token_of(row) : -1;
      row_low[n][r] = low_of(row_pos[n][r]);
    }
  int i = 0, gave_up = 0;                        // 1: at a page's keys, 2: at its values
  for (; i < n_tiles; ++i) {
    const uint32_t at = 2 * (i % AHEAD), parity = i / AHEAD & 1;
    const int next = i + 1 < n_tiles ? page_at(i + 1) : page, ahead = i + AHEAD < n_tiles ? page_at(i + AHEAD) : 0;
    const float next_k = a.scales[next * scale_stride + kvh], next_v = a.scales[next * scale_stride + a.n_kv_heads + kvh];
    const int e = exponent_of(v_scale);
    if (!__all_sync(0xffffffffu, mbar_wait(bars + 8 * at, parity, 31))) {
      gave_up = 1;
      break;
    }
    {
      float s[NT][4][4];
#pragma unroll
      for (int sub = 0; sub < 4; ++sub) {
        uint32_t w[STEP_WORDS];
        read_keys(w, my_tiles + at * TILE_SMEM + bytes_at(own_key), sub, t);
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) s[n][sub][i] = 0.0f;
        float s2[NT][4] = {};                    // every other step's sums: half as long a chain of products
#pragma unroll
        for (int i = 0; i < HD / 16; ++i) {
          const uint32_t x = w[i], y = w[K_WORDS + i];
          const uint32_t a0 = e4m3x2_to_half2(x & 0xffffu), a1 = e4m3x2_to_half2(y & 0xffffu);
          const uint32_t a2 = e4m3x2_to_half2(x >> 16), a3 = e4m3x2_to_half2(y >> 16);
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int j = 0; j < PARTS; ++j) mma_f16(i & 1 ? s2[n] : s[n][sub], a0, a1, a2, a3, qf[n][i][0][j], qf[n][i][1][j]);
        }
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) s[n][sub][i] += s2[n][i];
      }
      __syncwarp();
      if (lane == 0 && i + AHEAD < n_tiles) ask(i + AHEAD, ahead, 0);
      const int key0 = (tile_lo + warp + i * WARPS) * PAGE;
      const bool whole = key0 + PAGE - 1 <= first_pos && key0 >= high_low;      // every row sees every key
      uint32_t p[4][NT][2][PARTS];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float most[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const float f = fac[n][r] * k_scale;
#pragma unroll
          for (int j = 0; j < 8; ++j) s[n][j >> 1][2 * (j & 1) + r] *= f;
          if (!whole)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const int key = key0 + own_key + STEP_KEYS * (j >> 1) + HALF_KEYS * (j & 1);
              if (key > row_pos[n][r] || key < row_low[n][r]) s[n][j >> 1][2 * (j & 1) + r] = -INFINITY;
            }
#pragma unroll
          for (int j = 0; j < 8; ++j) most[r] = fmaxf(most[r], s[n][j >> 1][2 * (j & 1) + r]);
        }
        float shrink[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
#pragma unroll
          for (int x = 4; x < 32; x <<= 1) most[r] = fmaxf(most[r], __shfl_xor_sync(0xffffffffu, most[r], x));
          const float m_new = fmaxf(m[n][r], most[r]), ref_new = fmaxf(ref[n][r], most[r] + (float)e);
          const float m_at = m_new == -INFINITY ? 0.0f : m_new, ref_at = ref_new == -INFINITY ? 0.0f : ref_new;   // nothing seen: weights 0
          l[n][r] *= exp2_approx(m[n][r] - m_at);
          shrink[r] = exp2_approx(ref[n][r] - ref_at);
          // exp2(s + e - n) as exp2(s - m) exp2(e + m - n), unless the references are so far apart that a factor leaves its range
          const float apart = (float)e + m_at - ref_at;
          if (__any_sync(0xffffffffu, fabsf(apart) > 64.0f)) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              float& v = s[n][j >> 1][2 * (j & 1) + r];
              l[n][r] += exp2_approx(v - m_at);
              v = exp2_approx(v + ((float)e - ref_at + WEIGHT_BITS));
            }
          } else {
            const float factor = exp2_approx(apart + WEIGHT_BITS);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              float& v = s[n][j >> 1][2 * (j & 1) + r];
              const float weight = exp2_approx(v - m_at);
              l[n][r] += weight;
              v = weight * factor;
            }
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
      if (!__all_sync(0xffffffffu, mbar_wait(bars + 8 * (at + 1), parity, 32))) {
        gave_up = 2;
        break;
      }
#pragma unroll
      for (int sub = 0; sub < 4; ++sub) {
        uint32_t w[STEP_WORDS];
        read_values(w, my_tiles + (at + 1) * TILE_SMEM + bytes_at(even_key), my_tiles + (at + 1) * TILE_SMEM + bytes_at(odd_key), sub, g);
        if (!whole) {
          // Values that no row sees may hold anything, and 0 * NaN is NaN: they become 0.  A NaN that some rows see and others do
          // not goes to those that see it: it becomes 0 too, and a product of "is NaN" with "is seen" finds its rows.
          uint32_t nans = 0;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int key = key0 + (j & 1 ? odd_key : even_key) + STEP_KEYS * sub + HALF_KEYS * (j >> 1);
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
              const int row = row_base + 8 * n + g, pos = row < R ? sq.pos0 + token_of(row) : -1, lo = low_of(pos);
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const int first = key0 + STEP_KEYS * sub + HALF_KEYS * h, even = first + even_key, odd = first + odd_key;
                sees[n][h][0] = (even <= pos && even >= lo ? 0x3c00u : 0u) | (odd <= pos && odd >= lo ? 0x3c000000u : 0u);
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
      }
      __syncwarp();
      if (lane == 0 && i + AHEAD < n_tiles) ask(i + AHEAD, ahead, 1);
    }
    page = next;
    k_scale = next_k;
    v_scale = next_v;
  }
  if (gave_up)                                   // nothing is written; the block's memory outlives its copies
    for (int j = i; j < min(n_tiles, i + AHEAD + 1); ++j)
      for (int v = 0; v < 2; ++v)
        if (j < i + AHEAD || (v == 0 && gave_up == 2)) mbar_wait(bars + 8 * (2 * (j % AHEAD) + v), j / AHEAD & 1, 33);
  if (lane == 0) stopped[warp] = gave_up;

  // the warps' partial results, over the tiles
  __syncthreads();
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
  // merged in the warps' order: o relative to the largest score, that score, the weights' sum
  int failed = 0;
#pragma unroll
  for (int w = 0; w < WARPS; ++w) failed |= stopped[w];
  const int n_items = failed ? 0 : min(ROWS, R - row_base) * (HD / 4);
  for (int j = tid; j < n_items; j += WARPS * 32) {
    const int row = j / (HD / 4), c = 4 * (j % (HD / 4));
    float mm = -INFINITY;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) mm = fmaxf(mm, stat_m[w][row]);
    const float at = mm == -INFINITY ? 0.0f : mm;
    float sum = 0.0f;
    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      sum += stat_l[w][row] * exp2_approx(stat_m[w][row] - at);
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

// Four values of a row over some splits: sum of weights times values and of weights, relative to the largest score m.
struct Sum {
  float4 v;
  float m, l;
};
__device__ __forceinline__ void add(Sum& s, const Sum& x) {      // x, whose m is not above s.m
  const float f = exp2_approx(x.m - (s.m == -INFINITY ? 0.0f : s.m));
  s.v.x = fmaf(x.v.x, f, s.v.x); s.v.y = fmaf(x.v.y, f, s.v.y); s.v.z = fmaf(x.v.z, f, s.v.z); s.v.w = fmaf(x.v.w, f, s.v.w);
  s.l = fmaf(x.l, f, s.l);
}
// The splits of a row are added up in stretches of STRETCH, in ascending order and with their loads issued together, then the
// stretches in theirs: the same sums whoever forms them, so a row's bits depend on its sequence alone.
__device__ __forceinline__ Sum sum_of_stretch(const float* row_splits, int i, int n_splits, int c) {
  Sum x[STRETCH], s = {make_float4(0.0f, 0.0f, 0.0f, 0.0f), -INFINITY, 0.0f};
#pragma unroll
  for (int u = 0; u < STRETCH; ++u) {
    if (i * STRETCH + u >= n_splits) break;
    const float* src = row_splits + (size_t)(i * STRETCH + u) * PART;
    x[u].v = __ldcg(reinterpret_cast<const float4*>(src + c));
    const float2 ml = __ldcg(reinterpret_cast<const float2*>(src + HD));
    x[u].m = ml.x;
    x[u].l = ml.y;
  }
#pragma unroll
  for (int u = 0; u < STRETCH; ++u)
    if (i * STRETCH + u < n_splits) s.m = fmaxf(s.m, x[u].m);
#pragma unroll
  for (int u = 0; u < STRETCH; ++u)
    if (i * STRETCH + u < n_splits) add(s, x[u]);
  return s;
}
template <typename Stretch>
__device__ __forceinline__ float4 joined(Stretch stretch, int n) {
  Sum s = {make_float4(0.0f, 0.0f, 0.0f, 0.0f), -INFINITY, 0.0f};
  for (int i = 0; i < n; ++i) s.m = fmaxf(s.m, stretch(i).m);
  for (int i = 0; i < n; ++i) add(s, stretch(i));
  const float inv = 1.0f / s.l;
  return make_float4(s.v.x * inv, s.v.y * inv, s.v.z * inv, s.v.w * inv);
}

// Merges the splits of one row: a group of HD / 4 threads a stretch, as many groups as the longest sequence has stretches, up to
// MOST_GROUPS (eight groups a block whatever the splits took 1,792 rows of at most eight splits 14 us instead of 5).  The kernel before this one lets
// it start once it has waited itself, so the plan is there.  Dynamic shared memory: HD + 4 floats a stretch.
constexpr int MOST_GROUPS = 8;
template <typename T>
__global__ void __launch_bounds__(HD / 4 * MOST_GROUPS) attn_e4m3_merge_kernel(const Args a) {
  extern __shared__ __align__(16) float stretches[];                // [stretch][PART]: sums, then m and l
  sb_pdl_launch();
  const int tid = threadIdx.x, head = blockIdx.x, row = blockIdx.z;
  const Seq sq = sequence(a, blockIdx.y);
  sb_pdl_wait();
  if (row >= sq.n_new || !sq.reads || sq.split_lo == sq.split_hi) return;
  const int ns = sq.split_hi - sq.split_lo + 1, n_stretches = (ns + STRETCH - 1) / STRETCH;
  const size_t at_row = (size_t)(sq.row0 + row) * a.n_q_heads + head;
  const float* src = a.scratch + (at_row * a.n_splits + sq.split_lo) * PART;
  const int c = 4 * (tid % (HD / 4));
  for (int i = tid / (HD / 4); i < n_stretches; i += blockDim.x / (HD / 4)) {
    const Sum s = sum_of_stretch(src, i, ns, c);
    *reinterpret_cast<float4*>(stretches + (size_t)i * PART + c) = s.v;
    if (c == 0) *reinterpret_cast<float2*>(stretches + (size_t)i * PART + HD) = make_float2(s.m, s.l);
  }
  __syncthreads();
  if (tid >= HD / 4) return;
  store_row((T*)a.out + at_row * HD + c, joined([&](int i) {
    const float* s = stretches + (size_t)i * PART;
    return Sum{*reinterpret_cast<const float4*>(s + c), s[HD], s[HD + 1]};
  }, n_stretches));
}

template <int NT, typename T>
cudaError_t launch(const Args& a, dim3 grid, cudaStream_t stream) {
  constexpr int TILES = WARPS * 2 * AHEAD * TILE_SMEM, PARTIALS = WARPS * 8 * NT * PART * 4, SMEM = TILES > PARTIALS ? TILES : PARTIALS;
  if (cudaError_t e = sb_allow_shared<attn_e4m3_kernel<NT, T>>(SMEM)) return e;
  return sb_launch<SB_K_ATTENTION>(attn_e4m3_kernel<NT, T>, grid, dim3(WARPS * 32), SMEM, stream, a);
}

// Blocks of a key/value head: sixteen rows each where they fit the registers (the pages are read once for them), else eight.
bool sixteen_rows(int dtype, long rows) { return HD <= 128 && dtype == SB_BF16 && rows > 8; }
long row_groups(int dtype, long rows) { return sixteen_rows(dtype, rows) ? (rows + 15) / 16 : (rows + 7) / 8; }

}  // namespace

// 0 when no kernel of this file has given up on a wait since the last call, else the code of that wait.
extern "C" int sb_attention_e4m3_status() { return tc5_read_status(); }

extern "C" size_t sb_attention_e4m3_scratch_bytes(int n_rows, int n_q_heads, int max_len) {
  const long n = most_splits(max_len);
  return n <= 1 || n_rows <= 0 || n_q_heads <= 0 ? 0 : (size_t)n_rows * n_q_heads * n * PART * sizeof(float);
}

extern "C" int sb_attention_e4m3(const SbAttentionE4m3* args, cudaStream_t stream) {
  const char* who = "sb_attention_e4m3";
  if (!args) SB_FAIL(SB_ERR_ARG, "%s: no arguments", who);
  const SbAttentionE4m3 x = *args;
  const int dtype = x.dtype, n_seqs = x.n_seqs, max_new = x.max_new, n_q_heads = x.n_q_heads, n_kv_heads = x.n_kv_heads;
  if (x.hd != HD) SB_FAIL(SB_ERR_ARG, "%s: built for head size %d, called with %d", who, HD, x.hd);
  if (x.page_size != PAGE) SB_FAIL(SB_ERR_UNSUPPORTED, "%s: cache pages of %d keys (needs %d)", who, x.page_size, PAGE);
  if (!x.q || !x.out || !x.seq_row0 || !x.seq_pos0 || !x.page_off || !x.page_ids || !x.cache || !x.scales)
    SB_FAIL(SB_ERR_ARG, "%s: an array is missing", who);
  if (x.n_rows <= 0 || n_seqs <= 0 || max_new <= 0 || x.max_len <= 0 || n_q_heads <= 0 || n_kv_heads <= 0 || x.n_pages <= 0)
    SB_FAIL(SB_ERR_ARG, "%s: rows=%d seqs=%d max_new=%d max_len=%d heads=%d/%d pages=%d", who, x.n_rows, n_seqs, max_new, x.max_len, n_q_heads,
            n_kv_heads, x.n_pages);
  if (n_q_heads % n_kv_heads)
    SB_FAIL(SB_ERR_ARG, "%s: %d query heads are not a multiple of %d key/value heads", who, n_q_heads, n_kv_heads);
  if (x.window < 0) SB_FAIL(SB_ERR_ARG, "%s: window %d (0: none)", who, x.window);
  if (((uintptr_t)x.q | (uintptr_t)x.cache | (uintptr_t)x.scratch | (uintptr_t)x.out) & 15) SB_FAIL(SB_ERR_ARG, "%s: unaligned operands", who);
  if (!sb_valid_dtype(dtype)) SB_FAIL(SB_ERR_ARG, "%s: dtype code %d", who, dtype);
  const long rows = (long)max_new * (n_q_heads / n_kv_heads), groups = row_groups(dtype, rows);
  const long n_splits = most_splits(x.max_len), n_stretches = (n_splits + STRETCH - 1) / STRETCH;
  if (groups * n_kv_heads > 65535 || n_seqs > 65535 || max_new > 65535 || n_stretches * PART * 4 > 48 * 1024)
    SB_FAIL(SB_ERR_UNSUPPORTED, "%s: %d new rows of %d/%d heads, %d sequences, max_len %d", who, max_new, n_q_heads, n_kv_heads, n_seqs, x.max_len);
  const size_t need = sb_attention_e4m3_scratch_bytes(x.n_rows, n_q_heads, x.max_len);
  if (need > x.scratch_bytes || (need && !x.scratch))
    SB_FAIL(SB_ERR_ARG, "%s: %zu bytes of scratch needed, %zu given", who, need, x.scratch_bytes);
  const int group = n_q_heads / n_kv_heads;
  const uint32_t by_group = group > 1 && (uint64_t)(rows + 15) * group < 1ull << 32 ? (uint32_t)(((1ull << 32) + group - 1) / group) : 0;
  const Args a = {x.q, x.out, x.seq_row0, x.seq_pos0, x.page_off, x.page_ids, (const uint8_t*)x.cache, x.scales, (float*)x.scratch,
                  n_q_heads, n_kv_heads, group, x.n_pages, x.window, (int)n_splits, by_group, x.scale * LOG2E};
  const dim3 grid((unsigned)n_splits, (unsigned)(groups * n_kv_heads), n_seqs);
  cudaError_t e = cudaSuccess;
#if SB_HD <= 128
  if (sixteen_rows(dtype, rows)) e = launch<2, bf16>(a, grid, stream);
  else
#endif
    SB_DISPATCH_DTYPE(dtype, T, { e = launch<1, T>(a, grid, stream); });
  if (e != cudaSuccess) SB_FAIL(SB_ERR_CUDA, "%s: %s", who, cudaGetErrorString(e));
  SB_CHECK_LAUNCH(who);
  if (n_splits > 1) {
    const unsigned threads = HD / 4 * (unsigned)(n_stretches < MOST_GROUPS ? n_stretches : MOST_GROUPS);
    SB_DISPATCH_DTYPE(dtype, T, {
      sb_launch<SB_K_ATTENTION>(attn_e4m3_merge_kernel<T>, dim3(n_q_heads, n_seqs, max_new), dim3(threads),
                                n_stretches * PART * sizeof(float), stream, a);
    });
    SB_CHECK_LAUNCH(who);
  }
  return SB_OK;
}
