// Causal sliding-window attention with sinks and a bucketed relative position bias, for long text (driven by
// ops/window_ops.py): forward, backward, and the form for one new token over a ring cache.
//
//   visible(i, j) = j <= i and (i - j < W or j < sinks), tokens i and j both real (mask)
//   s_ij = scale q_i·k_j + bias[c, h, bucket(i − j)],  p = softmax over the visible j,  o_i = Σ p_ij v_j
//   D_i = dO_i·o_i,  dS = p (dO_i·v_j − D_i),  dq_i = scale Σ dS k_j,  dk_j = scale Σ dS q_i,  dv_j = Σ p dO_i
//   dbias[c, h, b] = Σ over the client's sequences and the visible pairs of bucket b of dS
//
// Layouts: token-major rows [sequence · S + token][heads · D], head h at column D·h; H query heads share KV heads of
// keys and values (head h reads kv head h / (H / KV)). Storage bf16 or fp32, sums and statistics fp32.
//
// All kernels work on 32×32 blocks of scores with the same maps of lanes (l = lane, hh = l >> 5):
//   C / D of the 32×32 products: column l & 31, row κ(r) + 4·hh, κ(r) = (r & 3) + 8·(r >> 2), r = 0 … 15;
//   row operands (both sides of a product over the head dim): lane l holds 16 bytes of row l & 31, unit 2c + hh of
//   the row for chunk c — one 32×32×16 bf16 product, or four 32×32×2 fp32 products; the order of the dims inside a
//   chunk is the same on both sides, so the sum is over all of them;
//   column operands (products over 32 rows of an LDS tile): the 16 accumulators of a lane ARE the other operand,
//   with the rows taken in the order κ(r) + 4·hh, so probabilities never leave the registers.
//
// Measured on MI355X (a large copy reaches 4.94 TB/s, an 8192³ product 1420 TFLOP/s bf16 and 154 fp32), medians:
//   forward, bf16:  32768 tokens, 32 heads over 8, D 128, W 1024: 813 us = 667 TFLOP/s; 16 · 1999 (a quarter padding),
//                   12 heads, D 64, W 256: 101 us
//   dq / dk, dv:    2 · 16384, 16 heads over 4, D 128, W 1024: 541 / 994 us = 762 / 553 TFLOP/s of the products they
//                   make (3 and 4 a block); 16 · 1999 as above: 106 / 157 us
//   step, bf16:     64 caches of 4100 slots, 32 heads over 8, D 128, with a bias: 239 us = 4.5 TB/s
// Shares of the wave cycles at these sizes, matrix unit / vector unit / waiting for loads, LDS and barriers / for a turn:
//   D 128: forward 19 / 26 / 26 / 34 %, dq 20 / 19 / 41 / 28, dk/dv 28 / 25 / 36 / 22;
//   D 64:  forward 6 / 19 / 37 / 34 %, dq 7 / 15 / 38 / 36, dk/dv 10 / 19 / 45 / 20.
// The wait is the largest share of both backward passes: a tile is stored to the one LDS buffer, waited for, used and
// waited for again, with two waves a SIMD in the forward and dq and one in dk/dv at D 128, whose sums, keys and values take
// 416 registers. At D 64 a short window's walk is 6 or 7 such tiles, half of them at its edges and masked.
// Tried at D 128: keys and values of dk/dv in LDS with two waves a SIMD 1091 us; two blocks interleaved: spills, 1407 us.
#include "common.h"
#include <type_traits>

namespace win {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short v4i16 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) v4i16 lds_v4i16;

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kMfma = 0x8, kDsRead = 0x100;      // classes of instructions for the scheduler
constexpr float kGrow = 8.f;      // see fwd_kernel
constexpr int kMaxBuckets = 128;
constexpr int kLutOff = 94;      // a processed block of 32 queries and <= 64 keys holds distances >= −94 (the negative
                                 // ones are masked), and below max_distance + 94 if it holds one below max_distance
constexpr int kBinPad = 64;      // distances of a block that starts below max_distance end below max_distance + 62

struct Args {
  const void *q, *k, *v, *dout;
  void *o, *dq, *dk, *dv;
  float *o32, *lse, *dsum, *part, *bpart, *dbias;
  const uint8_t* mask;
  const float* bias;
  int64_t ldq, ldk, ldv, lddo;
  int N, S, H, KV, C, W, sinks, NB, maxd;
  int nchunk, qchunk, nslot;     // sink pass of the backward: chunks of queries, partial sums of a kv head
  int exact;                     // forward: a gradient of the bias follows
  int tile, ktile;               // a workgroup's queries, forward and dq: 32 or 128; its keys, dk and dv: 64 or 128
  float scale;
  int start[kMaxBuckets];        // first distance of every bucket
};

__device__ __forceinline__ int kappa(int r) { return (r & 3) + 8 * (r >> 2); }

// consecutive work items to the same XCD (workgroup ids go round the 8 of them), so that tiles which read the same
// keys meet in one L2
__device__ __forceinline__ int xcd_swizzle(int id, int n) {
  const int per = n >> 3;
  return id < per * 8 ? (id & 7) * per + (id >> 3) : id;
}

template <typename T> struct Elem;
template <> struct Elem<uint16_t> {
  static __device__ __forceinline__ f32x16 mma(uint4 a, uint4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0,
                                                   0, 0);
  }
  // a unit times as many fp32 values
  static __device__ __forceinline__ float dot(uint4 a, const float* y, float s) {
    const uint32_t x[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 b = *reinterpret_cast<const float2*>(y + 2 * i);
      s = fmaf(__uint_as_float(x[i] << 16), b.x, s);
      s = fmaf(__uint_as_float(x[i] & 0xffff0000u), b.y, s);
    }
    return s;
  }
  // four consecutive columns
  static __device__ __forceinline__ void store4(uint16_t* p, float a, float b, float c, float d) {
    uint2 u;
    u.x = (uint32_t)f32_to_bf16(a) | ((uint32_t)f32_to_bf16(b) << 16);
    u.y = (uint32_t)f32_to_bf16(c) | ((uint32_t)f32_to_bf16(d) << 16);
    *reinterpret_cast<uint2*>(p) = u;
  }
  // what the rounding of a leaves over
  static __device__ __forceinline__ float left(float a) { return a - bf16_to_f32(f32_to_bf16(a)); }
};
template <> struct Elem<float> {
  static __device__ __forceinline__ f32x16 mma(uint4 a, uint4 b, f32x16 c) {
    const float4 x = __builtin_bit_cast(float4, a), y = __builtin_bit_cast(float4, b);
    c = __builtin_amdgcn_mfma_f32_32x32x2f32(x.x, y.x, c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_32x32x2f32(x.y, y.y, c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_32x32x2f32(x.z, y.z, c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_32x32x2f32(x.w, y.w, c, 0, 0, 0);
  }
  static __device__ __forceinline__ float dot(uint4 a, const float* y, float s) {
    const float4 x = __builtin_bit_cast(float4, a), b = *reinterpret_cast<const float4*>(y);
    return fmaf(x.x, b.x, fmaf(x.y, b.y, fmaf(x.z, b.z, fmaf(x.w, b.w, s))));
  }
  static __device__ __forceinline__ void store4(float* p, float a, float b, float c, float d) {
    *reinterpret_cast<float4*>(p) = make_float4(a, b, c, d);
  }
  static __device__ __forceinline__ float left(float) { return 0.f; }
};

__device__ __forceinline__ f32x16 zero16() {
  f32x16 z;
#pragma unroll
  for (int r = 0; r < 16; ++r) z[r] = 0.f;
  return z;
}

// A product's result may be read 18 instruction slots after its issue at fp32 (16 passes), 12 at bf16 (8). The compiler
// leaves that much room, but not over every branch: in an earlier form of the biased fp32 forward its assembly read an
// accumulator 17 slots behind the product. Wait here, in the product's own block, 20 slots for either type.
__device__ __forceinline__ void settle(f32x16& a) { asm volatile("s_nop 15\n\ts_nop 3" : "+v"(a)); }
__device__ __forceinline__ void settle(f32x16& a, f32x16& b) {
  asm volatile("s_nop 15\n\ts_nop 3" : "+v"(a), "+v"(b));
}

// over the two halves of the wave (which hold the same column)
__device__ __forceinline__ float half_max(float v) {
  const auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(x[0]), __uint_as_float(x[1]));
}
__device__ __forceinline__ float half_sum(float v) {
  const auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(x[0]) + __uint_as_float(x[1]);
}

// What a block of scores (32 queries from q, nk keys from k) is to a wave: seen at all, seen whole
__device__ __forceinline__ bool block_seen(const Args& a, int q, int k, int nk) {
  return q < a.S && k < a.S && k <= q + 31 && (q - k - nk + 1 < a.W || k < a.sinks);
}
__device__ __forceinline__ bool block_whole(const Args& a, int q, int k, int nk) {
  return k + nk - 1 <= q && (q + 31 - k < a.W || k + nk - 1 < a.sinks);
}

// lane j of ROWS: is row r0 + j < end a token (their ballot: a tile's bits)
template <int ROWS> __device__ __forceinline__ int token(const uint8_t* mask, int r0, int end, int lane) {
  const int r = r0 + lane % ROWS;
  const int m = mask ? mask[r < end ? r : end - 1] : 1;
  return r < end ? m : 0;
}
template <int ROWS> __device__ __forceinline__ uint64_t token_bits(int tok) {
  return (uint64_t)__ballot(tok != 0) & (~0ull >> (64 - ROWS));
}

// A head's rows and how they lie in registers and LDS
template <typename T, int D> struct Row {
  static constexpr int U = D * (int)sizeof(T) / 16;   // 16-byte units of a row
  static constexpr int NC = U / 2;                    // chunks: a unit for either half of the wave
  static constexpr int E = 16 / (int)sizeof(T);       // elements of a unit
  static constexpr int DB = D / 32;                   // 32-column blocks

  // LDS tiles. fp32: rows padded by 16 bytes. bf16: row r has its unit u at unit u ^ swz(r), and swz runs over the units
  // with 16 rows, so the 16 lanes that a ds_read_b128 serves at once meet 64 different banks, and the 4 rows of a
  // transposing read lie 4 units apart (padded rows cost its reads at D 128 2.5 times their cycles).
  static constexpr int P = sizeof(T) == 4 ? D + 4 : D;
  static __device__ __forceinline__ int swz(int r) {
    if constexpr (sizeof(T) == 4) return 0;
    else if constexpr (D == 64) return ((r & 2) << 1) | ((r >> 2) & 3);
    else return ((r & 3) << 2) | ((r >> 2) & 3);
  }
  static __device__ __forceinline__ int at(int r, int u) { return r * P + (u ^ swz(r)) * E; }
  // a lane's places in 32 rows of any tile, as row operand (by chunk) and as column operand (by column block and row
  // half); kept in registers as they are, so that tiles and blocks are constant offsets from them
  struct Lane {
    int row[NC], col[sizeof(T) == 4 ? 1 : 2 * (D / 32)];
    __device__ __forceinline__ explicit Lane(int lane) {
#pragma unroll
      for (int c = 0; c < NC; ++c) row[c] = at(lane & 31, 2 * c + (lane >> 5));
      if constexpr (sizeof(T) == 4) {
        col[0] = 4 * (lane >> 5) * P + (lane & 31);
      } else {
        // 16 lanes read 4 rows × 16 columns and get a column of 4 rows each
        const int g = lane >> 4, i = lane & 15;
#pragma unroll
        for (int k = 0; k < 2 * DB; ++k) {
          col[k] = at(4 * (g >> 1) + (i >> 2) + 8 * (k & 1), 4 * (k >> 1) + 2 * (g & 1) + ((i & 3) >> 1)) + 4 * (i & 1);
          asm volatile("" : "+v"(col[k]));
        }
#pragma unroll
        for (int c = 0; c < NC; ++c) asm volatile("" : "+v"(row[c]));
      }
    }
  };

  static __device__ __forceinline__ uint4 unit(const T* row, int u) {
    return *reinterpret_cast<const uint4*>(row + u * E);
  }
  // this lane's fragments of row l & 31 (zero where the row is none)
  static __device__ __forceinline__ void frags(uint4* f, const T* row, bool real, int hh) {
#pragma unroll
    for (int c = 0; c < NC; ++c) f[c] = real ? unit(row, 2 * c + hh) : make_uint4(0, 0, 0, 0);
  }
  // s0 and s1 += 32 rows each of two LDS tiles × this lane's columns: Σ over the head dim. DEEP: one tile's reads are all
  // in flight before its first product, the other's are made between those (left to itself the compiler keeps two in
  // flight, and every pair of products waits for LDS); it takes 2·NC·4 registers.
  template <bool DEEP> static __device__ __forceinline__ void rows2(f32x16& s0, f32x16& s1, const T* t0, const T* t1, const uint4* f0,
                                               const uint4* f1, const Lane& ln) {
    uint4 x[NC], y[NC];
#pragma unroll
    for (int c = 0; c < NC; ++c) x[c] = *reinterpret_cast<const uint4*>(t0 + ln.row[c]);
#pragma unroll
    for (int c = 0; c < NC; ++c) y[c] = *reinterpret_cast<const uint4*>(t1 + ln.row[c]);
#pragma unroll
    for (int c = 0; c < NC; ++c) s0 = Elem<T>::mma(x[c], f0[c], s0);
#pragma unroll
    for (int c = 0; c < NC; ++c) s1 = Elem<T>::mma(y[c], f1[c], s1);
    if constexpr (sizeof(T) == 2 && DEEP) {
      __builtin_amdgcn_sched_group_barrier(kDsRead, NC, 0);
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        __builtin_amdgcn_sched_group_barrier(kMfma, 1, 0);
        __builtin_amdgcn_sched_group_barrier(kDsRead, 1, 0);
      }
      __builtin_amdgcn_sched_group_barrier(kMfma, NC, 0);
    }
    settle(s0, s1);
  }
  static __device__ __forceinline__ f32x16 rows(const T* tile, const uint4* f, const Lane& ln) {
    f32x16 acc = zero16();
    uint4 x[NC];
#pragma unroll
    for (int c = 0; c < NC; ++c) x[c] = *reinterpret_cast<const uint4*>(tile + ln.row[c]);
#pragma unroll
    for (int c = 0; c < NC; ++c) acc = Elem<T>::mma(x[c], f[c], acc);
    if constexpr (sizeof(T) == 2) {
      __builtin_amdgcn_sched_group_barrier(kDsRead, NC, 0);
      __builtin_amdgcn_sched_group_barrier(kMfma, NC, 0);
    }
    settle(acc);
    return acc;
  }
  // acc[db][column][row] += Σ over 32 rows of the LDS tile of tile[row][32 db + ·] · p[row]. bf16: read() takes the
  // tile's fragments, ahead of the work that gives p
  struct Cols {
    const T* tile;
    bf16x8 f[sizeof(T) == 2 ? 2 * (D / 32) : 1];
    __device__ __forceinline__ void read(const T* t, const Lane& ln) {
      tile = t;
      if constexpr (sizeof(T) == 2) {
        const uint16_t* base = reinterpret_cast<const uint16_t*>(t);
#pragma unroll
        for (int k = 0; k < 2 * DB; ++k) {      // column block k / 2, rows 16 (k & 1) …; swz(row + 16) = swz(row)
          union {
            v4i16 h[2];
            bf16x8 v;
          } a;
          a.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16*)(base + 16 * (k & 1) * P + ln.col[k & ~1]));
          a.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16*)(base + 16 * (k & 1) * P + ln.col[k | 1]));
          f[k] = a.v;
        }
      }
    }
    __device__ __forceinline__ void mul(f32x16* acc, const float* p, const Lane& ln) const {
      if constexpr (sizeof(T) == 2) {
        bf16x8 b[2];
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int j = 0; j < 8; ++j) b[t][j] = (__bf16)p[8 * t + j];
#pragma unroll
        for (int k = 0; k < 2 * DB; ++k)
          acc[k / 2] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f[k], b[k & 1], acc[k / 2], 0, 0, 0);
      } else {
        const float* base = reinterpret_cast<const float*>(tile) + ln.col[0];
#pragma unroll
        for (int r = 0; r < 16; ++r)
#pragma unroll
          for (int db = 0; db < DB; ++db)
            acc[db] = __builtin_amdgcn_mfma_f32_32x32x2f32(base[kappa(r) * P + 32 * db], p[r], acc[db], 0, 0, 0);
      }
    }
  };
};

// ROWS rows of a [·][D] source between registers and an LDS tile, NT threads. Loads are unconditional, of rows up to
// `last`; a row without its bit in `bits` (no token, or behind the last) is zero in the tile, so that what it holds (NaN
// included) reaches no product.
template <typename T, int D, int ROWS, int NT> struct Stage {
  using R = Row<T, D>;
  static constexpr int NI = ROWS * R::U / NT;
  static_assert(NI >= 1 && ROWS * R::U % NT == 0 && ROWS <= 64, "staging");
  uint4 reg[NI];
  __device__ __forceinline__ void load(const T* src, int64_t ld, int row0, int last, int tid) {
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int u = tid + i * NT, row = row0 + u / R::U;
      reg[i] = R::unit(src + (row < last ? row : last) * ld, u % R::U);
    }
  }
  __device__ __forceinline__ void store(T* tile, uint64_t bits, int tid) {
    if (bits != ~0ull >> (64 - ROWS)) {
#pragma unroll
      for (int i = 0; i < NI; ++i)
        if (!((bits >> ((tid + i * NT) / R::U)) & 1)) reg[i] = make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int u = tid + i * NT;
      *reinterpret_cast<uint4*>(tile + R::at(u / R::U, u % R::U)) = reg[i];
    }
  }
};

// A bias in units of log 2. The type's lowest and highest values stay finite there (those beyond 2.08e38 count as one), and
// a product of q and k can be added to them: a row that sees nothing else than the lowest is shared out evenly.
__device__ __forceinline__ float log2_bias(float b) {
  const float x = b * kLog2e;
  if (!(fabsf(b) < INFINITY)) return x;
  return x > 3e38f ? 3e38f : x < -3e38f ? -3e38f : x;
}

// lut[d + kLutOff] = bias of distance d in units of log 2, for −94 <= d < max_distance + 94
__device__ __forceinline__ int lut_size(int maxd) { return maxd + 2 * kLutOff; }
__device__ __forceinline__ void fill_lut(float* lut, const Args& a, int client, int h, int tid, int nt) {
  const float* tab = a.bias + ((int64_t)client * a.H + h) * a.NB;
  for (int t = tid; t < lut_size(a.maxd); t += nt) {
    int b = 0;
    for (int i = 1; i < a.NB; ++i) b += (t - kLutOff >= a.start[i]) ? 1 : 0;
    lut[t] = log2_bias(tab[b]);
  }
}

// the key tiles that a tile of queries [q0, q0 + nq) sees: `first` tiles of sinks, then lo … hi
struct KeyTiles {
  int first, lo, count;
  __device__ __forceinline__ KeyTiles(const Args& a, int q0, int nq, int bk) {
    lo = q0 - a.W + 1 > 0 ? (q0 - a.W + 1) / bk : 0;
    const int last = q0 + nq - 1 < a.S - 1 ? q0 + nq - 1 : a.S - 1;
    first = (a.sinks + bk - 1) / bk;
    if (first > lo) first = lo;
    count = first + last / bk - lo + 1;
  }
  __device__ __forceinline__ int at(int i) const { return i < first ? i : lo + i - first; }
};

// ----------------------------------------------------------------------------------------------------------------
// Forward: a wave owns 32 queries (its columns), the workgroup 32·NW of one head, and walks the visible keys in tiles
// of BK with a running maximum and sum. The next tile's rows are in flight in registers during a tile's products.
// 64 keys at bf16: with 32, an iteration was shorter than a load's latency (dq, 16k tokens: 1105 us instead of 561);
// 256 queries a workgroup are no faster at D 128 and a quarter slower at D 64. At fp32 32 keys keep the registers for
// two waves a SIMD, and a block's products (4096 cycles at D 64) cover the latency.
// Probabilities are rounded to the storage type for the product with v (half a step each, 2^-8 in bf16, and the sum is
// of the unrounded ones). EXACT (bf16, before a gradient of the bias): what that rounding leaves over, and what the
// rounding of this leaves over, go through two more products, so that p in o, and with it D = dO·o of the unrounded
// output, is good to 2^-24 like the fp32 sums — dbias is fp32.
// ----------------------------------------------------------------------------------------------------------------
template <typename T, int D, int NW, int BK, bool BIAS, bool EXACT>
__global__ __launch_bounds__(64 * NW, NW == 1 ? 1 : 2) void fwd_kernel(const Args a) {
  using R = Row<T, D>;
  __shared__ __attribute__((aligned(16))) T Ks[BK * R::P];
  __shared__ __attribute__((aligned(16))) T Vs[BK * R::P];
  extern __shared__ float lut[];
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), hh = lane >> 5;
  const typename R::Lane ln(lane);
  const int G = a.H / a.KV, nqt = (a.S + 32 * NW - 1) / (32 * NW);
  int id = xcd_swizzle(blockIdx.x, gridDim.x);
  const int g = id % G;
  id /= G;
  const int qt = id % nqt;
  id /= nqt;
  const int kv = id % a.KV, n = id / a.KV, h = kv * G + g;
  const int64_t tok0 = (int64_t)n * a.S;
  const T* kp = (const T*)a.k + tok0 * a.ldk + kv * D;
  const T* vp = (const T*)a.v + tok0 * a.ldv + kv * D;
  const uint8_t* mask = a.mask ? a.mask + tok0 : nullptr;
  const int q0 = qt * 32 * NW, qw = q0 + 32 * w, qi = qw + (lane & 31);
  const bool real = qi < a.S && (!mask || mask[qi]);
  uint4 qf[R::NC];
  R::frags(qf, (const T*)a.q + (tok0 + qi) * a.ldq + h * D, real, hh);
  if (BIAS) fill_lut(lut, a, n / (a.N / a.C), h, tid, 64 * NW);
  const KeyTiles tiles(a, q0, 32 * NW, BK);
  const int count = __syncthreads_or(real) ? tiles.count : 0;
  const float c2 = a.scale * kLog2e;
  float m = -INFINITY, l = 0.f;
  f32x16 acc[R::DB];
#pragma unroll
  for (int db = 0; db < R::DB; ++db) acc[db] = zero16();
  Stage<T, D, BK, 64 * NW> sk, sv;
  int tok = 0;
  if (count) {
    tok = token<BK>(mask, tiles.at(0) * BK, a.S, lane);
    sk.load(kp, a.ldk, tiles.at(0) * BK, a.S - 1, tid);
    sv.load(vp, a.ldv, tiles.at(0) * BK, a.S - 1, tid);
  }
  for (int it = 0; it < count; ++it) {
    const int k0 = tiles.at(it) * BK;
    __syncthreads();
    const uint64_t bits = token_bits<BK>(tok);
    sk.store(Ks, bits, tid);
    sv.store(Vs, bits, tid);
    __syncthreads();
    if (it + 1 < count) {
      tok = token<BK>(mask, tiles.at(it + 1) * BK, a.S, lane);
      sk.load(kp, a.ldk, tiles.at(it + 1) * BK, a.S - 1, tid);
      sv.load(vp, a.ldv, tiles.at(it + 1) * BK, a.S - 1, tid);
    }
    constexpr int NB = BK / 32;
    if (!block_seen(a, qw, k0, BK)) continue;
    f32x16 s[NB];
    if constexpr (NB == 2) {
      s[0] = s[1] = zero16();
      R::template rows2<true>(s[0], s[1], Ks, Ks + 32 * R::P, qf, qf, ln);
    } else {
      s[0] = R::rows(Ks, qf, ln);
    }
    if (BIAS) {
      if (qw - k0 - (BK - 1) < a.maxd) {
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          const float* at = lut + kLutOff + qi - k0 - 32 * b - 4 * hh;
#pragma unroll
          for (int r = 0; r < 16; ++r) s[b][r] = fmaf(s[b][r], c2, at[-kappa(r)]);
        }
      } else {
        const float far = lut[lut_size(a.maxd) - 1];
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
          for (int r = 0; r < 16; ++r) s[b][r] = fmaf(s[b][r], c2, far);
      }
    }
    if (!block_whole(a, qw, k0, BK)) {
      const int d = qi - k0 - 4 * hh;              // of the lane's first key; the window is 0 <= distance < W
      if (k0 < a.sinks) {
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const int key = 32 * b + kappa(r);
            const bool see = d >= key && (d - key < a.W || k0 + 4 * hh + key < a.sinks);
            s[b][r] = see ? s[b][r] : -INFINITY;
          }
      } else {
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
          for (int r = 0; r < 16; ++r)
            s[b][r] = (uint32_t)(d - 32 * b - kappa(r)) < (uint32_t)a.W ? s[b][r] : -INFINITY;
      }
    }
    if (bits != ~0ull >> (64 - BK)) {
      const uint64_t mine = bits >> (4 * hh);
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int r = 0; r < 16; ++r) s[b][r] = (mine >> (32 * b + kappa(r))) & 1 ? s[b][r] : -INFINITY;
    }
    float mt = -INFINITY;
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int r = 0; r < 16; ++r) mt = fmaxf(mt, s[b][r]);
    mt = half_max(mt);
    if (!BIAS) mt *= c2;
    if (__any(mt > m + kGrow)) {
      const float mn = fmaxf(m, mt), al = __builtin_amdgcn_exp2f(m - mn);   // m = −inf: 0 (mn is finite or the row is NaN)
      const float x = mn == -INFINITY ? 1.f : al;
      l *= x;
#pragma unroll
      for (int db = 0; db < R::DB; ++db)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[db][r] *= x;
      m = mn;
    }
    const float mu = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      typename R::Cols vt;
      vt.read(Vs + 32 * b * R::P, ln);
      float p[16];
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        p[r] = __builtin_amdgcn_exp2f(BIAS ? s[b][r] - mu : fmaf(s[b][r], c2, -mu));
        l += p[r];
      }
      vt.mul(acc, p, ln);
      if (EXACT) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
#pragma unroll
          for (int r = 0; r < 16; ++r) p[r] = Elem<T>::left(p[r]);
          vt.mul(acc, p, ln);
        }
      }
    }
  }
#pragma unroll
  for (int db = 0; db < R::DB; ++db) settle(acc[db]);
  l = half_sum(l);
  if (qi >= a.S) return;
  // A token sees itself, so l is 1 at least; l = 0 are scores that are all −inf, and 0 · (1 / 0) is the NaN that the
  // softmax of such a row is. A NaN in l is one in every column.
  const float inv = 1.f / l;
  const int64_t at = (tok0 + qi) * (int64_t)(a.H * D) + h * D + 4 * hh;
#pragma unroll
  for (int db = 0; db < R::DB; ++db)
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      float x[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = real ? acc[db][4 * c + j] * inv : 0.f;
      Elem<T>::store4((T*)a.o + at + 32 * db + 8 * c, x[0], x[1], x[2], x[3]);
      if (sizeof(T) == 2 && a.o32) Elem<float>::store4(a.o32 + at + 32 * db + 8 * c, x[0], x[1], x[2], x[3]);
    }
  if (a.lse && hh == 0) {
    const int64_t row = ((int64_t)n * a.H + h) * a.S + qi, all = (int64_t)a.N * a.H * a.S;
    const float ll = __builtin_amdgcn_logf(l);
    if (BIAS) {      // apart: next to a bias of the lowest value the logarithm would be lost
      a.lse[row] = real ? m : 0.f;
      a.lse[all + row] = real ? ll : INFINITY;
    } else {
      a.lse[row] = real ? m + ll : INFINITY;
    }
  }
}

// ----------------------------------------------------------------------------------------------------------------
// Backward, dq (and D, dbias): the forward's walk. D_i = dO_i·o_i takes the forward's output as it was before its
// rounding to bf16: with the rounded one the rows of dS would not sum to zero, half as far off as by dS's own rounding.
// dbias: dS is summed per distance, in one order whatever the launch: a 32×32 block goes to LDS skewed by its row, so
// that a column holds one distance, and a lane adds up a column and adds it to the wave's own bin of that distance;
// blocks whose distances all lie in the last bucket are summed in registers.
// ----------------------------------------------------------------------------------------------------------------
template <typename T, int D, int NW, int BK, bool BIAS, bool DBIAS>
__global__ __launch_bounds__(64 * NW, NW == 1 || D * sizeof(T) > 256 ? 1 : 2) void dq_kernel(const Args a) {
  using R = Row<T, D>;
  __shared__ __attribute__((aligned(16))) T Ks[BK * R::P];
  __shared__ __attribute__((aligned(16))) T Vs[BK * R::P];
  __shared__ float skew[DBIAS ? NW * 2048 : 1];
  __shared__ float fars[NW];
  extern __shared__ float lut[];                 // BIAS: lut; DBIAS: then NW × (maxd + kBinPad) bins
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), hh = lane >> 5;
  const typename R::Lane ln(lane);
  const int G = a.H / a.KV, nqt = (a.S + 32 * NW - 1) / (32 * NW);
  int id = xcd_swizzle(blockIdx.x, gridDim.x);
  const int g = id % G;
  id /= G;
  const int qt = id % nqt;
  id /= nqt;
  const int kv = id % a.KV, n = id / a.KV, h = kv * G + g;
  const int64_t tok0 = (int64_t)n * a.S;
  const T* kp = (const T*)a.k + tok0 * a.ldk + kv * D;
  const T* vp = (const T*)a.v + tok0 * a.ldv + kv * D;
  const uint8_t* mask = a.mask ? a.mask + tok0 : nullptr;
  const int q0 = qt * 32 * NW, qw = q0 + 32 * w, qi = qw + (lane & 31);
  const bool real = qi < a.S && (!mask || mask[qi]);
  const int nbin = a.maxd + kBinPad;
  float* bins = lut + lut_size(a.maxd) + w * nbin;
  float* sk_w = skew + (DBIAS ? w * 2048 : 0);
  uint4 qf[R::NC], df[R::NC];
  R::frags(qf, (const T*)a.q + (tok0 + qi) * a.ldq + h * D, real, hh);
  R::frags(df, (const T*)a.dout + (tok0 + qi) * a.lddo + h * D, real, hh);
  float Dq = 0.f, L = BIAS ? 0.f : INFINITY, ll = INFINITY;      // BIAS: the maximum and the sum's logarithm
  if (real) {
    const float* op = a.o32 + (tok0 + qi) * (int64_t)(a.H * D) + h * D;
#pragma unroll
    for (int c = 0; c < R::NC; ++c) Dq = Elem<T>::dot(df[c], op + (2 * c + hh) * R::E, Dq);
    const int64_t row = ((int64_t)n * a.H + h) * a.S + qi;
    L = a.lse[row];
    if (BIAS) ll = a.lse[(int64_t)a.N * a.H * a.S + row];
  }
  Dq = half_sum(Dq);
  if (qi < a.S && hh == 0) a.dsum[((int64_t)n * a.H + h) * a.S + qi] = Dq;
  if (BIAS) {
    fill_lut(lut, a, n / (a.N / a.C), h, tid, 64 * NW);
  }
  if (DBIAS) {
    for (int i = lane; i < nbin; i += 64) bins[i] = 0.f;
    for (int i = lane; i < 2048; i += 64) sk_w[i] = 0.f;
  }
  float far = 0.f;
  const bool all_real = __all(real);
  const KeyTiles tiles(a, q0, 32 * NW, BK);
  const int count = __syncthreads_or(real) ? tiles.count : 0;
  const float c2 = a.scale * kLog2e;
  f32x16 acc[R::DB];
#pragma unroll
  for (int db = 0; db < R::DB; ++db) acc[db] = zero16();
  Stage<T, D, BK, 64 * NW> sk, sv;
  int tok = 0;
  if (count) {
    tok = token<BK>(mask, tiles.at(0) * BK, a.S, lane);
    sk.load(kp, a.ldk, tiles.at(0) * BK, a.S - 1, tid);
    sv.load(vp, a.ldv, tiles.at(0) * BK, a.S - 1, tid);
  }
  for (int it = 0; it < count; ++it) {
    const int k0 = tiles.at(it) * BK;
    __syncthreads();
    const uint64_t bits = token_bits<BK>(tok);
    sk.store(Ks, bits, tid);
    sv.store(Vs, bits, tid);
    __syncthreads();
    if (it + 1 < count) {
      tok = token<BK>(mask, tiles.at(it + 1) * BK, a.S, lane);
      sk.load(kp, a.ldk, tiles.at(it + 1) * BK, a.S - 1, tid);
      sv.load(vp, a.ldv, tiles.at(it + 1) * BK, a.S - 1, tid);
    }
    if (!block_seen(a, qw, k0, BK)) continue;
    const bool whole = block_whole(a, qw, k0, BK);
#pragma unroll
    for (int sub = 0; sub < BK / 32; ++sub) {
      const int kb = k0 + 32 * sub;
      if (!block_seen(a, qw, kb, 32)) continue;
      f32x16 s = zero16(), dp = zero16();
      R::template rows2<D * sizeof(T) <= 128>(s, dp, Ks + 32 * sub * R::P, Vs + 32 * sub * R::P, qf, df, ln);
      const bool near = BIAS && qw - kb - 31 < a.maxd;
      if (BIAS) {
        if (near) {
          const float* at = lut + kLutOff + qi - kb - 4 * hh;
#pragma unroll
          for (int r = 0; r < 16; ++r) s[r] = fmaf(s[r], c2, at[-kappa(r)]) - L - ll;
        } else {
          const float b = lut[lut_size(a.maxd) - 1];
#pragma unroll
          for (int r = 0; r < 16; ++r) s[r] = fmaf(s[r], c2, b) - L - ll;
        }
      } else {
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = fmaf(s[r], c2, -L);
      }
      float ds[16];
#pragma unroll
      for (int r = 0; r < 16; ++r) ds[r] = __builtin_amdgcn_exp2f(s[r]) * (dp[r] - Dq);
      if (!whole) {
        const int d = qi - kb - 4 * hh;
        if (kb < a.sinks) {
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const bool see = d >= kappa(r) && (d - kappa(r) < a.W || kb + 4 * hh + kappa(r) < a.sinks);
            ds[r] = see ? ds[r] : 0.f;
          }
        } else {
#pragma unroll
          for (int r = 0; r < 16; ++r) ds[r] = (uint32_t)(d - kappa(r)) < (uint32_t)a.W ? ds[r] : 0.f;
        }
      }
      if (bits != ~0ull >> (64 - BK)) {
        const uint32_t mine = (uint32_t)(bits >> (32 * sub)) >> (4 * hh);
#pragma unroll
        for (int r = 0; r < 16; ++r) ds[r] = (mine >> kappa(r)) & 1 ? ds[r] : 0.f;
      }
      if (DBIAS && !all_real) {      // e^−inf is 0, but for a bias that is not finite where only padding looks
#pragma unroll
        for (int r = 0; r < 16; ++r) ds[r] = real ? ds[r] : 0.f;
      }
      typename R::Cols kt;      // read ahead of ds it would cost a wave of occupancy (D 64) or spill (D 128)
      kt.read(Ks + 32 * sub * R::P, ln);
      kt.mul(acc, ds, ln);
      if (DBIAS) {
        if (near) {
          float* at = sk_w + (lane & 31) * 65 + 31 - 4 * hh;       // row i, column i − key + 31
#pragma unroll
          for (int r = 0; r < 16; ++r) at[-kappa(r)] = ds[r];
          __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
          __builtin_amdgcn_wave_barrier();
          float sum = 0.f;
#pragma unroll
          for (int i = 0; i < 32; ++i) sum += sk_w[i * 64 + lane];
          const int d = qw - kb + lane - 31;
          if (lane < 63 && d >= 0) bins[d] += sum;
          __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
          __builtin_amdgcn_wave_barrier();
        } else {
#pragma unroll
          for (int r = 0; r < 16; ++r) far += ds[r];
        }
      }
    }
  }
#pragma unroll
  for (int db = 0; db < R::DB; ++db) settle(acc[db]);
  if (qi < a.S) {
    T* out = (T*)a.dq + (tok0 + qi) * (int64_t)(a.H * D) + h * D + 4 * hh;
#pragma unroll
    for (int db = 0; db < R::DB; ++db)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        float x[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = real ? acc[db][4 * c + j] * a.scale : 0.f;
        Elem<T>::store4(out + 32 * db + 8 * c, x[0], x[1], x[2], x[3]);
      }
  }
  if (DBIAS) {
    far = wave_sum(far);
    if (lane == 0) fars[w] = far;
    __syncthreads();
    float* out = a.bpart + (((int64_t)n * a.H + h) * nqt + qt) * a.NB;
    for (int b = w; b < a.NB; b += NW) {
      const int end = b + 1 < a.NB ? a.start[b + 1] : nbin;
      float sum = 0.f;
      for (int d = a.start[b] + lane; d < end; d += 64)
#pragma unroll
        for (int i = 0; i < NW; ++i) sum += lut[lut_size(a.maxd) + i * nbin + d];
      sum = wave_sum(sum);
      if (b == a.NB - 1)
#pragma unroll
        for (int i = 0; i < NW; ++i) sum += fars[i];
      if (lane == 0) out[b] = sum;
    }
  }
}

// ----------------------------------------------------------------------------------------------------------------
// Backward, dk and dv: a wave owns 32 keys (its columns), the workgroup 32·NW of one kv head; it walks the queries
// that see them through the window, for every query head of the kv head. The first workgroups are the sink pass: what
// the sinks get from queries beyond the window, a chunk of queries each, as partial sums that finish_kernel adds up in
// order (the sinks' own rows of the window pass among them). There the blocks of a tile of queries go to as many waves,
// each with the same keys and a partial sum of its own (one wave taking all: 1041 instead of 980 us at 16k tokens).
// ----------------------------------------------------------------------------------------------------------------
template <typename T, int D, int NW, int BQ, bool BIAS>
__global__ __launch_bounds__(64 * NW, D * sizeof(T) > 128 ? 1 : 2) void dkv_kernel(const Args a) {
  using R = Row<T, D>;
  __shared__ __attribute__((aligned(16))) T Qs[BQ * R::P];
  __shared__ __attribute__((aligned(16))) T Os[BQ * R::P];
  __shared__ __attribute__((aligned(16))) float Ls[BQ], Ds[BQ], LLs[BIAS ? BQ : 4];      // LLs: see fwd_kernel
  extern __shared__ float lut[];
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), hh = lane >> 5;
  const typename R::Lane ln(lane);
  const int G = a.H / a.KV, nkt = (a.S + 32 * NW - 1) / (32 * NW);
  const int nsink = a.nchunk * a.N * a.KV;
  const bool sink = (int)blockIdx.x < nsink;
  int id = sink ? (int)blockIdx.x : xcd_swizzle(blockIdx.x - nsink, gridDim.x - nsink);
  const int kt = sink ? 0 : id % nkt, chunk = sink ? id % a.nchunk : 0;
  id /= sink ? a.nchunk : nkt;
  const int kv = id % a.KV, n = id / a.KV;
  const int64_t tok0 = (int64_t)n * a.S;
  const uint8_t* mask = a.mask ? a.mask + tok0 : nullptr;
  constexpr int kParts = BQ / 32;
  const int nkb = sink ? (a.sinks + 31) / 32 : NW, part = w / nkb;        // blocks of keys (sinks: ≤ 2); the wave's queries
  const int k0 = kt * 32 * NW, kw = k0 + 32 * (w % nkb), kj = kw + (lane & 31);
  const bool real = kj < a.S && (!mask || mask[kj]) && (!sink || kj < a.sinks);
  uint4 kf[R::NC], vf[R::NC];
  R::frags(kf, (const T*)a.k + (tok0 + kj) * a.ldk + kv * D, real, hh);
  R::frags(vf, (const T*)a.v + (tok0 + kj) * a.ldv + kv * D, real, hh);
  // queries [qs, qe): through the window (and to the end where the sinks have no pass of their own), or a chunk beyond
  const int own = a.nchunk ? 0 : a.sinks;
  int qs, qe;
  if (sink) {
    qs = a.W + chunk * a.qchunk;
    qe = qs + a.qchunk < a.S ? qs + a.qchunk : a.S;
  } else {
    qs = k0;
    qe = k0 >= own && (int64_t)k0 + 32 * NW - 1 + a.W < a.S ? k0 + 32 * NW - 1 + a.W : a.S;
  }
  const int nt = (qe - qs + BQ - 1) / BQ;
  const int count = __syncthreads_or(real) ? nt * G : 0;
  const float c2 = a.scale * kLog2e;
  f32x16 ak[R::DB], av[R::DB];
#pragma unroll
  for (int db = 0; db < R::DB; ++db) ak[db] = av[db] = zero16();
  Stage<T, D, BQ, 64 * NW> sq, so;
  int tok = 0;
  float sl = 0.f, sd = 0.f, sll = 0.f;             // threads below BQ: the row's statistics
  auto load = [&](int it) {
    const int h = kv * G + it / nt, q0 = qs + (it % nt) * BQ;
    tok = token<BQ>(mask, q0, qe, lane);
    sq.load((const T*)a.q + tok0 * a.ldq + h * D, a.ldq, q0, qe - 1, tid);
    so.load((const T*)a.dout + tok0 * a.lddo + h * D, a.lddo, q0, qe - 1, tid);
    if (tid < BQ) {
      const int64_t at = ((int64_t)n * a.H + h) * a.S + q0 + tid;
      sl = q0 + tid < qe ? a.lse[at] : BIAS ? 0.f : INFINITY;      // a masked query's (sum) is +inf, its D zero
      if (BIAS) sll = q0 + tid < qe ? a.lse[(int64_t)a.N * a.H * a.S + at] : INFINITY;
      sd = q0 + tid < qe ? a.dsum[at] : 0.f;
    }
  };
  if (count) load(0);
  for (int it = 0; it < count; ++it) {
    const int q0 = qs + (it % nt) * BQ;
    __syncthreads();
    const uint64_t bits = token_bits<BQ>(tok);
    sq.store(Qs, bits, tid);
    so.store(Os, bits, tid);
    if (tid < BQ) {
      Ls[tid] = sl;
      if (BIAS) LLs[tid] = sll;
      Ds[tid] = sd;
    }
    if (BIAS && it % nt == 0) fill_lut(lut, a, n / (a.N / a.C), kv * G + it / nt, tid, 64 * NW);
    __syncthreads();
    if (it + 1 < count) load(it + 1);
    const bool whole = sink ? q0 - kw - 31 >= a.W : q0 >= kw + 31 && (q0 + BQ - 1 - kw < a.W || kw + 31 < own);
#pragma unroll
    for (int sub = 0; sub < BQ / 32; ++sub) {
      const int qb = q0 + 32 * sub;
      if (kw >= a.S || qb >= qe || qb + 31 < kw || (sink && part != sub)) continue;
      if (sink ? (kw >= a.sinks || qb + 31 - kw < a.W) : (qb - kw - 31 >= a.W && kw >= own)) continue;
      f32x16 s = zero16(), dp = zero16();
      R::template rows2<true>(s, dp, Qs + 32 * sub * R::P, Os + 32 * sub * R::P, kf, vf, ln);
      typename R::Cols ot, qt;
      ot.read(Os + 32 * sub * R::P, ln);
      if (BIAS) {
        if (qb - kw - 31 < a.maxd) {
          const float* at = lut + kLutOff + qb - kj + 4 * hh;
#pragma unroll
          for (int r = 0; r < 16; ++r) s[r] = fmaf(s[r], c2, at[kappa(r)]);
        } else {
          const float far = lut[lut_size(a.maxd) - 1];
#pragma unroll
          for (int r = 0; r < 16; ++r) s[r] = fmaf(s[r], c2, far);
        }
      }
      float p[16], ds[16];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const float4 L4 = *reinterpret_cast<const float4*>(Ls + 32 * sub + 8 * c + 4 * hh);
        const float4 D4 = *reinterpret_cast<const float4*>(Ds + 32 * sub + 8 * c + 4 * hh);
        const float Lr[4] = {L4.x, L4.y, L4.z, L4.w}, Dr[4] = {D4.x, D4.y, D4.z, D4.w};
        float ll[4] = {0.f, 0.f, 0.f, 0.f};
        if (BIAS) {
          const float4 x = *reinterpret_cast<const float4*>(LLs + 32 * sub + 8 * c + 4 * hh);
          ll[0] = x.x; ll[1] = x.y; ll[2] = x.z; ll[3] = x.w;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int r = 4 * c + j;
          p[r] = __builtin_amdgcn_exp2f(BIAS ? s[r] - Lr[j] - ll[j] : fmaf(s[r], c2, -Lr[j]));
          ds[r] = p[r] * (dp[r] - Dr[j]);
        }
      }
      if (!whole) {
        const int d = qb + 4 * hh - kj;
        if (sink || kw < own) {
          const int least = sink ? a.W : 0, most = !sink && kj >= own ? a.W : 0x7fffffff;
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const bool see = d + kappa(r) >= least && d + kappa(r) < most;
            p[r] = see ? p[r] : 0.f;
            ds[r] = see ? ds[r] : 0.f;
          }
        } else {
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const bool see = (uint32_t)(d + kappa(r)) < (uint32_t)a.W;
            p[r] = see ? p[r] : 0.f;
            ds[r] = see ? ds[r] : 0.f;
          }
        }
      }
      if (BIAS && bits != ~0ull >> (64 - BQ)) {      // queries that are no token, as in dq_kernel
        const uint32_t mine = (uint32_t)(bits >> (32 * sub)) >> (4 * hh);
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          p[r] = (mine >> kappa(r)) & 1 ? p[r] : 0.f;
          ds[r] = (mine >> kappa(r)) & 1 ? ds[r] : 0.f;
        }
      }
      qt.read(Qs + 32 * sub * R::P, ln);
      ot.mul(av, p, ln);
      qt.mul(ak, ds, ln);
    }
  }
#pragma unroll
  for (int db = 0; db < R::DB; ++db) settle(ak[db], av[db]);
  if (kj >= a.S || (sink && (kj >= a.sinks || part >= kParts))) return;
  if (!real) {                                   // a column of no token: whatever its sums are, it has no gradient
#pragma unroll
    for (int db = 0; db < R::DB; ++db) ak[db] = av[db] = zero16();
  }
  if (a.nchunk && kj < a.sinks) {
    const int slot = sink ? 1 + chunk * kParts + part : 0;
    float* pk = a.part + ((((int64_t)n * a.KV + kv) * a.nslot + slot) * 2 * a.sinks + kj) * D + 4 * hh;
    float* pv = pk + (int64_t)a.sinks * D;
#pragma unroll
    for (int db = 0; db < R::DB; ++db)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        Elem<float>::store4(pk + 32 * db + 8 * c, ak[db][4 * c] * a.scale, ak[db][4 * c + 1] * a.scale,
                            ak[db][4 * c + 2] * a.scale, ak[db][4 * c + 3] * a.scale);
        Elem<float>::store4(pv + 32 * db + 8 * c, av[db][4 * c], av[db][4 * c + 1], av[db][4 * c + 2],
                            av[db][4 * c + 3]);
      }
    return;
  }
  const int64_t at = (tok0 + kj) * (int64_t)(a.KV * D) + kv * D + 4 * hh;
#pragma unroll
  for (int db = 0; db < R::DB; ++db)
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      Elem<T>::store4((T*)a.dk + at + 32 * db + 8 * c, ak[db][4 * c] * a.scale, ak[db][4 * c + 1] * a.scale,
                      ak[db][4 * c + 2] * a.scale, ak[db][4 * c + 3] * a.scale);
      Elem<T>::store4((T*)a.dv + at + 32 * db + 8 * c, av[db][4 * c], av[db][4 * c + 1], av[db][4 * c + 2],
                      av[db][4 * c + 3]);
    }
}

// The partial sums' last step, in a fixed order. Workgroups [0, C·H): dbias of a client and head over its sequences and
// query tiles (in fp64: dS sums to zero over a row, so buckets are small next to their terms); the others: the sinks'
// rows of dk and dv.
template <typename T>
__global__ __launch_bounds__(256) void finish_kernel(const Args a, int D, int nqt) {
  __shared__ double red[256];
  const int nb = a.dbias ? a.C * a.H : 0;
  if ((int)blockIdx.x < nb) {
    const int c = blockIdx.x / a.H, h = blockIdx.x % a.H, per = a.N / a.C;
    int wide = 1;
    while (wide < a.NB) wide *= 2;
    const int b = threadIdx.x % wide, row = threadIdx.x / wide, rows = 256 / wide;
    double sum = 0.;
    if (b < a.NB)
      for (int64_t i = row; i < (int64_t)per * nqt; i += rows)
        sum += a.bpart[((((int64_t)c * per + i / nqt) * a.H + h) * nqt + i % nqt) * a.NB + b];
    red[threadIdx.x] = sum;
    __syncthreads();
    if (row == 0 && b < a.NB) {
      for (int i = 1; i < rows; ++i) sum += red[i * wide + b];
      a.dbias[((int64_t)c * a.H + h) * a.NB + b] = (float)sum;
    }
    return;
  }
  const int64_t e = ((int64_t)blockIdx.x - nb) * 256 + threadIdx.x;       // [n][kv][dk | dv][sink][D / 4]
  const int64_t one = (int64_t)2 * a.sinks * (D / 4);
  if (e >= (int64_t)a.N * a.KV * one) return;
  const int64_t head = e / one;
  const int in = (int)(e % one);
  const float4* p = reinterpret_cast<const float4*>(a.part) + head * a.nslot * one + in;
  float4 s = p[0];
#pragma unroll 8
  for (int i = 1; i < a.nslot; ++i) {
    const float4 x = p[i * one];
    s.x += x.x; s.y += x.y; s.z += x.z; s.w += x.w;
  }
  const int which = in / (a.sinks * (D / 4)), rest = in % (a.sinks * (D / 4)), j = rest / (D / 4);
  const int64_t n = head / a.KV, kv = head % a.KV;
  T* out = (T*)(which ? a.dv : a.dk) + (n * a.S + j) * (a.KV * D) + kv * D + 4 * (rest % (D / 4));
  if (j < a.S) Elem<T>::store4(out, s.x, s.y, s.z, s.w);
}

// ----------------------------------------------------------------------------------------------------------------
// One new token per sequence over a ring cache [batch][sinks + W][KV·D]: slot s < sinks holds token s, slot
// sinks + (t − sinks) mod W token t. The query heads of a kv head are the columns; a wave reads 32 slots at a time
// into an LDS tile of its own (the next 32 in flight in registers), keeps its own softmax, and the workgroup's waves,
// then the splits of the cache, are joined by their maxima. The new token's rows are taken from the arguments, and
// written into their slot by the workgroup that reads them.
// ----------------------------------------------------------------------------------------------------------------
struct StepArgs {
  const void *q, *k, *v;
  void *kc, *vc, *o;
  const int* pos;
  const float* bias;
  float *pacc, *pml;             // splits > 1: [B·H][splits][D], [B·H][splits][2]
  int64_t ldq, ldk, ldv;
  int B, H, KV, C, W, sinks, NB, maxd, splits, per;   // per: slots of a split, a multiple of 32
  float scale;
  int start[kMaxBuckets];
};

constexpr int kRowsInCache = -1;      // what fa_window_step returns, nothing launched, where its rows lie in a cache

// the age (pos − token) of the token in a slot, −1 if there is none; cur = the new token's slot
__device__ __forceinline__ int slot_age(int s, int pos, int sinks, int W, int cur) {
  if (pos < 0) return -1;
  if (s < sinks) return s <= pos ? pos - s : -1;
  if (pos < sinks) return -1;
  int age = cur - s;
  if (age < 0) age += W;
  return pos - age >= sinks ? age : -1;
}

template <typename T, int D, int NW>
__global__ __launch_bounds__(64 * NW, D * sizeof(T) > 256 ? 1 : 2) void step_kernel(const StepArgs a) {
  using R = Row<T, D>;
  __shared__ __attribute__((aligned(16))) T tiles[NW][2][32 * R::P];
  __shared__ float ml[NW][2][32];
  extern __shared__ float tab[];                  // bias: [heads of the group][NB], then bytes: bucket of a distance
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), hh = lane >> 5;
  const typename R::Lane ln(lane);
  const int G = a.H / a.KV, groups = (G + 31) / 32;
  int id = blockIdx.x;
  const int split = id % a.splits;
  id /= a.splits;
  const int grp = id % groups;
  id /= groups;
  const int kv = id % a.KV, b = id / a.KV;
  const int n = a.sinks + a.W, pos = a.pos[b];
  const int cur = pos < a.sinks ? pos : a.sinks + (pos - a.sinks) % a.W;
  const int g = grp * 32 + (lane & 31), h = kv * G + g;
  const bool real = g < G;
  uint8_t* of = reinterpret_cast<uint8_t*>(tab + 32 * a.NB);
  if (a.bias) {
    const float* src = a.bias + ((int64_t)(b / (a.B / a.C)) * a.H + kv * G + grp * 32) * a.NB;
    const int have = (G - grp * 32 < 32 ? G - grp * 32 : 32) * a.NB;
    for (int i = tid; i < 32 * a.NB; i += 64 * NW) tab[i] = i < have ? log2_bias(src[i]) : 0.f;
    for (int d = tid; d <= a.maxd; d += 64 * NW) {
      int x = 0;
      for (int i = 1; i < a.NB; ++i) x += d >= a.start[i] ? 1 : 0;
      of[d] = (uint8_t)x;
    }
  }
  __syncthreads();
  uint4 qf[R::NC];
  R::frags(qf, (const T*)a.q + b * a.ldq + (int64_t)h * D, real, hh);
  T* kc = (T*)a.kc + (int64_t)b * n * a.KV * D + kv * D;
  T* vc = (T*)a.vc + (int64_t)b * n * a.KV * D + kv * D;
  const T* kn = (const T*)a.k + b * a.ldk + kv * D;
  const T* vn = (const T*)a.v + b * a.ldv + kv * D;
  const int ld = a.KV * D;
  const int s0 = split * a.per, s1 = s0 + a.per < n ? s0 + a.per : n;
  constexpr int NI = 32 * R::U / 64;
  uint4 rk[NI], rv[NI];
  const bool full = pos >= n - 1;                 // every slot holds a token
  // a block of 32 slots whose rows all come from the cache
  auto plain = [&](int base) { return full && base + 32 <= s1 && (cur < base || cur >= base + 32); };
  auto load = [&](int base) {
    const int row = lane / R::U, c = (lane % R::U) * R::E;
    if (plain(base)) {
      const T *pk = kc + (int64_t)(base + row) * ld + c, *pv = vc + (int64_t)(base + row) * ld + c;
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        rk[i] = *reinterpret_cast<const uint4*>(pk + (int64_t)(i * (64 / R::U)) * ld);
        rv[i] = *reinterpret_cast<const uint4*>(pv + (int64_t)(i * (64 / R::U)) * ld);
      }
      return;
    }
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int s = base + row + i * (64 / R::U);
      rk[i] = rv[i] = make_uint4(0, 0, 0, 0);
      if (s >= s1 || slot_age(s, pos, a.sinks, a.W, cur) < 0) continue;
      if (s == cur) {
        rk[i] = *reinterpret_cast<const uint4*>(kn + c);
        rv[i] = *reinterpret_cast<const uint4*>(vn + c);
        if (grp == 0) {
          *reinterpret_cast<uint4*>(kc + (int64_t)s * ld + c) = rk[i];
          *reinterpret_cast<uint4*>(vc + (int64_t)s * ld + c) = rv[i];
        }
      } else {
        rk[i] = *reinterpret_cast<const uint4*>(kc + (int64_t)s * ld + c);
        rv[i] = *reinterpret_cast<const uint4*>(vc + (int64_t)s * ld + c);
      }
    }
  };
  const float c2 = a.scale * kLog2e;
  const float far = a.bias ? tab[(lane & 31) * a.NB + a.NB - 1] : 0.f;
  float m = -INFINITY, l = 0.f;
  f32x16 acc[R::DB];
#pragma unroll
  for (int db = 0; db < R::DB; ++db) acc[db] = zero16();
  T *Ks = tiles[w][0], *Vs = tiles[w][1];
  if (pos >= 0) {
    int base = s0 + 32 * w;
    if (base < s1) load(base);
    for (; base < s1; base += 32 * NW) {
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const int u = lane + 64 * i;
        *reinterpret_cast<uint4*>(Ks + R::at(u / R::U, u % R::U)) = rk[i];
        *reinterpret_cast<uint4*>(Vs + R::at(u / R::U, u % R::U)) = rv[i];
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
      if (base + 32 * NW < s1) load(base + 32 * NW);
      f32x16 s = R::rows(Ks, qf, ln);
      // whole blocks of the ring whose tokens are all max_distance old or older have one bias
      const int last = base + 31, age = last < cur ? cur - last : a.W + cur - last;
      if (plain(base) && (!a.bias || (base >= a.sinks && age >= a.maxd))) {
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = fmaf(s[r], c2, far);
      } else {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int slot = base + kappa(r) + 4 * hh;
          const int age = slot < s1 ? slot_age(slot, pos, a.sinks, a.W, cur) : -1;
          float x = s[r] * c2;
          if (a.bias && age >= 0) x += tab[(lane & 31) * a.NB + of[age < a.maxd ? age : a.maxd]];
          s[r] = age >= 0 ? x : -INFINITY;
        }
      }
      float mt = s[0];
#pragma unroll
      for (int r = 1; r < 16; ++r) mt = fmaxf(mt, s[r]);
      mt = half_max(mt);
      if (__any(mt > m + kGrow)) {
        const float mn = fmaxf(m, mt), x = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - mn);
        l *= x;
#pragma unroll
        for (int db = 0; db < R::DB; ++db)
#pragma unroll
          for (int r = 0; r < 16; ++r) acc[db][r] *= x;
        m = mn;
      }
      const float mu = m == -INFINITY ? 0.f : m;
      float p[16];
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        p[r] = __builtin_amdgcn_exp2f(s[r] - mu);
        l += p[r];
      }
      typename R::Cols vt;
      vt.read(Vs, ln);
      vt.mul(acc, p, ln);
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
    }
  }
#pragma unroll
  for (int db = 0; db < R::DB; ++db) settle(acc[db]);
  l = half_sum(l);
  if (hh == 0) {
    ml[w][0][lane] = m;
    ml[w][1][lane] = l;
  }
  // the waves' sums, scaled to the common maximum, through their own tiles
  float* mine = reinterpret_cast<float*>(tiles[w]);
  static_assert(2 * 32 * R::P * sizeof(T) >= 32 * D * sizeof(float), "the tiles hold a wave's sums");
  __syncthreads();
  float M = -INFINITY, L = 0.f;
#pragma unroll
  for (int i = 0; i < NW; ++i) M = fmaxf(M, ml[i][0][lane & 31]);
  const float Mu = M == -INFINITY ? 0.f : M;
#pragma unroll
  for (int i = 0; i < NW; ++i) L += ml[i][1][lane & 31] * __builtin_amdgcn_exp2f(ml[i][0][lane & 31] - Mu);
  const float al = __builtin_amdgcn_exp2f(m - Mu);
#pragma unroll
  for (int db = 0; db < R::DB; ++db)
#pragma unroll
    for (int r = 0; r < 16; ++r)
      if (real) mine[(lane & 31) * D + 32 * db + kappa(r) + 4 * hh] = acc[db][r] * al;
  __syncthreads();
  // a column (head) of D sums at a time
  const int heads = G - grp * 32 < 32 ? G - grp * 32 : 32;
  for (int e = tid * 4; e < heads * D; e += 64 * NW * 4) {
    float4 s = *reinterpret_cast<const float4*>(reinterpret_cast<float*>(tiles[0]) + e);
#pragma unroll
    for (int i = 1; i < NW; ++i) {
      const float4 x = *reinterpret_cast<const float4*>(reinterpret_cast<float*>(tiles[i]) + e);
      s.x += x.x; s.y += x.y; s.z += x.z; s.w += x.w;
    }
    const int hd = e / D, d = e % D;
    const int64_t row = (int64_t)b * a.H + kv * G + grp * 32 + hd;
    if (a.splits > 1) {
      Elem<float>::store4(a.pacc + (row * a.splits + split) * D + d, s.x, s.y, s.z, s.w);
    } else {
      float Mh = -INFINITY, Lh = 0.f;
#pragma unroll
      for (int i = 0; i < NW; ++i) Mh = fmaxf(Mh, ml[i][0][hd]);
#pragma unroll
      for (int i = 0; i < NW; ++i)
        Lh += ml[i][1][hd] * __builtin_amdgcn_exp2f(ml[i][0][hd] - (Mh == -INFINITY ? 0.f : Mh));
      const float inv = pos < 0 ? 0.f : 1.f / Lh;     // scores that are all −inf: 0 · (1 / 0), NaN as in fwd_kernel
      Elem<T>::store4((T*)a.o + row * D + d, s.x * inv, s.y * inv, s.z * inv, s.w * inv);
    }
  }
  if (a.splits > 1 && w == 0 && lane < heads) {
    float* out = a.pml + (((int64_t)b * a.H + kv * G + grp * 32 + lane) * a.splits + split) * 2;
    out[0] = M;
    out[1] = L;
  }
}

// joins the splits of a (sequence, head): one wave each
template <typename T, int D>
__global__ __launch_bounds__(64) void step_join_kernel(const StepArgs a) {
  const int64_t row = blockIdx.x;
  const int lane = threadIdx.x;
  float M = -INFINITY;
  for (int i = lane; i < a.splits; i += 64) M = fmaxf(M, a.pml[(row * a.splits + i) * 2]);
  M = wave_max(M);
  const float Mu = M == -INFINITY ? 0.f : M;
  float L = 0.f;
  for (int i = lane; i < a.splits; i += 64)
    L += a.pml[(row * a.splits + i) * 2 + 1] * __builtin_amdgcn_exp2f(a.pml[(row * a.splits + i) * 2] - Mu);
  L = wave_sum(L);
  const float inv = a.pos[row / a.H] < 0 ? 0.f : 1.f / L;
  for (int d = lane; d < D; d += 64) {
    float s = 0.f;
    for (int i = 0; i < a.splits; ++i)
      s += a.pacc[(row * a.splits + i) * D + d] * __builtin_amdgcn_exp2f(a.pml[(row * a.splits + i) * 2] - Mu);
    if constexpr (sizeof(T) == 2) ((T*)a.o)[row * D + d] = f32_to_bf16(s * inv);
    else ((T*)a.o)[row * D + d] = s * inv;
  }
}

// a prompt's rows into the cache: what the slots hold after token len − 1; slots of no token stay as they were
__global__ __launch_bounds__(256) void fill_kernel(const uint4* __restrict__ k, const uint4* __restrict__ v,
                                                   int64_t ldk, int64_t ldv, uint4* __restrict__ kc,
                                                   uint4* __restrict__ vc, const int* __restrict__ lengths, int B,
                                                   int S, int W, int sinks, int U) {
  const int n = sinks + W;
  const int64_t total = (int64_t)B * n * U;
  for (int64_t e = blockIdx.x * 256ll + threadIdx.x; e < total; e += gridDim.x * 256ll) {
    const int u = (int)(e % U), s = (int)(e / U % n), b = (int)(e / U / n);
    int len = lengths ? lengths[b] : S;
    len = len < 0 ? 0 : len > S ? S : len;
    const int pos = len - 1, cur = pos < sinks ? pos : sinks + (pos - sinks) % W;
    const int age = slot_age(s, pos, sinks, W, cur);
    if (age < 0) continue;
    const int64_t row = (int64_t)b * S + pos - age;
    kc[e] = k[row * ldk + u];
    vc[e] = v[row * ldv + u];
  }
}

template <typename T, int D, int NW, int BK> int launch_fwd_tile(const Args& a, hipStream_t st) {
  const size_t lds = a.bias ? (a.maxd + 2 * kLutOff) * sizeof(float) : 0;
  const dim3 grid((unsigned)((int64_t)a.N * a.H * ((a.S + 32 * NW - 1) / (32 * NW)))), block(64 * NW);
  if (!a.bias) hipLaunchKernelGGL((fwd_kernel<T, D, NW, BK, false, false>), grid, block, 0, st, a);
  else if (sizeof(T) == 2 && a.exact)
    hipLaunchKernelGGL((fwd_kernel<T, D, NW, BK, true, sizeof(T) == 2>), grid, block, lds, st, a);
  else hipLaunchKernelGGL((fwd_kernel<T, D, NW, BK, true, false>), grid, block, lds, st, a);
  return (int)hipGetLastError();
}

template <typename T, int D> int launch_fwd(const Args& a, hipStream_t st) {
  if (a.tile == 128) return launch_fwd_tile<T, D, 4, sizeof(T) == 2 ? 64 : 32>(a, st);
  return launch_fwd_tile<T, D, 1, 32>(a, st);
}

template <typename T, int D, int NW, int BK> int launch_dq(const Args& a, hipStream_t st) {
  const int64_t n = (int64_t)a.N * a.H * ((a.S + 32 * NW - 1) / (32 * NW));
  const size_t lut = (a.maxd + 2 * kLutOff) * sizeof(float), bins = NW * (a.maxd + kBinPad) * sizeof(float);
  const dim3 grid((unsigned)n), block(64 * NW);
  if (a.dbias) hipLaunchKernelGGL((dq_kernel<T, D, NW, BK, true, true>), grid, block, lut + bins, st, a);
  else if (a.bias) hipLaunchKernelGGL((dq_kernel<T, D, NW, BK, true, false>), grid, block, lut, st, a);
  else hipLaunchKernelGGL((dq_kernel<T, D, NW, BK, false, false>), grid, block, 0, st, a);
  return (int)hipGetLastError();
}

template <typename T, int D> int launch_bwd(const Args& a, hipStream_t st) {
  const size_t lds = a.bias ? (a.maxd + 2 * kLutOff) * sizeof(float) : 0;
  int rc;
  if (a.tile == 128) rc = launch_dq<T, D, 4, sizeof(T) == 2 ? 64 : 32>(a, st);
  else rc = launch_dq<T, D, 1, 32>(a, st);
  if (rc) return rc;
  const int64_t nsink = (int64_t)a.nchunk * a.N * a.KV;
  const int64_t n = nsink + (int64_t)a.N * a.KV * ((a.S + a.ktile - 1) / a.ktile);
  if (a.ktile == 128) {
    constexpr int BQ = sizeof(T) == 2 ? 64 : 32;
    if (a.bias) hipLaunchKernelGGL((dkv_kernel<T, D, 4, BQ, true>), dim3((unsigned)n), dim3(256), lds, st, a);
    else hipLaunchKernelGGL((dkv_kernel<T, D, 4, BQ, false>), dim3((unsigned)n), dim3(256), 0, st, a);
  } else if constexpr (D * sizeof(T) <= 256) {
    if (a.bias) hipLaunchKernelGGL((dkv_kernel<T, D, 2, 32, true>), dim3((unsigned)n), dim3(128), lds, st, a);
    else hipLaunchKernelGGL((dkv_kernel<T, D, 2, 32, false>), dim3((unsigned)n), dim3(128), 0, st, a);
  } else {
    return (int)hipErrorInvalidValue;
  }
  if ((rc = (int)hipGetLastError())) return rc;
  const int nqt = (a.S + a.tile - 1) / a.tile;
  const int64_t blocks = (a.dbias ? (int64_t)a.C * a.H : 0) +
                         (a.nchunk ? ((int64_t)a.N * a.KV * 2 * a.sinks * (D / 4) + 255) / 256 : 0);
  if (blocks) hipLaunchKernelGGL(finish_kernel<T>, dim3((unsigned)blocks), dim3(256), 0, st, a, D, nqt);
  return (int)hipGetLastError();
}

// Rows [B][ld], `width` elements of each, that share memory with a cache: the kernel would read them while it writes there
inline bool rows_in_cache(const StepArgs& a, const void* rows, int64_t ld, int64_t width, int64_t cache, int64_t e) {
  const char *p = (const char*)rows, *k = (const char*)a.kc, *v = (const char*)a.vc;
  const int64_t span = ((a.B - 1) * ld + width) * e, size = cache * e;
  return (p < k + size && p + span > k) || (p < v + size && p + span > v);
}

template <typename T, int D> int launch_step(const StepArgs& a, hipStream_t st) {
  const int64_t kv = (int64_t)a.KV * D, cache = (int64_t)a.B * (a.sinks + a.W) * kv, e = sizeof(T);
  if (rows_in_cache(a, a.q, a.ldq, (int64_t)a.H * D, cache, e) || rows_in_cache(a, a.k, a.ldk, kv, cache, e) ||
      rows_in_cache(a, a.v, a.ldv, kv, cache, e))
    return kRowsInCache;
  constexpr int NW = D * sizeof(T) > 256 ? 2 : 4;
  const size_t lds = a.bias ? 32 * a.NB * sizeof(float) + (a.maxd + 4) / 4 * 4 : 0;
  const int64_t n = (int64_t)a.B * a.KV * ((a.H / a.KV + 31) / 32) * a.splits;
  hipLaunchKernelGGL((step_kernel<T, D, NW>), dim3((unsigned)n), dim3(64 * NW), lds, st, a);
  int rc = (int)hipGetLastError();
  if (rc || a.splits == 1) return rc;
  hipLaunchKernelGGL((step_join_kernel<T, D>), dim3((unsigned)(a.B * a.H)), dim3(64), 0, st, a);
  return (int)hipGetLastError();
}

}  // namespace win

#define FA_WIN_DISPATCH(FN, A, ST)                                             \
  if (bf16 && D == 64) return win::FN<uint16_t, 64>(A, ST);                    \
  if (bf16 && D == 128) return win::FN<uint16_t, 128>(A, ST);                  \
  if (!bf16 && D == 64) return win::FN<float, 64>(A, ST);                      \
  if (!bf16 && D == 128) return win::FN<float, 128>(A, ST);                    \
  return (int)hipErrorInvalidValue;

FA_EXPORT int fa_window_fwd(const win::Args* a, int bf16, int D, hipStream_t stream) {
  FA_WIN_DISPATCH(launch_fwd, *a, stream)
}
FA_EXPORT int fa_window_bwd(const win::Args* a, int bf16, int D, hipStream_t stream) {
  FA_WIN_DISPATCH(launch_bwd, *a, stream)
}
FA_EXPORT int fa_window_step(const win::StepArgs* a, int bf16, int D, hipStream_t stream) {
  FA_WIN_DISPATCH(launch_step, *a, stream)
}
FA_EXPORT int fa_window_fill(const void* k, const void* v, int64_t ldk, int64_t ldv, void* kc, void* vc,
                             const int* lengths, int B, int S, int W, int sinks, int U, hipStream_t stream) {
  const int64_t n = (int64_t)B * (sinks + W) * U;
  hipLaunchKernelGGL(win::fill_kernel, dim3(fa_grid(n, 256, 16384)), dim3(256), 0, stream, (const uint4*)k,
                     (const uint4*)v, ldk, ldv, (uint4*)kc, (uint4*)vc, lengths, B, S, W, sinks, U);
  return (int)hipGetLastError();
}
