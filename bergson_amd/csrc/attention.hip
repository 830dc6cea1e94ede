// Causal self-attention over whole sequences, grouped heads, sequences of different lengths: forward and backward.
//
//   s_ij = scale q_i . k_j for j <= i of the same sequence,  p = softmax_j(s),  o_i = sum_j p_ij v_j
//   dp_ij = do_i . v_j,  delta_i = do_i . o_i,  ds_ij = p_ij (dp_ij - delta_i)
//   dq_i = scale sum_j ds_ij k_j,  dk_j = scale sum_i ds_ij q_i,  dv_j = sum_i p_ij do_i
//   (dk, dv also summed over the query heads that share the key/value head)
//
// Everything is built from 32 x 32 matrix instructions on operands laid out so that no score ever leaves the
// registers.  The forward pass forms S^T = K Q^T: a lane then holds one query and 16 keys of every 32, the running
// maximum, the sum and the rescaling are per lane, and the probabilities are already where the next product,
// O^T += V^T P^T, wants its second operand -- the instruction's contraction index is only a label, so the keys may
// be taken in the order the first product left them, as long as V^T is read in the same order (read_tr).
// The backward pass uses the same trick twice: one kernel walks the keys for a block of queries (dq), one walks the
// queries for a block of keys (dk, dv).  Two walks form seven products instead of five, but every sum has one owner:
// no atomics, the same bits every time.
//
// Scores, softmax statistics, probabilities' sums and all accumulators are fp32.  For 16-bit inputs P and dS are
// rounded to the inputs' type as operands of the matrix instructions (the products of 16-bit operands are what runs
// at the card's rate; each rounding is relative to the value, and their sum over a row averages out).
#include "rows.hpp"
#include "mma32.hpp"

namespace bgx {

constexpr int AT_WAVES = 4;
constexpr int AT_THREADS = AT_WAVES * WAVE;
constexpr int AT_TILE = 32 * AT_WAVES;  // rows a workgroup owns: 32 per wave
constexpr int AT_MAX_D = 128;
constexpr float AT_LOG2E = 1.4426950408889634f;

struct AttnView {
  const void* p;
  int64_t seq, tok, head;  // strides in elements
};

struct AttnArgs {
  AttnView q, k, v, o, grad_o, dq, dk, dv;
  // Of the softmax, per head and row: a shift of the exponents (the largest score in units of log 2) and the sum of
  // 2^(score - shift).  Kept apart: the rounding of a shift cancels between a row's weights and their sum, that of a
  // logarithm of the sum would not.
  float* shift;           // [Hq][rows]
  float* sum;             // [Hq][rows]
  void* rest;             // [rows][Hq][D], 16-bit types: o minus its rounded value, rounded
  float* delta;           // [Hq][rows]
  float* peak;            // [Hq][rows]: largest |do| of the row (fp16 only)
  const int4* table;      // packed: {first row, length, tile, limit} per tile of AT_TILE rows, heaviest first
  const int32_t* lengths; // batch layout: [N] or NULL
  int64_t rows;           // N * S, or the packed rows
  int N, S, tiles;        // tiles: per sequence (batch layout) or entries (packed)
  int Hq, Hk, group, D;
  float scale;
};

// ---- LDS tiles -------------------------------------------------------------------------------------------------
// Rows of DP elements in 16-byte chunks.  Chunk c of row r sits at c ^ key(r): 16 consecutive rows of one chunk (the
// operand read by rows) and 4 consecutive rows of 4 chunks (the transposed read) then both cover all banks.
template <typename T, int DP>
struct Tile {
  static constexpr int PITCH = (DP == 96 ? 128 : DP) * (int)sizeof(T);
  static constexpr int CHUNKS = DP * (int)sizeof(T) / 16;
  __device__ static int key(int row) {
    if constexpr (PITCH == 64) return (row >> 2) & 3;
    if constexpr (PITCH == 128) return (((row >> 1) & 1) << 2) | ((row >> 2) & 3);
    if constexpr (PITCH == 256) return ((row & 3) << 2) | ((row >> 2) & 3);
    return row & 15;
  }
  __device__ static int at(int row, int chunk) { return row * PITCH + ((chunk ^ key(row)) << 4); }
};

// Matrix-instruction operands per element type.  A "group" is the stretch of the contraction index one accumulator
// block feeds into one operand: 16 rows of the first product (two of its 4-register runs) at 16 bits, 8 in fp32.
template <typename T>
struct Attn {
  static constexpr int EPL = 8, GROUP = 16, REGS = 8;
  // registers g * REGS .. of an accumulator block as a second operand
  __device__ static uint4 pack(const f32x16& s, int g) {
    float f[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = s[g * 8 + i];
    return Chunk<T>::pack(f);
  }
  // first operand: column dt * 32 + lane % 32 of the tile, rows base + g * 16 + {4 h .. 4 h + 3, 8 + 4 h ..}
  // (h = lane / 32) -- the rows registers g * 8 .. g * 8 + 7 of an accumulator hold on this half of the wave.  Each 16
  // lanes hand the transposing read 4 rows of 16 columns and get one column of 4 rows each.
  template <int DP>
  __device__ static uint4 read_tr(const char* tile, int base, int dt, int lane) {
    typedef short s4 __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) s4 lds_s4;
    const int row = base + 4 * (lane >> 5) + ((lane >> 2) & 3);
    const int chunk = dt * 4 + ((lane >> 4) & 1) * 2 + ((lane >> 1) & 1), sub = (lane & 1) * 8;
    const s4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(tile + Tile<T, DP>::at(row, chunk) + sub));
    const s4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(tile + Tile<T, DP>::at(row + 8, chunk) + sub));
    const uint2 a = __builtin_bit_cast(uint2, lo), b = __builtin_bit_cast(uint2, hi);
    return make_uint4(a.x, a.y, b.x, b.y);
  }
};
template <>
struct Attn<float> {
  static constexpr int EPL = 4, GROUP = 8, REGS = 4;
  __device__ static uint4 pack(const f32x16& s, int g) {
    return make_uint4(__float_as_uint(s[g * 4]), __float_as_uint(s[g * 4 + 1]), __float_as_uint(s[g * 4 + 2]),
                      __float_as_uint(s[g * 4 + 3]));
  }
  template <int DP>
  __device__ static uint4 read_tr(const char* tile, int base, int dt, int lane) {
    const int row = base + 4 * (lane >> 5), col = dt * 32 + (lane & 31);
    uint32_t w[4];
#pragma unroll
    for (int e = 0; e < 4; ++e)
      w[e] = *reinterpret_cast<const uint32_t*>(tile + Tile<float, DP>::at(row + e, col >> 2) + (col & 3) * 4);
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};

// operand read by rows: chunk 2 ks + h of row base + lane % 32
template <typename T, int DP>
__device__ inline uint4 read_rows(const char* tile, int base, int ks, int lane) {
  return *reinterpret_cast<const uint4*>(tile + Tile<T, DP>::at(base + (lane & 31), 2 * ks + (lane >> 5)));
}

// larger / sum of a lane's value and that of the lane in the wave's other half
__device__ inline float2 both_halves(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return make_float2(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// BK rows of a [rows, D] operand on their way to an LDS tile: loaded into registers a tile ahead, stored after the
// current tile's work.  Rows from `len` on and columns from D on become zeros and are not read.
template <typename T, int DP, int BK>
struct Staged {
  static constexpr int CH = Tile<T, DP>::CHUNKS, PER = (BK * CH + AT_THREADS - 1) / AT_THREADS;
  uint4 v[PER];
  __device__ void load(const T* base, int64_t tok, int row0, int len, int D) {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int idx = threadIdx.x + i * AT_THREADS, row = idx / CH, col = (idx % CH) * Chunk<T>::N;
      v[i] = make_uint4(0u, 0u, 0u, 0u);
      if (row < BK && row0 + row < len && col < D) v[i] = load_chunk_tail(base + (row0 + row) * tok, col, D);
    }
  }
  __device__ void store(char* tile) const {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int idx = threadIdx.x + i * AT_THREADS, row = idx / CH;
      if (row < BK) *reinterpret_cast<uint4*>(tile + Tile<T, DP>::at(row, idx % CH)) = v[i];
    }
  }
};

// ---- what a workgroup works on -----------------------------------------------------------------------------------
struct AttnItem {
  int64_t seq;   // sequence index of the batch layout (0 when packed)
  int64_t row0;  // first packed row of the sequence (0 in the batch layout)
  int64_t stat;  // index of the sequence's first row among all rows
  int len;       // rows of the sequence
  int limit;     // rows up to here (len .. limit - 1) belong to no sequence and become zero
  int tile;
};

// Consecutive workgroups go to the chip's eight dies in turn.  `u` = index within one rank of tiles, over all
// (sequence, query head) pairs: the heads that share keys and values, and all tiles of a head, land on one die, whose
// L2 then holds that head's K and V.
__device__ inline void spread_heads(int u, int streams, int group, int& stream, int& g) {
  if (streams % 8 == 0) {
    const int j = u / 8, per = streams / 8;
    stream = (j % per) * 8 + u % 8;
    g = j / per;
  } else {
    stream = u % streams;
    g = u / streams;
  }
}

// keys: the workgroup owns key rows (all query heads of one key/value head, first tile heaviest) instead of query rows
// (one query head, last tile heaviest).
__device__ inline bool attn_item(const AttnArgs& A, bool keys, AttnItem& it, int& kv_head, int& q_head) {
  const int group = keys ? 1 : A.group;
  int g;
  if (A.table != nullptr) {
    const int per = A.Hk * group;
    const int4 e = A.table[blockIdx.x / per];
    if (e.w <= 0) return false;
    spread_heads(blockIdx.x % per, A.Hk, group, kv_head, g);
    it.seq = 0;
    it.row0 = it.stat = e.x;
    it.len = e.y;
    it.limit = e.w;
    const int tiles = (e.y + AT_TILE - 1) / AT_TILE;
    it.tile = keys && e.y > 0 ? tiles - 1 - e.z : e.z;
  } else {
    const int per = A.N * A.Hk * group, rank = blockIdx.x / per;
    int stream;
    spread_heads(blockIdx.x % per, A.N * A.Hk, group, stream, g);
    it.seq = stream / A.Hk;
    kv_head = stream % A.Hk;
    it.row0 = 0;
    it.stat = it.seq * A.S;
    int len = A.S;
    if (A.lengths != nullptr) len = min(max(A.lengths[it.seq], 0), A.S);
    it.len = len;
    it.limit = A.S;
    it.tile = keys ? rank : A.tiles - 1 - rank;
  }
  q_head = kv_head * A.group + g;
  return true;
}

template <typename T>
__device__ inline const T* attn_rows(const AttnView& v, const AttnItem& it, int head) {
  return (const T*)v.p + it.seq * v.seq + it.row0 * v.tok + head * v.head;
}

// 32 rows (one per lane % 32) of an accumulator set [d, row], times `f`, written as rows of D elements from `out` (this
// lane's row).  An accumulator holds 4 consecutive elements here and the next 4 in the wave's other half: at 16 bits two
// such runs are exchanged between the halves, so that every store has 16 bytes.  REST: what the rounding cuts off
// goes to `rest` in the same layout.
template <typename T, int DP, bool REST = false>
__device__ inline void store_rows(T* out, T* rest, const f32x16 (&acc)[DP / 32], float f, bool in, int D, int lane) {
  const int half = lane >> 5;
#pragma unroll
  for (int dt = 0; dt < DP / 32; ++dt) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = acc[dt][4 * b + e] * f;
        const int d = dt * 32 + 8 * b + 4 * half;
        if (in && d < D) store_chunk_tail(out, d, D, Chunk<T>::pack(v));
      }
    } else {
#pragma unroll
      for (int pair = 0; pair < 2; ++pair) {
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = acc[dt][8 * pair + e] * f;
        const int d = dt * 32 + 8 * (2 * pair + half);
        auto exchange = [](const uint4& w) {
          const auto a = __builtin_amdgcn_permlane32_swap(w.x, w.z, false, false);
          const auto b = __builtin_amdgcn_permlane32_swap(w.y, w.w, false, false);
          return make_uint4(a[0], b[0], a[1], b[1]);
        };
        const uint4 w = Chunk<T>::pack(v);
        const uint4 whole = exchange(w);
        if (in && d < D) store_chunk_tail(out, d, D, whole);
        if constexpr (REST) {
          float r[8];
          Chunk<T>::unpack(w, r);
#pragma unroll
          for (int e = 0; e < 8; ++e) r[e] = v[e] - r[e];
          const uint4 low = exchange(Chunk<T>::pack(r));
          if (in && d < D) store_chunk_tail(rest, d, D, low);
        }
      }
    }
  }
}

// this lane's half of a row becomes zero
template <typename T, int DP>
__device__ inline void zero_row(T* out, int D, int lane) {
#pragma unroll
  for (int c = 0; c < DP / Chunk<T>::N / 2; ++c) {
    const int d = (2 * c + (lane >> 5)) * Chunk<T>::N;
    if (d < D) store_chunk_tail(out, d, D, make_uint4(0u, 0u, 0u, 0u));
  }
}

template <typename T>
__device__ inline T* attn_row(const AttnView& v, const AttnItem& it, int head, int row) {
  return const_cast<T*>(attn_rows<T>(v, it, head)) + row * v.tok;
}

// first-operand fragments of one row kept in registers (zeros for rows past the end)
template <typename T, int DP>
__device__ inline void load_own(const T* base, int64_t tok, int row, bool in, int D, int lane, uint4 (&f)[DP / (2 * Attn<T>::EPL)]) {
  constexpr int EPL = Attn<T>::EPL;
#pragma unroll
  for (int ks = 0; ks < DP / (2 * EPL); ++ks) {
    const int col = (2 * ks + (lane >> 5)) * EPL;
    f[ks] = make_uint4(0u, 0u, 0u, 0u);
    if (in && col < D) f[ks] = load_chunk_tail(base + row * tok, col, D);
  }
}

__device__ inline float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }

template <typename T>
constexpr int attn_block_keys() {
  return sizeof(T) == 4 ? 32 : 64;
}

// ---- forward -----------------------------------------------------------------------------------------------------
template <typename T, int DP>
__global__ __launch_bounds__(AT_THREADS, 2) void attention_forward_kernel(AttnArgs A) {
  using M = Attn<T>;
  constexpr int BK = attn_block_keys<T>(), KS = DP / (2 * M::EPL), SUB = BK / 32, G = 32 / M::GROUP, DT = DP / 32;
  constexpr int BYTES = BK * Tile<T, DP>::PITCH;
  __shared__ __attribute__((aligned(16))) char lds[2][2][BYTES];
  AttnItem it;
  int kvh, qh;
  if (!attn_item(A, false, it, kvh, qh)) return;
  const int lane = threadIdx.x & (WAVE - 1), wave = threadIdx.x / WAVE;
  const int first = it.tile * AT_TILE, mine = first + wave * 32, row = mine + (lane & 31), half = lane >> 5;
  if (first >= it.len) {  // nothing of the sequence in this tile
    if (row < it.limit) zero_row<T, DP>(attn_row<T>(A.o, it, qh, row), A.D, lane);
    return;
  }
  const T* q = attn_rows<T>(A.q, it, qh);
  const T* k = attn_rows<T>(A.k, it, kvh);
  const T* v = attn_rows<T>(A.v, it, kvh);
  uint4 qf[KS];
  load_own<T, DP>(q, A.q.tok, row, row < it.len, A.D, lane, qf);
  f32x16 o[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[dt][i] = 0.f;
  float m = -INFINITY, l = 0.f;
  const float c = A.scale * AT_LOG2E;
  const int n_tiles = (min(first + AT_TILE, it.len) + BK - 1) / BK;
  Staged<T, DP, BK> sk, sv;
  sk.load(k, A.k.tok, 0, it.len, A.D);
  sv.load(v, A.v.tok, 0, it.len, A.D);
  sk.store(lds[0][0]);
  sv.store(lds[0][1]);
  for (int t = 0; t < n_tiles; ++t) {
    __syncthreads();  // this tile is in LDS, and nobody reads the other buffer any more
    const bool more = t + 1 < n_tiles;
    if (more) {
      sk.load(k, A.k.tok, (t + 1) * BK, it.len, A.D);
      sv.load(v, A.v.tok, (t + 1) * BK, it.len, A.D);
    }
    const char* tk = lds[t & 1][0];
    const char* tv = lds[t & 1][1];
    const int k0 = t * BK;
    if (k0 <= mine + 31 && mine < it.len) {
      f32x16 s[SUB];
#pragma unroll
      for (int u = 0; u < SUB; ++u) {
#pragma unroll
        for (int i = 0; i < 16; ++i) s[u][i] = 0.f;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) Mma32<T>::mma(read_rows<T, DP>(tk, u * 32, ks, lane), qf[ks], s[u]);
      }
      if (k0 + BK - 1 > mine) {  // the tile reaches past some row's own position
#pragma unroll
        for (int u = 0; u < SUB; ++u)
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (k0 + u * 32 + 8 * (i / 4) + 4 * half + i % 4 > row) s[u][i] = -INFINITY;
      }
      float top = m;
#pragma unroll
      for (int u = 0; u < SUB; ++u)
#pragma unroll
        for (int i = 0; i < 16; ++i) top = fmaxf(top, s[u][i]);
      const float2 halves = both_halves(top);
      top = fmaxf(halves.x, halves.y);
      // a row all of whose scores so far are -inf keeps a maximum of -inf; its weights are 0, not 0 - 0
      const float shift = top == -INFINITY ? 0.f : top * c;
      if (__any(top > m)) {
        const float f = exp2_of(m * c - shift);
        l *= f;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
          for (int i = 0; i < 16; ++i) o[dt][i] *= f;
        m = top;
      }
#pragma unroll
      for (int u = 0; u < SUB; ++u)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          s[u][i] = exp2_of(fmaf(s[u][i], c, -shift));
          l += s[u][i];
        }
#pragma unroll
      for (int u = 0; u < SUB; ++u)
#pragma unroll
        for (int g = 0; g < G; ++g) {
          const uint4 p = M::pack(s[u], g);
#pragma unroll
          for (int dt = 0; dt < DT; ++dt)
            Mma32<T>::mma(M::template read_tr<DP>(tv, u * 32 + g * M::GROUP, dt, lane), p, o[dt]);
        }
    }
    if (more) {
      sk.store(lds[(t + 1) & 1][0]);
      sv.store(lds[(t + 1) & 1][1]);
    }
  }
  const float2 ls = both_halves(l);
  l = ls.x + ls.y;
  const bool in = row < it.len;
  T* out = attn_row<T>(A.o, it, qh, row);
  if (A.shift == nullptr) {
    store_rows<T, DP>(out, nullptr, o, 1.0f / l, in, A.D, lane);
  } else {
    if (in && half == 0) {
      const int64_t stat = (int64_t)qh * A.rows + it.stat + row;
      A.shift[stat] = m * c;
      A.sum[stat] = l;
    }
    if constexpr (sizeof(T) == 2)
      store_rows<T, DP, true>(out, (T*)A.rest + ((it.stat + row) * A.Hq + qh) * A.D, o, 1.0f / l, in, A.D, lane);
    else
      store_rows<T, DP>(out, nullptr, o, 1.0f / l, in, A.D, lane);
  }
  if (!in && row < it.limit) zero_row<T, DP>(out, A.D, lane);
}

// ---- backward: queries -------------------------------------------------------------------------------------------
// dq of 32 queries a wave; also leaves delta (and, for fp16, the largest |do| of a row) for the other kernel.
template <typename T, int DP>
__global__ __launch_bounds__(AT_THREADS, 2) void attention_backward_q_kernel(AttnArgs A) {
  using M = Attn<T>;
  constexpr bool HALF = std::is_same<T, f16_t>::value;
  constexpr int BK = attn_block_keys<T>(), KS = DP / (2 * M::EPL), SUB = BK / 32, G = 32 / M::GROUP, DT = DP / 32;
  constexpr int BYTES = BK * Tile<T, DP>::PITCH;
  __shared__ __attribute__((aligned(16))) char lds[2][2][BYTES];
  AttnItem it;
  int kvh, qh;
  if (!attn_item(A, false, it, kvh, qh)) return;
  const int lane = threadIdx.x & (WAVE - 1), wave = threadIdx.x / WAVE;
  const int first = it.tile * AT_TILE, mine = first + wave * 32, row = mine + (lane & 31), half = lane >> 5;
  if (first >= it.len) {
    if (row < it.limit) zero_row<T, DP>(attn_row<T>(A.dq, it, qh, row), A.D, lane);
    return;
  }
  const bool in = row < it.len;
  const T* k = attn_rows<T>(A.k, it, kvh);
  const T* v = attn_rows<T>(A.v, it, kvh);
  uint4 qf[KS], gf[KS];
  load_own<T, DP>(attn_rows<T>(A.grad_o, it, qh), A.grad_o.tok, row, in, A.D, lane, gf);
  float delta = 0.f, peak = 0.f;
  {
    load_own<T, DP>(attn_rows<T>(A.o, it, qh), A.o.tok, row, in, A.D, lane, qf);
    uint4 rf[KS];
    if constexpr (sizeof(T) == 2)
      load_own<T, DP>((const T*)A.rest + (it.stat * A.Hq + qh) * A.D, (int64_t)A.Hq * A.D, row, in, A.D, lane, rf);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      float a[M::EPL], b[M::EPL];
      Chunk<T>::unpack(qf[ks], a);
      Chunk<T>::unpack(gf[ks], b);
      if constexpr (sizeof(T) == 2) {  // delta stands against dp in fp32: it needs o unrounded
        float r[M::EPL];
        Chunk<T>::unpack(rf[ks], r);
#pragma unroll
        for (int e = 0; e < M::EPL; ++e) a[e] += r[e];
      }
#pragma unroll
      for (int e = 0; e < M::EPL; ++e) {
        delta = fmaf(a[e], b[e], delta);
        peak = fmaxf(peak, fabsf(b[e]));
      }
    }
    const float2 d = both_halves(delta), p = both_halves(peak);
    delta = d.x + d.y;
    peak = fmaxf(p.x, p.y);
  }
  load_own<T, DP>(attn_rows<T>(A.q, it, qh), A.q.tok, row, in, A.D, lane, qf);
  const int64_t stat = (int64_t)qh * A.rows + it.stat + row;
  if (in && half == 0) {
    A.delta[stat] = delta;
    if constexpr (HALF) A.peak[stat] = peak;
  }
  // dS is P times something of the size of do: with small gradients it would fall among fp16's subnormals.  The
  // row's power of two is taken out of it (in the exponent of P, at no cost) and put back on dq.
  float lift = 0.f;
  if constexpr (HALF) lift = peak > 0.f && peak < INFINITY ? -(float)ilogbf(peak) : 0.f;
  const float shift = in ? A.shift[stat] - lift : 0.f, over_sum = in ? 1.0f / A.sum[stat] : 0.f;
  const float c = A.scale * AT_LOG2E;
  f32x16 dq[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int i = 0; i < 16; ++i) dq[dt][i] = 0.f;
  const int n_tiles = (min(first + AT_TILE, it.len) + BK - 1) / BK;
  Staged<T, DP, BK> sk, sv;
  sk.load(k, A.k.tok, 0, it.len, A.D);
  sv.load(v, A.v.tok, 0, it.len, A.D);
  sk.store(lds[0][0]);
  sv.store(lds[0][1]);
  for (int t = 0; t < n_tiles; ++t) {
    __syncthreads();
    const bool more = t + 1 < n_tiles;
    if (more) {
      sk.load(k, A.k.tok, (t + 1) * BK, it.len, A.D);
      sv.load(v, A.v.tok, (t + 1) * BK, it.len, A.D);
    }
    const char* tk = lds[t & 1][0];
    const char* tv = lds[t & 1][1];
    const int k0 = t * BK;
    if (k0 <= mine + 31 && mine < it.len) {
#pragma unroll
      for (int u = 0; u < SUB; ++u) {
        f32x16 s, dp;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          s[i] = 0.f;
          dp[i] = -delta;
        }
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          Mma32<T>::mma(read_rows<T, DP>(tk, u * 32, ks, lane), qf[ks], s);
          Mma32<T>::mma(read_rows<T, DP>(tv, u * 32, ks, lane), gf[ks], dp);
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] = exp2_of(fmaf(s[i], c, -shift)) * dp[i];
        if (k0 + u * 32 + 31 > mine) {
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (k0 + u * 32 + 8 * (i / 4) + 4 * half + i % 4 > row) s[i] = 0.f;
        }
#pragma unroll
        for (int g = 0; g < G; ++g) {
          const uint4 ds = M::pack(s, g);
#pragma unroll
          for (int dt = 0; dt < DT; ++dt)
            Mma32<T>::mma(M::template read_tr<DP>(tk, u * 32 + g * M::GROUP, dt, lane), ds, dq[dt]);
        }
      }
    }
    if (more) {
      sk.store(lds[(t + 1) & 1][0]);
      sv.store(lds[(t + 1) & 1][1]);
    }
  }
  T* out = attn_row<T>(A.dq, it, qh, row);
  store_rows<T, DP>(out, nullptr, dq, A.scale * over_sum * exp2_of(-lift), in, A.D, lane);
  if (!in && row < it.limit) zero_row<T, DP>(out, A.D, lane);
}

// ---- backward: keys and values -----------------------------------------------------------------------------------
template <typename T, int DP>
__global__ __launch_bounds__(AT_THREADS, 1) void attention_backward_kv_kernel(AttnArgs A) {
  using M = Attn<T>;
  constexpr bool HALF = std::is_same<T, f16_t>::value;
  constexpr int BQ = attn_block_keys<T>(), KS = DP / (2 * M::EPL), SUB = BQ / 32, G = 32 / M::GROUP, DT = DP / 32;
  constexpr int BYTES = BQ * Tile<T, DP>::PITCH;
  __shared__ __attribute__((aligned(16))) char lds[2][2][BYTES];
  constexpr int NSTAT = std::is_same<T, bf16_t>::value ? 2 : 3;
  __shared__ __attribute__((aligned(16))) float stats[2][NSTAT][BQ];
  AttnItem it;
  int kvh, qh0;
  if (!attn_item(A, true, it, kvh, qh0)) return;
  const int lane = threadIdx.x & (WAVE - 1), wave = threadIdx.x / WAVE;
  const int first = it.tile * AT_TILE, mine = first + wave * 32, row = mine + (lane & 31), half = lane >> 5;
  if (first >= it.len) {
    if (row < it.limit) {
      zero_row<T, DP>(attn_row<T>(A.dk, it, kvh, row), A.D, lane);
      zero_row<T, DP>(attn_row<T>(A.dv, it, kvh, row), A.D, lane);
    }
    return;
  }
  const bool in = row < it.len;
  uint4 kf[KS], vf[KS];
  load_own<T, DP>(attn_rows<T>(A.k, it, kvh), A.k.tok, row, in, A.D, lane, kf);
  load_own<T, DP>(attn_rows<T>(A.v, it, kvh), A.v.tok, row, in, A.D, lane, vf);
  f32x16 dk[DT], dv[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int i = 0; i < 16; ++i) dk[dt][i] = dv[dt][i] = 0.f;
  const float c = A.scale * AT_LOG2E;
  const int t0 = first / BQ, per_head = (it.len + BQ - 1) / BQ - t0, n_tiles = per_head * A.group;
  Staged<T, DP, BQ> sq, sg;
  float stage[NSTAT];
#pragma unroll
  for (int i = 0; i < NSTAT; ++i) stage[i] = 0.f;
  auto load = [&](int t) {
    const int qh = qh0 + t / per_head, q0 = (t0 + t % per_head) * BQ;
    sq.load(attn_rows<T>(A.q, it, qh), A.q.tok, q0, it.len, A.D);
    sg.load(attn_rows<T>(A.grad_o, it, qh), A.grad_o.tok, q0, it.len, A.D);
    if (threadIdx.x < BQ) {
      const bool ok = q0 + (int)threadIdx.x < it.len;
      const int64_t stat = (int64_t)qh * A.rows + it.stat + q0 + threadIdx.x;
      const float sum = ok ? A.sum[stat] : 1.f;
      stage[0] = ok ? A.shift[stat] : 0.f;
      // at 16 bits the sum joins the exponent (its rounding there is far below that of the weights); in fp32 it does not
      if constexpr (sizeof(T) == 2)
        stage[0] += log2f(sum);
      else
        stage[2] = 1.0f / sum;
      stage[1] = ok ? A.delta[stat] : 0.f;
      if constexpr (HALF) stage[2] = ok ? A.peak[stat] : 0.f;
    }
  };
  auto store = [&](int b) {
    sq.store(lds[b][0]);
    sg.store(lds[b][1]);
    if (threadIdx.x < BQ) {
#pragma unroll
      for (int i = 0; i < NSTAT; ++i) stats[b][i][threadIdx.x] = stage[i];
    }
  };
  // fp16: dS carries a power of two that keeps it out of the subnormals, the one that fits the largest |do| seen so
  // far; when a tile brings a larger one, what has been summed is rescaled (exactly) to the new power.
  int lift = 0;
  bool lifted = false;
  load(0);
  store(0);
  for (int t = 0; t < n_tiles; ++t) {
    __syncthreads();
    const bool more = t + 1 < n_tiles;
    if (more) load(t + 1);
    const char* tq = lds[t & 1][0];
    const char* tg = lds[t & 1][1];
    const float(*st)[BQ] = stats[t & 1];
    const int q0 = (t0 + t % per_head) * BQ;
    if (q0 + BQ > mine && mine < it.len) {
      float raise = 1.f;
      if constexpr (HALF) {
        const float peak = wave_max(st[2][lane % BQ]);
        if (peak > 0.f && peak < INFINITY) {
          const int want = -ilogbf(peak);
          if (!lifted || want < lift) {
            if (lifted) {
              const float f = exp2_of((float)(want - lift));
#pragma unroll
              for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                for (int i = 0; i < 16; ++i) dk[dt][i] *= f;
            }
            lift = want;
            lifted = true;
          }
        }
        raise = exp2_of((float)lift);
      }
#pragma unroll
      for (int u = 0; u < SUB; ++u) {
        if (q0 + u * 32 + 31 < mine) continue;  // all of these queries come before this wave's keys
        f32x16 s, dp;
        float lse[16], over_sum[sizeof(T) == 4 ? 16 : 1];
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          const float4 a = *reinterpret_cast<const float4*>(&st[0][u * 32 + 8 * b + 4 * half]);
          const float4 d = *reinterpret_cast<const float4*>(&st[1][u * 32 + 8 * b + 4 * half]);
          lse[4 * b] = a.x, lse[4 * b + 1] = a.y, lse[4 * b + 2] = a.z, lse[4 * b + 3] = a.w;
          dp[4 * b] = -d.x, dp[4 * b + 1] = -d.y, dp[4 * b + 2] = -d.z, dp[4 * b + 3] = -d.w;
          if constexpr (sizeof(T) == 4) {
            const float4 w = *reinterpret_cast<const float4*>(&st[2][u * 32 + 8 * b + 4 * half]);
            over_sum[4 * b] = w.x, over_sum[4 * b + 1] = w.y, over_sum[4 * b + 2] = w.z, over_sum[4 * b + 3] = w.w;
          }
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] = 0.f;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          Mma32<T>::mma(read_rows<T, DP>(tq, u * 32, ks, lane), kf[ks], s);
          Mma32<T>::mma(read_rows<T, DP>(tg, u * 32, ks, lane), vf[ks], dp);
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          s[i] = exp2_of(fmaf(s[i], c, -lse[i]));
          if constexpr (sizeof(T) == 4) s[i] *= over_sum[i];
          dp[i] = HALF ? s[i] * raise * dp[i] : s[i] * dp[i];
        }
        if (q0 + u * 32 < mine + 31) {
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (q0 + u * 32 + 8 * (i / 4) + 4 * half + i % 4 < row) s[i] = dp[i] = 0.f;
        }
#pragma unroll
        for (int g = 0; g < G; ++g) {
          const uint4 p = M::pack(s, g), ds = M::pack(dp, g);
#pragma unroll
          for (int dt = 0; dt < DT; ++dt) {
            Mma32<T>::mma(M::template read_tr<DP>(tg, u * 32 + g * M::GROUP, dt, lane), p, dv[dt]);
            Mma32<T>::mma(M::template read_tr<DP>(tq, u * 32 + g * M::GROUP, dt, lane), ds, dk[dt]);
          }
        }
      }
    }
    if (more) store((t + 1) & 1);
  }
  T* out_k = attn_row<T>(A.dk, it, kvh, row);
  T* out_v = attn_row<T>(A.dv, it, kvh, row);
  store_rows<T, DP>(out_k, nullptr, dk, A.scale * exp2_of(-(float)lift), in, A.D, lane);
  store_rows<T, DP>(out_v, nullptr, dv, 1.0f, in, A.D, lane);
  if (!in && row < it.limit) {
    zero_row<T, DP>(out_k, A.D, lane);
    zero_row<T, DP>(out_v, A.D, lane);
  }
}

// ---- packed sequences: the list of tiles -------------------------------------------------------------------------
// One entry per AT_TILE rows of a sequence, entries of a higher tile (more keys to walk) first, and entries that only
// clear the rows outside every sequence.  The sequences' ends are device data: they are clamped to the packed rows and
// to each other, and an entry that would not fit in the list is dropped, so that no offsets lead out of bounds.
constexpr int PLAN_LEVELS = 4096;

__device__ inline int2 plan_sequence(const int32_t* cu, int n, int rows) {
  const int a = min(max(cu[n], 0), rows), b = min(max(cu[n + 1], a), rows);
  return make_int2(a, b - a);
}

__global__ __launch_bounds__(1024) void attention_plan_kernel(const int32_t* __restrict__ cu, int N, int rows,
                                                              int4* table, int entries) {
  __shared__ int level[PLAN_LEVELS];  // sequences with exactly that many tiles; then: entries before the level's first
  __shared__ int carry[1024];
  const int most = (rows + AT_TILE - 1) / AT_TILE;
  int fold = 0;  // levels are grouped by 2^fold tiles when there are more than PLAN_LEVELS
  while ((most >> fold) >= PLAN_LEVELS) ++fold;
  for (int i = threadIdx.x; i < PLAN_LEVELS; i += 1024) level[i] = 0;
  for (int i = threadIdx.x; i < entries; i += 1024) table[i] = make_int4(0, 0, 0, 0);
  __syncthreads();
  // tiles per level: a sequence of n tiles has one tile at each of 0 .. n - 1
  for (int n = threadIdx.x; n < N; n += 1024) {
    const int tiles = (plan_sequence(cu, n, rows).y + AT_TILE - 1) / AT_TILE;
    for (int t = 0; t < tiles; t += 1 << fold) atomicAdd(&level[t >> fold], min(1 << fold, tiles - t));
  }
  __syncthreads();
  // entries before each level, the highest first: thread i sums a run of levels from the top
  constexpr int RUN = PLAN_LEVELS / 1024;
  int sum = 0;
  for (int j = 0; j < RUN; ++j) sum += level[PLAN_LEVELS - 1 - (threadIdx.x * RUN + j)];
  carry[threadIdx.x] = sum;
  __syncthreads();
  for (int d = 1; d < 1024; d <<= 1) {
    const int add = threadIdx.x >= d ? carry[threadIdx.x - d] : 0;
    __syncthreads();
    carry[threadIdx.x] += add;
    __syncthreads();
  }
  int before = threadIdx.x > 0 ? carry[threadIdx.x - 1] : 0;
  const int total = carry[1023];
  for (int j = 0; j < RUN; ++j) {
    const int l = PLAN_LEVELS - 1 - (threadIdx.x * RUN + j), here = level[l];
    level[l] = before;
    before += here;
  }
  __syncthreads();
  // within a level the order is whatever the counters hand out: it decides when a tile runs, not what it computes
  const int lane = threadIdx.x & (WAVE - 1), wave = threadIdx.x / WAVE;
  for (int n = wave; n < N; n += 1024 / WAVE) {
    const int2 s = plan_sequence(cu, n, rows);
    const int tiles = (s.y + AT_TILE - 1) / AT_TILE;
    for (int t = lane; t < tiles; t += WAVE) {
      const int at = atomicAdd(&level[t >> fold], 1);
      if ((unsigned)at < (unsigned)entries) table[at] = make_int4(s.x, s.y, t, s.y);
    }
  }
  // rows before the first and after the last sequence
  const int head = N > 0 ? plan_sequence(cu, 0, rows).x : 0;
  const int2 last = N > 0 ? plan_sequence(cu, N - 1, rows) : make_int2(0, 0);
  const int tail = last.x + last.y, head_tiles = (head + AT_TILE - 1) / AT_TILE;
  const int tail_tiles = (rows - tail + AT_TILE - 1) / AT_TILE;
  for (int i = threadIdx.x; i < head_tiles + tail_tiles; i += 1024) {
    const int at = total + i;
    if ((unsigned)at >= (unsigned)entries) break;
    table[at] = i < head_tiles ? make_int4(0, 0, i, head) : make_int4(tail, 0, i - head_tiles, rows - tail);
  }
}

int64_t attention_plan_entries(int64_t rows, int N) { return rows / AT_TILE + N + 2; }

// ---- host side ---------------------------------------------------------------------------------------------------
static int attn_check(const bgx_attention_shape* a, const char* what) {
  BGX_REQUIRE(a != nullptr, BGX_E_ARG, "%s: null shape", what);
  BGX_REQUIRE(a->n_seqs >= 0 && a->rows >= 0, BGX_E_ARG, "%s: n_seqs=%d rows=%lld", what, a->n_seqs, (long long)a->rows);
  BGX_REQUIRE(a->heads >= 1 && a->kv_heads >= 1 && a->heads % a->kv_heads == 0, BGX_E_SHAPE,
              "%s: %d query heads on %d key/value heads", what, a->heads, a->kv_heads);
  BGX_REQUIRE(a->head_dim >= 1 && a->head_dim <= AT_MAX_D, BGX_E_SHAPE, "%s: head_dim=%d, supported are 1 to %d", what,
              a->head_dim, AT_MAX_D);
  BGX_REQUIRE(a->dtype >= BGX_F32 && a->dtype <= BGX_BF16, BGX_E_DTYPE, "%s: dtype %d", what, a->dtype);
  BGX_REQUIRE(a->scale > 0.f && a->scale < INFINITY, BGX_E_ARG, "%s: scale %g must be positive and finite", what, a->scale);
  // tile bounds are formed in 32 bits
  BGX_REQUIRE(a->rows < (1ll << 31) - 4 * AT_TILE, BGX_E_SHAPE, "%s: %lld rows", what, (long long)a->rows);
  if (a->plan_dev == nullptr)
    BGX_REQUIRE(a->n_seqs == 0 ? a->rows == 0 : a->rows % a->n_seqs == 0, BGX_E_ARG,
                "%s: %lld rows are not %d sequences of one width", what, (long long)a->rows, a->n_seqs);
  return 0;
}

static int64_t attn_items(const bgx_attention_shape* a) {
  if (a->plan_dev != nullptr) return attention_plan_entries(a->rows, a->n_seqs);
  const int64_t S = a->n_seqs ? a->rows / a->n_seqs : 0;
  return (S + AT_TILE - 1) / AT_TILE * a->n_seqs;
}

static AttnArgs attn_args(const bgx_attention_shape* a) {
  AttnArgs A{};
  A.table = (const int4*)a->plan_dev;
  A.lengths = a->lengths_dev;
  A.rows = a->rows;
  A.N = a->n_seqs;
  A.S = a->plan_dev == nullptr && a->n_seqs ? (int)(a->rows / a->n_seqs) : 0;
  A.tiles = (A.S + AT_TILE - 1) / AT_TILE;
  A.Hq = a->heads;
  A.Hk = a->kv_heads;
  A.group = a->heads / a->kv_heads;
  A.D = a->head_dim;
  A.scale = a->scale;
  return A;
}

static AttnView attn_view(const bgx_attention_rows* t) {
  AttnView v{};
  if (t != nullptr) {
    v.p = t->data;
    v.seq = t->seq_stride;
    v.tok = t->tok_stride;
    v.head = t->head_stride;
  }
  return v;
}

#define BGX_ATTN_WIDTHS(KERNEL, T, D, GRID, S, A)            \
  do {                                                       \
    if ((D) <= 32)                                           \
      KERNEL<T, 32><<<(GRID), AT_THREADS, 0, (S)>>>(A);      \
    else if ((D) <= 64)                                      \
      KERNEL<T, 64><<<(GRID), AT_THREADS, 0, (S)>>>(A);      \
    else if ((D) <= 96)                                      \
      KERNEL<T, 96><<<(GRID), AT_THREADS, 0, (S)>>>(A);      \
    else                                                     \
      KERNEL<T, 128><<<(GRID), AT_THREADS, 0, (S)>>>(A);     \
  } while (0)
#define BGX_ATTN_LAUNCH(KERNEL, DTYPE, D, GRID, S, A)        \
  do {                                                       \
    if ((DTYPE) == BGX_F32)                                  \
      BGX_ATTN_WIDTHS(KERNEL, float, D, GRID, S, A);         \
    else if ((DTYPE) == BGX_F16)                             \
      BGX_ATTN_WIDTHS(KERNEL, f16_t, D, GRID, S, A);         \
    else                                                     \
      BGX_ATTN_WIDTHS(KERNEL, bf16_t, D, GRID, S, A);        \
    BGX_HIP(hipGetLastError());                              \
  } while (0)

size_t attention_plan_bytes(int64_t rows, int n_seqs) {
  if (rows < 0 || n_seqs < 0) return 0;
  return (size_t)attention_plan_entries(rows, n_seqs) * sizeof(int4);
}

int attention_plan_impl(const int32_t* cu, int n_seqs, int64_t rows, void* plan, size_t plan_bytes, void* stream) {
  BGX_REQUIRE(n_seqs >= 0 && rows >= 0 && rows < (1ll << 31) - 4 * AT_TILE, BGX_E_ARG, "attention plan: n_seqs=%d rows=%lld",
              n_seqs, (long long)rows);
  BGX_REQUIRE(cu != nullptr || n_seqs == 0, BGX_E_ARG, "attention plan: null cu_seqlens");
  const int64_t entries = attention_plan_entries(rows, n_seqs);
  BGX_REQUIRE(entries < (1ll << 31), BGX_E_SHAPE, "attention plan: %lld entries", (long long)entries);
  BGX_REQUIRE(plan != nullptr && plan_bytes >= attention_plan_bytes(rows, n_seqs), BGX_E_WORKSPACE,
              "attention plan: %zu bytes, %zu needed", plan_bytes, attention_plan_bytes(rows, n_seqs));
  attention_plan_kernel<<<1, 1024, 0, (hipStream_t)stream>>>(cu, n_seqs, (int)rows, (int4*)plan, (int)entries);
  BGX_HIP(hipGetLastError());
  return 0;
}

// the saved buffer: shift and sum of every head and row, then the rest of the output
size_t attention_saved_bytes(const bgx_attention_shape* a) {
  if (a == nullptr || a->rows <= 0 || a->heads <= 0 || a->head_dim <= 0) return 0;
  const size_t n = (size_t)a->rows * a->heads;
  return n * 2 * sizeof(float) + (a->dtype == BGX_F32 ? 0 : n * a->head_dim * dtype_size(a->dtype));
}

static void attn_saved(AttnArgs& A, const bgx_attention_shape* a, void* saved) {
  const int64_t n = a->rows * a->heads;
  A.shift = (float*)saved;
  A.sum = saved == nullptr ? nullptr : A.shift + n;
  A.rest = saved == nullptr ? nullptr : A.sum + n;
}

int attention_forward_impl(const bgx_attention_shape* a, const bgx_attention_rows* q, const bgx_attention_rows* k,
                           const bgx_attention_rows* v, const bgx_attention_rows* o, void* saved, void* stream) {
  if (int rc = attn_check(a, "attention")) return rc;
  if (a->rows == 0) return 0;
  BGX_REQUIRE(q && k && v && o && q->data && k->data && v->data && o->data, BGX_E_ARG, "attention: null operand");
  AttnArgs A = attn_args(a);
  A.q = attn_view(q);
  A.k = attn_view(k);
  A.v = attn_view(v);
  A.o = attn_view(o);
  attn_saved(A, a, saved);
  const int64_t grid = attn_items(a) * a->heads;
  BGX_REQUIRE(grid < (1ll << 31), BGX_E_SHAPE, "attention: %lld workgroups", (long long)grid);
  BGX_ATTN_LAUNCH(attention_forward_kernel, a->dtype, a->head_dim, dim3((unsigned)grid), (hipStream_t)stream, A);
  return 0;
}

size_t attention_backward_workspace_bytes(const bgx_attention_shape* a) {
  if (a == nullptr || a->rows <= 0 || a->heads <= 0) return 0;
  return (size_t)a->rows * a->heads * sizeof(float) * (a->dtype == BGX_F16 ? 2 : 1);
}

int attention_backward_impl(const bgx_attention_shape* a, const bgx_attention_rows* q, const bgx_attention_rows* k,
                            const bgx_attention_rows* v, const bgx_attention_rows* o, const void* saved,
                            const bgx_attention_rows* grad_o, const bgx_attention_rows* dq, const bgx_attention_rows* dk,
                            const bgx_attention_rows* dv, void* ws, size_t ws_bytes, void* stream) {
  if (int rc = attn_check(a, "attention backward")) return rc;
  if (a->rows == 0) return 0;
  const bgx_attention_rows* all[] = {q, k, v, o, grad_o, dq, dk, dv};
  for (const bgx_attention_rows* t : all)
    BGX_REQUIRE(t != nullptr && t->data != nullptr, BGX_E_ARG, "attention backward: null operand");
  BGX_REQUIRE(saved != nullptr, BGX_E_ARG, "attention backward: null saved");
  const size_t need = attention_backward_workspace_bytes(a);
  BGX_REQUIRE(ws != nullptr && ws_bytes >= need, BGX_E_WORKSPACE, "attention backward: workspace of %zu bytes, %zu needed",
              ws_bytes, need);
  AttnArgs A = attn_args(a);
  A.q = attn_view(q);
  A.k = attn_view(k);
  A.v = attn_view(v);
  A.o = attn_view(o);
  A.grad_o = attn_view(grad_o);
  A.dq = attn_view(dq);
  A.dk = attn_view(dk);
  A.dv = attn_view(dv);
  attn_saved(A, a, const_cast<void*>(saved));
  A.delta = (float*)ws;
  A.peak = A.delta + a->rows * a->heads;
  const int64_t items = attn_items(a);
  BGX_REQUIRE(items * a->heads < (1ll << 31), BGX_E_SHAPE, "attention backward: %lld workgroups",
              (long long)(items * a->heads));
  hipStream_t s = (hipStream_t)stream;
  BGX_ATTN_LAUNCH(attention_backward_q_kernel, a->dtype, a->head_dim, dim3((unsigned)(items * a->heads)), s, A);
  BGX_ATTN_LAUNCH(attention_backward_kv_kernel, a->dtype, a->head_dim, dim3((unsigned)(items * a->kv_heads)), s, A);
  return 0;
}

}  // namespace bgx
