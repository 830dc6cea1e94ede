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
// at the card's rate; each rounding is relative to the value, and their sum over a row averages out; small calls and
// short sequences keep the rests, see Work; fp16 operands carry powers of two that keep them within the type, see DS_FIRST
// and P_LIFT).  delta is formed from o as it was before its rounding: dp - delta cancels.
//
// What bounds them: a 32 x 32 block of scores costs a wave 16 exponentials a lane beside 2 (forward), 3 (dq) or 4 (dk,
// dv) products.  At heads of 128 the products win: forward 303 us for 2 x 4096 positions, 32 query on 8 key/value heads
// (0.27 TFLOP of the causal half: 0.91 PFLOP/s), 2.2 ms for 1 x 16384 (1.0), dq 432 us (three products: 0.95), dk and
// dv 615 us (four: 0.89), where a large library product reaches 1.11.  At heads of 64 a block has half the products for
// the same vector work, which then takes longer than they do; long walks still overlap the two: 2 x 16384 positions, 16
// heads, fp16: forward 1.28 ms (0.86 PFLOP/s), dq, dk and dv 4.79 ms (seven products: 0.80).  Short walks do not hide
// what comes before and after them: 24 documents of 16 to 2048 positions (nine tiles a workgroup) take 85 us forward
// (0.55 PFLOP/s), 122 for dq (0.56), 185 for dk and dv (0.51), and without the walks, loading and storing the rows
// alone (4 to 5 TB/s), 28, 40 and 44.  There tiles of 32 or 128 keys instead of 64, four waves a SIMD instead of three,
// and raised wave priority around the products were no faster (forward 86, 93, 87, 84 us), nor long and short walks in
// turn instead of longest first (105), results turned through LDS to whole rows (84) or stored past the caches (97);
// eight waves for 64 rows made 4 x 1024 positions of 12 heads 23 us forward instead of 19.
#include <cfloat>
#include <initializer_list>

#include "mma32.hpp"
#include "rows.hpp"

namespace bgx {

constexpr int AT_WAVES = 4;
constexpr int AT_THREADS = AT_WAVES * WAVE;
constexpr int AT_TILES[3] = {128, 64, 32};  // rows a workgroup owns (see Work)
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
  float* peak;            // [Hq][rows]: no |dS| of the row is larger (fp16 only)
  float* part_k;          // [rows][Hq][D]: dk and dv of every query head by itself (attention_backward_join_kernel),
  float* part_v;          // NULL where a workgroup sums over the heads that share its keys
  const int4* table;      // packed: {first row, length, tile, limit} per tile of rows, heaviest first
  const int32_t* bounds;  // packed without a table: the sequences' boundaries
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

// what the rounding of pack() cuts off, as a second operand of its own (16-bit types)
template <typename T>
__device__ inline uint4 pack_rest(const f32x16& s, int g, const uint4& rounded) {
  float f[8];
  Chunk<T>::unpack(rounded, f);
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = s[g * 8 + i] - f[i];
  return Chunk<T>::pack(f);
}

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

// `rows` rows of D elements from `base` as a buffer: a load past them returns zeros and touches no memory, so that the
// ragged end of a sequence costs no branch (a branch around a load makes the compiler wait for the load where the paths
// meet).  Rows are at least D elements apart.
template <typename T>
__device__ inline __amdgpu_buffer_rsrc_t row_buffer(const T* base, int64_t tok, int rows, int D) {
  const int bytes = rows > 0 ? (int)(((rows - 1) * tok + D) * (int64_t)sizeof(T)) : 0;
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(base), 0, bytes, 0x00020000);
}
constexpr uint32_t NO_ROW = 0x7ffffff0u;  // an offset past every buffer, also with a tile's passes added

// The whole offset goes through the lane's register: the bounds check is defined for that part only.
__device__ inline uint4 buffer_load16(__amdgpu_buffer_rsrc_t r, uint32_t offset) {
  typedef uint32_t raw4 __attribute__((ext_vector_type(4)));
  const raw4 v = __builtin_bit_cast(raw4, __builtin_amdgcn_raw_buffer_load_b128(r, (int)offset, 0, 0));
  return make_uint4(v.x, v.y, v.z, v.w);
}
__device__ inline float buffer_load4(__amdgpu_buffer_rsrc_t r, uint32_t offset) {
  return __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(r, (int)offset, 0, 0));
}

// BK rows of a [rows, D] operand on their way to an LDS tile: loaded into registers a tile ahead, stored after the
// current tile's work.  Rows past the end and columns from D on become zeros.  A thread keeps one
// chunk of columns and takes every RPI-th row: its place in a tile is one 32-bit offset, made once; what changes from
// tile to tile is a uniform base.
template <typename T, int DP, int BK, int THREADS = AT_THREADS>
struct Staged {
  static constexpr int CH = Tile<T, DP>::PITCH / 16;  // threads per row (with DP = 96 a quarter of them idles)
  static constexpr int RPI = THREADS / CH, PER = BK / RPI;
  static_assert(BK % RPI == 0, "whole passes over a tile");
  uint4 v[PER];
  uint32_t offset, pass;
  __device__ void init(int64_t tok, int D) {
    const int chunk = threadIdx.x % CH, row = threadIdx.x / CH;
    offset = chunk * Chunk<T>::N < D ? (uint32_t)(row * (int)tok + chunk * Chunk<T>::N) * (uint32_t)sizeof(T) : NO_ROW;
    pass = (uint32_t)(RPI * (int)tok) * (uint32_t)sizeof(T);
  }
  // rows: how many rows there are from the tile's first on
  __device__ void load(const T* base, int64_t tok, int rows, int D) {
    const __amdgpu_buffer_rsrc_t r = row_buffer(base, tok, min(rows, BK), D);
#pragma unroll
    for (int i = 0; i < PER; ++i) v[i] = buffer_load16(r, offset + i * pass);
  }
  __device__ void store(char* tile) const {
    if (DP == 96 && (int)threadIdx.x % CH >= Tile<T, DP>::CHUNKS) return;
#pragma unroll
    for (int i = 0; i < PER; ++i)
      *reinterpret_cast<uint4*>(tile + Tile<T, DP>::at(threadIdx.x / CH + i * RPI, threadIdx.x % CH)) = v[i];
  }
};

// ---- which sequences a kernel takes ------------------------------------------------------------------------------
// Short sequences (AT_SHORT) have a body of their own: second products behind a branch in the others' walk would take the
// walk's registers.  Where the host cannot tell that there are none, one kernel has both bodies (AT_MIXED), which costs the
// walk some registers all the same, or each has a kernel: AT_BRIEF the first tile of every short sequence, AT_LONG
// everything else.  A launch more is the better at heads of more than 64 and 128 rows a workgroup.  Measured (us; without
// the short body / one kernel / two): 24 documents of 16 to 2048 positions, 16 heads of 64, fp16, forward and backward 369 / 385 /
// 390; 2 x 4096 positions with lengths, 32 / 8 heads of 128, the same 1332 / 1370 / 1337; 1 x 16384, forward 2166 / 2225 / 2203.
enum AttnKind {
  AT_ALL,    // fp32, and workgroups that take every sequence like a short one (Work::FINE)
  AT_LONG,
  AT_BRIEF,
  AT_MIXED,
};

// ---- how a workgroup's waves divide the work ---------------------------------------------------------------------
// A workgroup owns 32 * RW rows (queries, or keys in the kernel for dk and dv) and walks the other side in tiles of
// STEP rows.  RW = 4: every wave owns 32 rows and takes each tile whole.  RW = 2, 1: two or all four waves share 32
// rows, each takes its part of every tile, and their sums are joined through LDS at the end -- more workgroups with
// shorter walks, at twice or four times the traffic to LDS: for calls that would not fill the chip otherwise.
constexpr int AT_SHORT = 64;
template <typename T, int DP, int RW, int WAVES = AT_WAVES>
struct Work {
  static constexpr int THREADS = WAVES * WAVE, ROWS = 32 * RW, SPLIT = WAVES / RW;
  static constexpr int SUB = SPLIT == 1 && sizeof(T) == 2 ? 2 : 1;  // blocks of 32 a wave takes of a tile
  static constexpr int STEP = 32 * SUB * SPLIT;
  // Few workgroups leave the matrix units idle, and with few rows the roundings of P and dS do not average out (a
  // sequence of two rows shows that of its one dS in every gradient): there both go in as two operands, the rounded
  // value and the rest, which gives them 16 or more bits.
  static constexpr bool FINE = RW == 1 && sizeof(T) == 2;
  // Elsewhere P (in the forward pass) and dS of 16-bit sequences of up to AT_SHORT rows go in like that, whatever the call holds
  // beside them: dq and dk of 2 to 8 positions are 1.5 to 1.6 times as far off as their own rounding without it, 1.0 times
  // with it; of 64 and more 1.45 times.  See AttnKind.
  static_assert(sizeof(T) == 4 || STEP >= AT_SHORT || RW == 1, "a short sequence is one tile");
  // waves a SIMD has room for without spilling registers to memory in the walk (the compiler's budget: 512 / 3, / 2 or
  // 512; fp16's dq at heads of 64 keeps a few outside it: 73 us with two waves where three take 63, as above)
  static constexpr int PER_SIMD_Q = sizeof(T) == 4 ? (DP <= 32 ? 2 : 1) : DP <= 64 && RW == 4 ? 3 : (RW == 4 || DP <= 64 ? 2 : 1);
  static constexpr int PER_SIMD_KV = sizeof(T) == 4 ? (DP <= 32 ? 2 : 1) : (DP <= 64 || WAVES == 8 ? 2 : 1);
  static constexpr int BYTES = STEP * Tile<T, DP>::PITCH;
  static constexpr int BUFFERS = 4 * BYTES <= 65536 ? 2 : 1;  // two workgroups of a CU fit at 16 bits
  static constexpr int JOIN = (SPLIT - 1) * RW * (DP / 32) * 16 * WAVE * 4;
  static constexpr int LDS = 2 * BUFFERS * BYTES > JOIN ? 2 * BUFFERS * BYTES : JOIN;
};

// Sums of the waves that share rows: the others hand theirs to the first through LDS, which adds them in order.
template <typename W, int DT>
__device__ inline void join_waves(f32x16 (&acc)[DT], char* lds, int part, int group, int lane) {
  if constexpr (W::SPLIT > 1) {
    float4* box = reinterpret_cast<float4*>(lds) + group * (W::SPLIT - 1) * DT * 4 * WAVE;
    __syncthreads();
    if (part > 0) {
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int b = 0; b < 4; ++b)
          box[(((part - 1) * DT + dt) * 4 + b) * WAVE + lane] =
              make_float4(acc[dt][4 * b], acc[dt][4 * b + 1], acc[dt][4 * b + 2], acc[dt][4 * b + 3]);
    }
    __syncthreads();
    if (part == 0) {
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int b = 0; b < 4; ++b)
#pragma unroll
          for (int w = 0; w < W::SPLIT - 1; ++w) {
            const float4 v = box[((w * DT + dt) * 4 + b) * WAVE + lane];
            acc[dt][4 * b] += v.x;
            acc[dt][4 * b + 1] += v.y;
            acc[dt][4 * b + 2] += v.z;
            acc[dt][4 * b + 3] += v.w;
          }
    }
  }
}

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

// Boundaries of sequence n as any of its users takes them: clamped to the rows and to each other.
__device__ inline int2 sequence_span(const int32_t* cu, int n, int rows) {
  const int a = min(max(cu[n], 0), rows), b = min(max(cu[n + 1], a), rows);
  return make_int2(a, b - a);
}

// Entry `entry` of the list of tiles, found by every wave from the boundaries themselves, one sequence a lane (at most
// 64): sequences in order, a sequence's heaviest tile first, then what lies outside the sequences.
constexpr int FIND_MAX = WAVE;
template <int ROWS>
__device__ inline bool find_item(const AttnArgs& A, bool keys, int entry, AttnItem& it) {
  const int lane = threadIdx.x & (WAVE - 1), rows = (int)A.rows;
  int2 span = make_int2(0, 0);
  if (lane < A.N) span = sequence_span(A.bounds, lane, rows);
  const int tiles = (span.y + ROWS - 1) / ROWS;
  int upto = tiles;  // tiles of this and the earlier sequences
#pragma unroll
  for (int d = 1; d < WAVE; d <<= 1) {
    const int below = __shfl_up(upto, d, WAVE);
    if (lane >= d) upto += below;
  }
  const int total = __builtin_amdgcn_readlane(upto, WAVE - 1);
  it.seq = 0;
  if (entry < total) {
    const int n = __popcll(__ballot(upto <= entry));
    const int here = __builtin_amdgcn_readlane(tiles, n), at = entry - (__builtin_amdgcn_readlane(upto, n) - here);
    it.row0 = it.stat = __builtin_amdgcn_readlane(span.x, n);
    it.len = it.limit = __builtin_amdgcn_readlane(span.y, n);
    it.tile = keys ? at : here - 1 - at;
    return true;
  }
  const int first = A.N > 0 ? __builtin_amdgcn_readlane(span.x, 0) : 0;
  const int last = A.N > 0 ? __builtin_amdgcn_readlane(span.x + span.y, A.N - 1) : 0;
  const int head = (first + ROWS - 1) / ROWS;
  it.len = 0;
  it.tile = entry - total;
  if (it.tile < head) {
    it.row0 = it.stat = 0;
    it.limit = first;
  } else {
    it.tile -= head;
    it.row0 = it.stat = last;
    it.limit = rows - last;
  }
  return it.tile * ROWS < it.limit;
}

// keys: the workgroup owns key rows (of one key/value head for all its query heads, or for one of them; first tile
// heaviest) instead of query rows (one query head, last tile heaviest).
template <int ROWS>
__device__ inline bool attn_item(const AttnArgs& A, bool keys, AttnItem& it, int& kv_head, int& q_head) {
  const int group = keys && A.part_k == nullptr ? 1 : A.group;
  int g;
  if (A.bounds != nullptr) {
    const int per = A.Hk * group;
    if (!find_item<ROWS>(A, keys, blockIdx.x / per, it)) return false;
    spread_heads(blockIdx.x % per, A.Hk, group, kv_head, g);
  } else if (A.table != nullptr) {
    const int per = A.Hk * group;
    const int4 e = A.table[blockIdx.x / per];
    if (e.w <= 0) return false;
    spread_heads(blockIdx.x % per, A.Hk, group, kv_head, g);
    it.seq = 0;
    it.row0 = it.stat = e.x;
    it.len = e.y;
    it.limit = e.w;
    const int tiles = (e.y + ROWS - 1) / ROWS;
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
        if (in && d < D) store_chunk_any(out + d, Chunk<T>::pack(v));
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
        if (in && d < D) store_chunk_any(out + d, whole);
        if constexpr (REST) {
          float r[8];
          Chunk<T>::unpack(w, r);
#pragma unroll
          for (int e = 0; e < 8; ++e) r[e] = v[e] - r[e];
          const uint4 low = exchange(Chunk<T>::pack(r));
          if (in && d < D) store_chunk_any(rest + d, low);
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
    if (d < D) store_chunk_any(out + d, make_uint4(0u, 0u, 0u, 0u));
  }
}

template <typename T>
__device__ inline T* attn_row(const AttnView& v, const AttnItem& it, int head, int row) {
  return const_cast<T*>(attn_rows<T>(v, it, head)) + row * v.tok;
}

// first-operand fragments of one row kept in registers: row `row` of the workgroup's ROWS from `base`, of which `rows`
// exist (zeros past the end).  A buffer spans the workgroup's rows, never the sequence: its size is a 32-bit number.
template <typename T, int DP, int ROWS>
__device__ inline void load_own(const T* base, int64_t tok, int row, int rows, int D, int lane, uint4 (&f)[DP / (2 * Attn<T>::EPL)]) {
  constexpr int EPL = Attn<T>::EPL;
  const __amdgpu_buffer_rsrc_t r = row_buffer(base, tok, min(rows, ROWS), D);
#pragma unroll
  for (int ks = 0; ks < DP / (2 * EPL); ++ks) {
    const int col = (2 * ks + (lane >> 5)) * EPL;
    f[ks] = buffer_load16(r, col < D && row < rows ? (uint32_t)(row * (int)tok + col) * (uint32_t)sizeof(T) : NO_ROW);
  }
}

__device__ inline float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }

template <AttnKind KIND>
__device__ inline bool leaves_out(const AttnItem& it) {
  const bool brief = it.tile == 0 && it.len > 0 && it.len <= AT_SHORT;
  return KIND == AT_LONG ? brief : KIND == AT_BRIEF ? !brief : false;
}

// ---- forward -----------------------------------------------------------------------------------------------------
// SHORT: of a sequence of up to AT_SHORT rows; KIND: for which kernel (here and in the backward pass).  KIND only keeps the
// code of the kernels apart: shared between them, the compiler spilled registers in both (dq of 2 x 4096 positions, 32 / 8
// heads of 128, bf16: 428 -> 480 us).
template <typename T, int DP, int RW, AttnKind KIND, bool SHORT>
__device__ __forceinline__ void forward_rows(const AttnArgs& A, const AttnItem& it, int kvh, int qh, char* lds) {
  using M = Attn<T>;
  using W = Work<T, DP, RW>;
  constexpr bool FINE = W::FINE || SHORT;
  constexpr int BK = W::STEP, KS = DP / (2 * M::EPL), SUB = W::SUB, G = 32 / M::GROUP, DT = DP / 32;
  const int lane = threadIdx.x & (WAVE - 1), wave = threadIdx.x / WAVE;
  const int part = wave / RW;  // which of the waves that share rows
  const int first = it.tile * W::ROWS, mine = first + (wave % RW) * 32, row = mine + (lane & 31), half = lane >> 5;
  if (first >= it.len) {  // nothing of the sequence in this tile
    if (row < it.limit) zero_row<T, DP>(attn_row<T>(A.o, it, qh, row), A.D, lane);
    return;
  }
  const T* q = attn_rows<T>(A.q, it, qh);
  const T* k = attn_rows<T>(A.k, it, kvh);
  const T* v = attn_rows<T>(A.v, it, kvh);
  uint4 qf[KS];
  load_own<T, DP, W::ROWS>(q + first * A.q.tok, A.q.tok, row - first, it.len - first, A.D, lane, qf);
  f32x16 o[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[dt][i] = 0.f;
  float m = -INFINITY, l = 0.f;
  const float c = A.scale * AT_LOG2E;
  const int n_tiles = SHORT ? 1 : (min(first + W::ROWS, it.len) + BK - 1) / BK;
  // (a guard around the walk lets the compiler put q's loads behind it, and then every tile waits for the next one's: 4 x 1024
  // positions, 12 heads of 64, in the kernel of both kinds: 20.4 us with the guard, 19.4 without)
  if constexpr (KIND == AT_MIXED) __builtin_assume(n_tiles > 0);
  Staged<T, DP, BK> sk, sv;
  sk.init(A.k.tok, A.D);
  sv.init(A.v.tok, A.D);
  sk.load(k, A.k.tok, it.len, A.D);
  sv.load(v, A.v.tok, it.len, A.D);
  sk.store(lds);
  sv.store(lds + W::BYTES);
  for (int t = 0; t < n_tiles; ++t) {
    __syncthreads();  // this tile is in LDS, and nobody reads the other buffer any more
    const bool more = t + 1 < n_tiles;
    if (more) {
      const int next = (t + 1) * BK;
      sk.load(k + next * A.k.tok, A.k.tok, it.len - next, A.D);
      sv.load(v + next * A.v.tok, A.v.tok, it.len - next, A.D);
    }
    const char* buf = lds + (W::BUFFERS == 2 ? (t & 1) * 2 * W::BYTES : 0);
    const char* tk = buf + part * (SUB * 32) * Tile<T, DP>::PITCH;
    const char* tv = tk + W::BYTES;
    const int k0 = t * BK + part * (SUB * 32);
    if (k0 <= mine + 31 && mine < it.len) {
      f32x16 s[SUB];
#pragma unroll
      for (int u = 0; u < SUB; ++u) {
#pragma unroll
        for (int i = 0; i < 16; ++i) s[u][i] = 0.f;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) Mma32<T>::mma(read_rows<T, DP>(tk, u * 32, ks, lane), qf[ks], s[u]);
      }
      if (k0 + SUB * 32 - 1 > mine) {  // the tile reaches past some row's own position
        const int last = row - k0 - 4 * half;
#pragma unroll
        for (int u = 0; u < SUB; ++u)
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (u * 32 + 8 * (i / 4) + i % 4 > last) s[u][i] = -INFINITY;
      }
      float top = m;
#pragma unroll
      for (int u = 0; u < SUB; ++u)
#pragma unroll
        for (int i = 0; i < 16; ++i) top = fmaxf(top, s[u][i]);
      const float2 halves = both_halves(top);
      top = fmaxf(halves.x, halves.y);
      // The shift of the exponents follows the maximum only when it is 2^8 behind for some row: weights up to 2^8
      // round like smaller ones, and what has been summed is rescaled a few times a row instead of at most tiles.
      if (__any((top - m) * c > 8.f)) {
        const float f = top == -INFINITY ? 0.f : exp2_of((m - top) * c);
        l *= f;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
          for (int i = 0; i < 16; ++i) o[dt][i] *= f;
        m = top;
      }
      // a row all of whose scores so far are -inf keeps a maximum of -inf; its weights are 0, not 0 - 0
      // (and where the factor takes the type's lowest value past the numbers, its weights become 0, not inf - inf)
      const float shift = m == -INFINITY ? 0.f : fmaxf(m * c, -FLT_MAX);
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
          uint4 rest = p;
          if constexpr (FINE) rest = pack_rest<T>(s[u], g, p);
#pragma unroll
          for (int dt = 0; dt < DT; ++dt) {
            const uint4 a = M::template read_tr<DP>(tv, u * 32 + g * M::GROUP, dt, lane);
            Mma32<T>::mma(a, p, o[dt]);
            if constexpr (FINE) Mma32<T>::mma(a, rest, o[dt]);
          }
        }
    }
    if constexpr (W::BUFFERS == 1) __syncthreads();
    if (more) {
      char* next = lds + (W::BUFFERS == 2 ? ((t + 1) & 1) * 2 * W::BYTES : 0);
      sk.store(next);
      sv.store(next + W::BYTES);
    }
  }
  const float2 ls = both_halves(l);
  l = ls.x + ls.y;
  if constexpr (W::SPLIT > 1) {  // bring the waves' sums to the largest maximum of them
    __shared__ float maxima[AT_WAVES][WAVE], sums[AT_WAVES][WAVE];
    maxima[wave][lane] = m;
    __syncthreads();
    float top = m;
#pragma unroll
    for (int w = 0; w < W::SPLIT; ++w) top = fmaxf(top, maxima[w * RW + wave % RW][lane]);
    const float f = m == -INFINITY ? 0.f : exp2_of((m - top) * c);
    m = top;
    l *= f;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[dt][i] *= f;
    sums[wave][lane] = l;
    join_waves<W, DT>(o, lds, part, wave % RW, lane);
    if (part > 0) return;
#pragma unroll
    for (int w = 1; w < W::SPLIT; ++w) l += sums[w * RW + wave % RW][lane];
  }
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

template <typename T, int DP, int RW, AttnKind KIND>
__global__ __launch_bounds__(AT_THREADS, (Work<T, DP, RW>::PER_SIMD_Q)) void attention_forward_kernel(AttnArgs A) {
  using W = Work<T, DP, RW>;
  __shared__ __attribute__((aligned(16))) char lds[W::LDS];
  AttnItem it;
  int kvh, qh;
  if (!attn_item<W::ROWS>(A, false, it, kvh, qh)) return;
  if (leaves_out<KIND>(it)) return;
  if constexpr (KIND == AT_MIXED || KIND == AT_BRIEF) {
    if (KIND == AT_BRIEF || it.len <= AT_SHORT) {
      forward_rows<T, DP, RW, KIND, true>(A, it, kvh, qh, lds);
      return;
    }
  }
  if constexpr (KIND != AT_BRIEF) forward_rows<T, DP, RW, KIND, false>(A, it, kvh, qh, lds);
}

// ---- backward: queries -------------------------------------------------------------------------------------------
// dq of 32 queries a wave; also leaves delta (and, for fp16, a bound of the row's |dS|) for the other kernel.
//
// fp16 holds numbers of 2^-14 to 2^16, and dS may be of any size: small with the gradients, large with the values, small
// where the weights spread.  A row's dS is at most its largest |dp - delta| times the largest weight that a shift
// which lags by 2^8 and the weights' sum allow.  It carries the power of two that brings this bound to 2^12, set by the row's first
// block and, with what has been summed, lowered when a later one brings the bound past 2^15: what is lost among
// the subnormals is 2^-37 of the bound.  The power stands in the exponent of P, at no cost; what this takes is the
// largest of 16 values a block and a vote (24 documents of 16 to 2048 positions, 16 heads of 64: 58 -> 63 us).
constexpr int DS_FIRST = 12, DS_MOST = 15;
constexpr float DS_LIFT_MAX = 60.f;  // fp32 keeps weights up to 2^8 times |do| |v| of 2^40 times that

template <typename T, int DP, int RW, AttnKind KIND, bool SHORT>
__device__ __forceinline__ void backward_q_rows(const AttnArgs& A, const AttnItem& it, int kvh, int qh, char* lds) {
  using M = Attn<T>;
  using W = Work<T, DP, RW>;
  constexpr bool FINE = W::FINE || SHORT;
  constexpr bool HALF = std::is_same<T, f16_t>::value;
  constexpr int BK = W::STEP, KS = DP / (2 * M::EPL), SUB = W::SUB, G = 32 / M::GROUP, DT = DP / 32;
  const int lane = threadIdx.x & (WAVE - 1), wave = threadIdx.x / WAVE;
  const int part = wave / RW;  // which of the waves that share rows
  const int first = it.tile * W::ROWS, mine = first + (wave % RW) * 32, row = mine + (lane & 31), half = lane >> 5;
  if (first >= it.len) {  // nothing of the sequence in this tile
    if (row < it.limit) zero_row<T, DP>(attn_row<T>(A.dq, it, qh, row), A.D, lane);
    return;
  }
  const bool in = row < it.len;
  const T* k = attn_rows<T>(A.k, it, kvh);
  const T* v = attn_rows<T>(A.v, it, kvh);
  uint4 qf[KS], gf[KS];
  const int own = row - first, left = it.len - first;
  const int64_t stat = (int64_t)qh * A.rows + it.stat + row;
  // everything the walk starts with is on its way before the first value is used
  load_own<T, DP, W::ROWS>(attn_rows<T>(A.grad_o, it, qh) + first * A.grad_o.tok, A.grad_o.tok, own, left, A.D, lane, gf);
  const float shift = in ? A.shift[stat] : 0.f, sum = in ? A.sum[stat] : 1.f;
  Staged<T, DP, BK> sk, sv;
  sk.init(A.k.tok, A.D);
  sv.init(A.v.tok, A.D);
  float delta = 0.f;
  {
    uint4 of[KS], rf[KS];
    load_own<T, DP, W::ROWS>(attn_rows<T>(A.o, it, qh) + first * A.o.tok, A.o.tok, own, left, A.D, lane, of);
    if constexpr (sizeof(T) == 2)
      load_own<T, DP, W::ROWS>((const T*)A.rest + ((it.stat + first) * A.Hq + qh) * A.D, (int64_t)A.Hq * A.D, own, left, A.D, lane, rf);
    load_own<T, DP, W::ROWS>(attn_rows<T>(A.q, it, qh) + first * A.q.tok, A.q.tok, own, left, A.D, lane, qf);
    sk.load(k, A.k.tok, it.len, A.D);
    sv.load(v, A.v.tok, it.len, A.D);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      float a[M::EPL], b[M::EPL];
      Chunk<T>::unpack(of[ks], a);
      Chunk<T>::unpack(gf[ks], b);
      if constexpr (sizeof(T) == 2) {  // delta stands against dp in fp32: it needs o unrounded
        float r[M::EPL];
        Chunk<T>::unpack(rf[ks], r);
#pragma unroll
        for (int e = 0; e < M::EPL; ++e) a[e] += r[e];
      }
#pragma unroll
      for (int e = 0; e < M::EPL; ++e) delta = fmaf(a[e], b[e], delta);
    }
    const float2 d = both_halves(delta);
    delta = d.x + d.y;
  }
  if (in && half == 0 && part == 0) A.delta[stat] = delta;
  // fp16: the power of two of dS stands in `arg` (as far as fp32 holds their sum: it is what arg and the shift say, to the
  // end); `room` is the |dp - delta| it has room for, `most` the largest so far
  float arg = -shift, room = 0.f, most = 0.f;
  const float over_sum = 1.0f / sum, heaviest = fminf(sum, 256.f);
  const float c = A.scale * AT_LOG2E;
  f32x16 dq[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int i = 0; i < 16; ++i) dq[dt][i] = 0.f;
  const int n_tiles = SHORT ? 1 : (min(first + W::ROWS, it.len) + BK - 1) / BK;
  sk.store(lds);
  sv.store(lds + W::BYTES);
  for (int t = 0; t < n_tiles; ++t) {
    __syncthreads();
    const bool more = t + 1 < n_tiles;
    if (more) {
      const int next = (t + 1) * BK;
      sk.load(k + next * A.k.tok, A.k.tok, it.len - next, A.D);
      sv.load(v + next * A.v.tok, A.v.tok, it.len - next, A.D);
    }
    const char* buf = lds + (W::BUFFERS == 2 ? (t & 1) * 2 * W::BYTES : 0);
    const char* tk = buf + part * (SUB * 32) * Tile<T, DP>::PITCH;
    const char* tv = tk + W::BYTES;
    const int k0 = t * BK + part * (SUB * 32);
    if (k0 <= mine + 31 && mine < it.len) {
#pragma unroll DP > 96 || (HALF && KIND == AT_MIXED && DP == 64) ? 1 : SUB  // registers
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
        // a sequence's first row has one key and a constant softmax: its dS is 0, not the rounding of dp - delta
        const bool diagonal = k0 + u * 32 + 31 > mine;
        const int last = (row == 0 ? -1 : row) - k0 - u * 32 - 4 * half;
        if constexpr (HALF) {
          if (diagonal) {  // what is not seen does not count
#pragma unroll
            for (int i = 0; i < 16; ++i)
              if (8 * (i / 4) + i % 4 > last) dp[i] = 0.f;
          }
          float big = most;
#pragma unroll
          for (int i = 0; i < 16; ++i) big = fmaxf(big, fabsf(dp[i]));
          const float2 halves = both_halves(big);
          most = fmaxf(halves.x, halves.y);
          if (__any(most > room)) {
            const bool change = most > room && most < INFINITY;
            const float lift = fminf((float)(DS_FIRST - ilogbf(most * heaviest)), DS_LIFT_MAX);
            const float to = change ? lift - shift : arg, f = exp2_of(to - arg);
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
              for (int i = 0; i < 16; ++i) dq[dt][i] *= f;
            arg = to;
            if (change) room = exp2_of(DS_MOST - lift) / heaviest;
          }
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] = exp2_of(fmaf(s[i], c, arg)) * dp[i];
        if (diagonal) {
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (8 * (i / 4) + i % 4 > last) s[i] = 0.f;
        }
#pragma unroll
        for (int g = 0; g < G; ++g) {
          const uint4 ds = M::pack(s, g);
          uint4 rest = ds;
          if constexpr (FINE) rest = pack_rest<T>(s, g, ds);
#pragma unroll
          for (int dt = 0; dt < DT; ++dt) {
            const uint4 a = M::template read_tr<DP>(tk, u * 32 + g * M::GROUP, dt, lane);
            Mma32<T>::mma(a, ds, dq[dt]);
            if constexpr (FINE) Mma32<T>::mma(a, rest, dq[dt]);
          }
        }
      }
    }
    if constexpr (W::BUFFERS == 1) __syncthreads();
    if (more) {
      char* next = lds + (W::BUFFERS == 2 ? ((t + 1) & 1) * 2 * W::BYTES : 0);
      sk.store(next);
      sv.store(next + W::BYTES);
    }
  }
  float unlift = 1.f;
  if constexpr (HALF) {
    unlift = exp2_of(-(arg + shift));
    if constexpr (W::SPLIT > 1) {  // the waves' powers of two may differ
      __shared__ float largest[AT_WAVES][WAVE];
      largest[wave][lane] = most;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int i = 0; i < 16; ++i) dq[dt][i] *= unlift;
      unlift = 1.f;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < W::SPLIT; ++w) most = fmaxf(most, largest[w * RW + wave % RW][lane]);
    }
    // (a row with infinities has no dS that would have to fit)
    if (in && half == 0 && part == 0) A.peak[stat] = most < INFINITY ? most * heaviest * over_sum : 0.f;
  }
  join_waves<W, DT>(dq, lds, part, wave % RW, lane);
  if (part > 0) return;
  T* out = attn_row<T>(A.dq, it, qh, row);
  store_rows<T, DP>(out, nullptr, dq, A.scale * over_sum * unlift, in, A.D, lane);
  if (!in && row < it.limit) zero_row<T, DP>(out, A.D, lane);
}

template <typename T, int DP, int RW, AttnKind KIND>
__global__ __launch_bounds__(AT_THREADS, (Work<T, DP, RW>::PER_SIMD_Q)) void attention_backward_q_kernel(AttnArgs A) {
  using W = Work<T, DP, RW>;
  __shared__ __attribute__((aligned(16))) char lds[W::LDS];
  AttnItem it;
  int kvh, qh;
  if (!attn_item<W::ROWS>(A, false, it, kvh, qh)) return;
  if (leaves_out<KIND>(it)) return;
  if constexpr (KIND == AT_MIXED || KIND == AT_BRIEF) {
    if (KIND == AT_BRIEF || it.len <= AT_SHORT) {
      backward_q_rows<T, DP, RW, KIND, true>(A, it, kvh, qh, lds);
      return;
    }
  }
  if constexpr (KIND != AT_BRIEF) backward_q_rows<T, DP, RW, KIND, false>(A, it, kvh, qh, lds);
}

// ---- backward: keys and values -----------------------------------------------------------------------------------
// Wide heads at 16 bits with enough keys (RW = 4, DP > 64): dk and dv of 32 keys take half of a wave's registers, and with
// k, v and a tile on its way in the other half only one wave fits a SIMD, which then waits for every LDS read and every
// exponential itself (643 TFLOP/s of the four products at 2 x 4096 positions, 32 / 8 heads of 128).  There the
// workgroup has eight waves, two for the same 32 keys that take the queries of a tile in halves, and k and v are read
// from LDS as the products need them.
template <typename T, int DP, int RW>
constexpr int kv_waves() {
  return RW == 4 && DP > 64 && sizeof(T) == 2 ? 8 : AT_WAVES;
}

// What the workgroup has in LDS.
template <typename T, int DP, int RW>
struct KvStore {
  using W = Work<T, DP, RW, kv_waves<T, DP, RW>()>;
  static constexpr bool OWN = W::THREADS > AT_THREADS;  // k and v of the workgroup's keys live here
  static constexpr int KEEP = OWN ? W::ROWS * Tile<T, DP>::PITCH : 0;
  static constexpr int NSTAT = std::is_same<T, f16_t>::value ? 4 : 3;
  __attribute__((aligned(16))) char lds[W::LDS];
  __attribute__((aligned(16))) char keep[OWN ? 2 * KEEP : 16];
  __attribute__((aligned(16))) float stats[W::BUFFERS][NSTAT][W::STEP];
};

// dk and dv of one key tile become zero: of the key/value head, or the parts of one query head (alone)
template <typename T, int DP>
__device__ inline void clear_kv(const AttnArgs& A, const AttnItem& it, int kvh, int qh, int row, int lane) {
  if (A.part_k != nullptr) {
    const int64_t part_row = ((it.stat + row) * A.Hq + qh) * A.D;
    zero_row<float, DP>(A.part_k + part_row, A.D, lane);
    zero_row<float, DP>(A.part_v + part_row, A.D, lane);
  } else {
    zero_row<T, DP>(attn_row<T>(A.dk, it, kvh, row), A.D, lane);
    zero_row<T, DP>(attn_row<T>(A.dv, it, kvh, row), A.D, lane);
  }
}

template <typename T, int DP, int RW, AttnKind KIND, bool SHORT>
__device__ __forceinline__ void backward_kv_rows(const AttnArgs& A, const AttnItem& it, int kvh, int qh0, KvStore<T, DP, RW>& store_in) {
  using M = Attn<T>;
  using Store = KvStore<T, DP, RW>;
  using W = typename Store::W;
  constexpr bool FINE = W::FINE || SHORT;  // dS as two operands
  constexpr bool OWN = Store::OWN;
  constexpr bool HALF = std::is_same<T, f16_t>::value;
  // fp16: P goes in 2^14 times its value, or the weights of long flat sequences would be subnormal numbers (at 32768
  // positions alike dv was 2.5 times as far off as its own rounding; 2^14 leaves room for a P that rounding takes past 1)
  constexpr float P_LIFT = HALF ? 14.f : 0.f;
  constexpr int BQ = W::STEP, KS = DP / (2 * M::EPL), SUB = W::SUB, G = 32 / M::GROUP, DT = DP / 32;
  constexpr int KEEP = Store::KEEP;
  char *lds = store_in.lds, *keep = store_in.keep;
  auto& stats = store_in.stats;
  const int lane = threadIdx.x & (WAVE - 1), wave = threadIdx.x / WAVE;
  const int part = wave / RW;  // which of the waves that share rows
  const int first = it.tile * W::ROWS, mine = first + (wave % RW) * 32, row = mine + (lane & 31), half = lane >> 5;
  const bool alone = A.part_k != nullptr;  // one query head of the group
  const int64_t part_row = ((it.stat + row) * A.Hq + qh0) * A.D;
  if (first >= it.len) {
    if (row < it.limit) clear_kv<T, DP>(A, it, kvh, qh0, row, lane);
    return;
  }
  const bool in = row < it.len;
  uint4 kf[OWN ? 1 : KS], vf[OWN ? 1 : KS];
  const int own = row - first, left = it.len - first;
  const T* k = attn_rows<T>(A.k, it, kvh) + first * A.k.tok;
  const T* v = attn_rows<T>(A.v, it, kvh) + first * A.v.tok;
  if constexpr (OWN) {
    Staged<T, DP, W::ROWS, W::THREADS> once;
    once.init(A.k.tok, A.D);
    once.load(k, A.k.tok, left, A.D);
    once.store(keep);
    once.init(A.v.tok, A.D);
    once.load(v, A.v.tok, left, A.D);
    once.store(keep + KEEP);
  } else {
    load_own<T, DP, W::ROWS>(k, A.k.tok, own, left, A.D, lane, kf);
    load_own<T, DP, W::ROWS>(v, A.v.tok, own, left, A.D, lane, vf);
  }
  f32x16 dk[DT], dv[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int i = 0; i < 16; ++i) dk[dt][i] = dv[dt][i] = 0.f;
  const float c = A.scale * AT_LOG2E;
  const int t0 = SHORT ? 0 : first / BQ, per_head = SHORT ? 1 : (it.len + BQ - 1) / BQ - t0, n_tiles = alone ? per_head : per_head * A.group;
  Staged<T, DP, BQ, W::THREADS> sq, sg;
  float stage[4];
  // tile t is tile t % per_head of the queries, for query head t / per_head of the group
  int load_head = qh0, load_tile = t0;
  auto load = [&]() {
    const int q0 = load_tile * BQ, rows = it.len - q0;
    sq.load(attn_rows<T>(A.q, it, load_head) + q0 * A.q.tok, A.q.tok, rows, A.D);
    sg.load(attn_rows<T>(A.grad_o, it, load_head) + q0 * A.grad_o.tok, A.grad_o.tok, rows, A.D);
    const int64_t stat = (int64_t)load_head * A.rows + it.stat + q0;
    const uint32_t mine4 = threadIdx.x < BQ ? threadIdx.x * 4 : NO_ROW;
    const int n = min(rows, BQ);
    stage[0] = buffer_load4(row_buffer(A.shift + stat, 1, n, 1), mine4);
    stage[1] = buffer_load4(row_buffer(A.delta + stat, 1, n, 1), mine4);
    stage[2] = buffer_load4(row_buffer(A.sum + stat, 1, n, 1), mine4);
    if constexpr (HALF) stage[3] = buffer_load4(row_buffer(A.peak + stat, 1, n, 1), mine4);
    if (++load_tile == t0 + per_head) {
      load_tile = t0;
      ++load_head;
    }
  };
  auto store = [&](int b) {
    sq.store(lds + b * 2 * W::BYTES);
    sg.store(lds + b * 2 * W::BYTES + W::BYTES);
    if (threadIdx.x < BQ) {
      const float sum = stage[2] == 0.f ? 1.f : stage[2];  // rows past the end read as zeros
      stats[b][0][threadIdx.x] = stage[0];
      stats[b][1][threadIdx.x] = stage[1];
      stats[b][2][threadIdx.x] = exp2_of(P_LIFT) / sum;  // a factor of its own: see AttnArgs
      if constexpr (HALF) stats[b][3][threadIdx.x] = stage[3];
    }
  };
  // fp16: dS carries a power of two here too, the one that brings the largest of the rows' bounds so far to 2^14; when a
  // tile brings a larger one, what has been summed is rescaled (exactly) to the new power.
  int lift = 0;
  bool lifted = false;
  sq.init(A.q.tok, A.D);
  sg.init(A.grad_o.tok, A.D);
  load();
  store(0);
  int tile = t0;
  for (int t = 0; t < n_tiles; ++t) {
    __syncthreads();
    const bool more = t + 1 < n_tiles;
    if (more) load();
    const int b = W::BUFFERS == 2 ? t & 1 : 0, skip = part * (SUB * 32);
    const char* tq = lds + b * 2 * W::BYTES + skip * Tile<T, DP>::PITCH;
    const char* tg = tq + W::BYTES;
    const float(*st)[BQ] = stats[b];
    const int q0 = tile * BQ + skip;
    if (++tile == t0 + per_head) tile = t0;
    if (q0 + SUB * 32 > mine && mine < it.len) {
      float raise = 1.f;
      if constexpr (HALF) {
        const float peak = wave_max(st[3][skip + lane % (SUB * 32)]);
        if (peak > 0.f && peak < INFINITY) {
          const int want = min(DS_MOST - 1 - ilogbf(peak), (int)DS_LIFT_MAX);
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
        raise = exp2_of((float)lift - P_LIFT);
      }
#pragma unroll 1
      for (int u = 0; u < SUB; ++u) {
        if (q0 + u * 32 + 31 < mine) continue;  // all of these queries come before this wave's keys
        f32x16 s, dp;
        float shift[16];
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          const float4 a = *reinterpret_cast<const float4*>(&st[0][skip + u * 32 + 8 * b + 4 * half]);
          const float4 d = *reinterpret_cast<const float4*>(&st[1][skip + u * 32 + 8 * b + 4 * half]);
          shift[4 * b] = a.x, shift[4 * b + 1] = a.y, shift[4 * b + 2] = a.z, shift[4 * b + 3] = a.w;
          dp[4 * b] = -d.x, dp[4 * b + 1] = -d.y, dp[4 * b + 2] = -d.z, dp[4 * b + 3] = -d.w;
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] = 0.f;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          if constexpr (OWN) {
            Mma32<T>::mma(read_rows<T, DP>(tq, u * 32, ks, lane), read_rows<T, DP>(keep, mine - first, ks, lane), s);
            Mma32<T>::mma(read_rows<T, DP>(tg, u * 32, ks, lane), read_rows<T, DP>(keep + KEEP, mine - first, ks, lane), dp);
          } else {
            Mma32<T>::mma(read_rows<T, DP>(tq, u * 32, ks, lane), kf[ks], s);
            Mma32<T>::mma(read_rows<T, DP>(tg, u * 32, ks, lane), vf[ks], dp);
          }
        }
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          // read here and no earlier: beside the products there are no registers for it at heads of 128 (2 x 4096 positions,
          // 32 / 8 heads, bf16: 691 us with the read in front of them, 638 where the compiler puts it, 598 this way)
          __builtin_amdgcn_sched_barrier(0);
          const float4 w = *reinterpret_cast<const float4*>(&st[2][skip + u * 32 + 8 * b + 4 * half]);
          const float over_sum[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int i = 4 * b + e;
            s[i] = exp2_of(fmaf(s[i], c, -shift[i])) * over_sum[e];
            dp[i] = HALF ? s[i] * raise * dp[i] : s[i] * dp[i];
          }
        }
        if (q0 + u * 32 < mine + 31) {
          const int first_query = row - q0 - u * 32 - 4 * half;
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (8 * (i / 4) + i % 4 < first_query) s[i] = dp[i] = 0.f;
          // a sequence's first row has one key and a constant softmax: its dS is 0, not the rounding of dp - delta
          if (q0 + u * 32 == 0 && half == 0) dp[0] = 0.f;
        }
#pragma unroll
        for (int g = 0; g < G; ++g) {
          const uint4 p = M::pack(s, g), ds = M::pack(dp, g);
          uint4 p_rest = p, ds_rest = ds;
          if constexpr (W::FINE) p_rest = pack_rest<T>(s, g, p);
          if constexpr (FINE) ds_rest = pack_rest<T>(dp, g, ds);
#pragma unroll
          for (int dt = 0; dt < DT; ++dt) {
            const uint4 a = M::template read_tr<DP>(tg, u * 32 + g * M::GROUP, dt, lane);
            const uint4 b = M::template read_tr<DP>(tq, u * 32 + g * M::GROUP, dt, lane);
            Mma32<T>::mma(a, p, dv[dt]);
            Mma32<T>::mma(b, ds, dk[dt]);
            if constexpr (W::FINE) Mma32<T>::mma(a, p_rest, dv[dt]);
            if constexpr (FINE) Mma32<T>::mma(b, ds_rest, dk[dt]);
          }
        }
      }
    }
    if constexpr (W::BUFFERS == 1) __syncthreads();
    if (more) store(W::BUFFERS == 2 ? (t + 1) & 1 : 0);
  }
  if constexpr (HALF && W::SPLIT > 1) {  // the waves' powers of two may differ
    const float f = exp2_of(-(float)lift);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int i = 0; i < 16; ++i) dk[dt][i] *= f;
    lift = 0;
  }
  join_waves<W, DT>(dk, lds, part, wave % RW, lane);
  join_waves<W, DT>(dv, lds, part, wave % RW, lane);
  if (part > 0) return;
  const float scale = A.scale * exp2_of(-(float)lift), scale_v = exp2_of(-P_LIFT);
  if (alone) {
    store_rows<float, DP>(A.part_k + part_row, nullptr, dk, scale, in, A.D, lane);
    store_rows<float, DP>(A.part_v + part_row, nullptr, dv, scale_v, in, A.D, lane);
  } else {
    store_rows<T, DP>(attn_row<T>(A.dk, it, kvh, row), nullptr, dk, scale, in, A.D, lane);
    store_rows<T, DP>(attn_row<T>(A.dv, it, kvh, row), nullptr, dv, scale_v, in, A.D, lane);
  }
  if (!in && row < it.limit) clear_kv<T, DP>(A, it, kvh, qh0, row, lane);
}

template <typename T, int DP, int RW, AttnKind KIND>
__global__ __launch_bounds__((kv_waves<T, DP, RW>() * WAVE),
                             (Work<T, DP, RW, kv_waves<T, DP, RW>()>::PER_SIMD_KV)) void attention_backward_kv_kernel(AttnArgs A) {
  using W = typename KvStore<T, DP, RW>::W;
  __shared__ KvStore<T, DP, RW> store;
  AttnItem it;
  int kvh, qh;
  if (!attn_item<W::ROWS>(A, true, it, kvh, qh)) return;
  if (leaves_out<KIND>(it)) return;
  if constexpr (KIND == AT_MIXED || KIND == AT_BRIEF) {
    if (KIND == AT_BRIEF || it.len <= AT_SHORT) {
      backward_kv_rows<T, DP, RW, KIND, true>(A, it, kvh, qh, store);
      return;
    }
  }
  if constexpr (KIND != AT_BRIEF) backward_kv_rows<T, DP, RW, KIND, false>(A, it, kvh, qh, store);
}

// dk and dv of every key/value head: the sums over its query heads in their order, rounded once.  One thread per 16
// bytes of the fp32 parts; grid.y = 0: dk, 1: dv.
template <typename T>
__global__ __launch_bounds__(256) void attention_backward_join_kernel(AttnArgs A) {
  const int pieces = A.D / 4;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= A.rows * A.Hk * pieces) return;
  const int d = (int)(i % pieces) * 4, head = (int)(i / pieces % A.Hk);
  const int64_t row = i / pieces / A.Hk;
  const float* part = (blockIdx.y == 0 ? A.part_k : A.part_v) + (row * A.Hq + (int64_t)head * A.group) * A.D + d;
  float4 s = *reinterpret_cast<const float4*>(part);
  for (int g = 1; g < A.group; ++g) {
    const float4 v = *reinterpret_cast<const float4*>(part + (int64_t)g * A.D);
    s.x += v.x;
    s.y += v.y;
    s.z += v.z;
    s.w += v.w;
  }
  const AttnView& view = blockIdx.y == 0 ? A.dk : A.dv;
  const int64_t seq = A.S > 0 ? row / A.S : 0, at = A.S > 0 ? row % A.S : row;
  T* out = (T*)const_cast<void*>(view.p) + seq * view.seq + at * view.tok + head * view.head + d;
  store_as(out, 0, s.x, Elem<T>::code);
  store_as(out, 1, s.y, Elem<T>::code);
  store_as(out, 2, s.z, Elem<T>::code);
  store_as(out, 3, s.w, Elem<T>::code);
}

// ---- packed sequences: the list of tiles -------------------------------------------------------------------------
// One entry per tile of a sequence, entries of a higher tile (more of the other side to walk) first, and entries that
// only clear the rows outside every sequence; one list per tile height, each made by one workgroup.  The sequences'
// ends are device data: they are clamped to the packed rows and to each other, and an entry that would not fit in the
// list is dropped, so that no boundaries lead out of bounds.
constexpr int PLAN_THREADS = 1024;

// sum of v over the threads from this one on
__device__ inline int suffix_sum(int v, int* waves) {
  const int lane = threadIdx.x & (WAVE - 1), wave = threadIdx.x / WAVE;
#pragma unroll
  for (int d = 1; d < WAVE; d <<= 1) {
    const int up = __shfl_down(v, d, WAVE);
    if (lane + d < WAVE) v += up;
  }
  __syncthreads();
  if (lane == 0) waves[wave] = v;
  __syncthreads();
  int later = lane > wave && lane < PLAN_THREADS / WAVE ? waves[lane] : 0;  // the waves after this one
#pragma unroll
  for (int d = 1; d < PLAN_THREADS / WAVE; d <<= 1) later += __shfl_xor(later, d, WAVE);
  return v + __shfl(later, 0, WAVE);
}

__global__ __launch_bounds__(PLAN_THREADS) void attention_plan_kernel(const int32_t* __restrict__ cu, int N, int rows,
                                                                      int4* tables, int entries0, int entries1,
                                                                      int entries2) {
  // a level is a tile's index, or 2^fold of them where there are more levels than threads
  __shared__ int whole[PLAN_THREADS], partial[PLAN_THREADS], cursor[PLAN_THREADS], waves[PLAN_THREADS / WAVE];
  __shared__ int total;
  const int height = AT_TILES[blockIdx.x], entries = blockIdx.x == 0 ? entries0 : blockIdx.x == 1 ? entries1 : entries2;
  int4* table = tables + (blockIdx.x == 0 ? 0 : blockIdx.x == 1 ? entries0 : entries0 + entries1);
  auto tiles_of = [&](int length) { return (length + height - 1) / height; };
  int fold = 0;
  while ((tiles_of(rows) >> fold) >= PLAN_THREADS) ++fold;
  whole[threadIdx.x] = partial[threadIdx.x] = 0;
  __syncthreads();
  for (int n = threadIdx.x; n < N; n += PLAN_THREADS) {
    const int tiles = tiles_of(sequence_span(cu, n, rows).y);
    if (tiles > 0) {
      atomicAdd(&whole[tiles >> fold], 1);  // levels below this one it fills, this one in part
      if (fold > 0) atomicAdd(&partial[tiles >> fold], tiles & ((1 << fold) - 1));
    }
  }
  __syncthreads();
  // tiles of a level: 2^fold of every sequence that reaches past it, and what ends in it
  const int reach = suffix_sum(whole[threadIdx.x], waves) - whole[threadIdx.x];
  const int here = (reach << fold) + partial[threadIdx.x];
  const int from_here = suffix_sum(here, waves);
  cursor[threadIdx.x] = from_here - here;
  if (threadIdx.x == 0) total = from_here;
  __syncthreads();
  // within a level the order is whatever the counters hand out: it decides when a tile runs, not what it computes
  const int lane = threadIdx.x & (WAVE - 1), wave = threadIdx.x / WAVE;
  for (int n = wave; n < N; n += PLAN_THREADS / WAVE) {
    const int2 s = sequence_span(cu, n, rows);
    for (int t = lane; t < tiles_of(s.y); t += WAVE) {
      const int at = atomicAdd(&cursor[t >> fold], 1);
      if ((unsigned)at < (unsigned)entries) table[at] = make_int4(s.x, s.y, t, s.y);
    }
  }
  // rows before the first and after the last sequence, then entries without work
  const int head = N > 0 ? sequence_span(cu, 0, rows).x : 0;
  const int2 last = N > 0 ? sequence_span(cu, N - 1, rows) : make_int2(0, 0);
  const int tail = last.x + last.y, head_tiles = tiles_of(head), clear = head_tiles + tiles_of(rows - tail);
  for (int at = total + (int)threadIdx.x; at < entries; at += PLAN_THREADS) {
    if (at < 0) break;
    const int i = at - total;
    table[at] = i >= clear       ? make_int4(0, 0, 0, 0)
                : i < head_tiles ? make_int4(0, 0, i, head)
                                 : make_int4(tail, 0, i - head_tiles, rows - tail);
  }
}

static int64_t plan_entries(int64_t rows, int n_seqs, int which) { return rows / AT_TILES[which] + n_seqs + 2; }

// ---- host side ---------------------------------------------------------------------------------------------------
static int attn_check(const bgx_attention_shape* a, const char* what) {
  BGX_REQUIRE(a != nullptr, BGX_E_ARG, "%s: null shape", what);
  BGX_REQUIRE(a->n_seqs >= 0 && a->rows >= 0, BGX_E_ARG, "%s: n_seqs=%d rows=%lld", what, a->n_seqs, (long long)a->rows);
  BGX_REQUIRE(a->heads >= 1 && a->kv_heads >= 1 && a->heads % a->kv_heads == 0, BGX_E_SHAPE,
              "%s: %d query heads on %d key/value heads", what, a->heads, a->kv_heads);
  BGX_REQUIRE(a->head_dim >= 1 && a->head_dim <= AT_MAX_D, BGX_E_SHAPE, "%s: head_dim=%d, supported are 1 to %d", what,
              a->head_dim, AT_MAX_D);
  BGX_REQUIRE(a->dtype >= BGX_F32 && a->dtype <= BGX_BF16, BGX_E_DTYPE, "%s: dtype %d", what, a->dtype);
  BGX_REQUIRE(a->head_dim % (16 / (int)dtype_size(a->dtype)) == 0, BGX_E_SHAPE,
              "%s: head_dim=%d is not whole 16-byte pieces; pad it with zeros", what, a->head_dim);
  BGX_REQUIRE(a->scale > 0.f && a->scale < INFINITY, BGX_E_ARG, "%s: scale %g must be positive and finite", what, a->scale);
  // tile bounds are formed in 32 bits
  BGX_REQUIRE(a->rows < (1ll << 31) - 4 * AT_TILES[0], BGX_E_SHAPE, "%s: %lld rows", what, (long long)a->rows);
  BGX_REQUIRE(a->cu_seqlens_dev == nullptr || (a->plan_dev == nullptr && a->n_seqs <= FIND_MAX), BGX_E_ARG,
              "%s: boundaries of %d sequences; up to %d go without a plan", what, a->n_seqs, FIND_MAX);
  if (a->plan_dev == nullptr && a->cu_seqlens_dev == nullptr)
    BGX_REQUIRE(a->n_seqs == 0 ? a->rows == 0 : a->rows % a->n_seqs == 0, BGX_E_ARG,
                "%s: %lld rows are not %d sequences of one width", what, (long long)a->rows, a->n_seqs);
  return 0;
}

// tiles of the given height, over all sequences
static int64_t attn_items(const bgx_attention_shape* a, int which) {
  if (a->plan_dev != nullptr || a->cu_seqlens_dev != nullptr) return plan_entries(a->rows, a->n_seqs, which);
  const int64_t S = a->n_seqs ? a->rows / a->n_seqs : 0;
  return (S + AT_TILES[which] - 1) / AT_TILES[which] * a->n_seqs;
}

static AttnArgs attn_args(const bgx_attention_shape* a) {
  AttnArgs A{};
  A.bounds = a->cu_seqlens_dev;
  A.lengths = a->lengths_dev;
  A.rows = a->rows;
  A.N = a->n_seqs;
  A.S = a->plan_dev == nullptr && a->cu_seqlens_dev == nullptr && a->n_seqs ? (int)(a->rows / a->n_seqs) : 0;
  A.Hq = a->heads;
  A.Hk = a->kv_heads;
  A.group = a->heads / a->kv_heads;
  A.D = a->head_dim;
  A.scale = a->scale;
  return A;
}

// Which tile height a launch over `heads` heads takes, and its number of workgroups (0: too many).
// By the number of workgroups that 128 rows each would make.  With few of them the longest walk decides and shorter
// walks win; with many the traffic to LDS does, and wide heads, whose smaller workgroups run one wave a SIMD, turn
// earlier.  Measured (us, 128 / 64 / 32 rows): bf16, heads of 64, forward of 1 x 512 positions, 12 heads (48
// workgroups) 11.7 / 10.3 / 8.4, 2 x 1024 (192) 18.8 / 17.3 / 17.8, 4 x 1024 (384) 21.1 / 18.5 / 27.8, 6 x 1024 (576)
// 23.3 / 24.6 / 41.4; heads of 128, 8 heads, 1 x 2048 (128) 50.0 / 48.0 / 42.1, 32 heads, 1 x 1024 (256)
// 29.3 / 33.8 / 52.1; dk and dv of 8 x 256, 16 heads (256) 17.2 / 23.2 / 40.9, 2 x 1024, 12 heads (192) 40.8 / 37.8 / 50.2;
// fp32, heads of 64, forward of 6 x 1024 (576) 125 / 107 / 121.  dk and dv of wide fp32 heads need more registers than there
// are with 128 rows (2 x 2048, 8 key/value heads: 2653 / 1201 / 2510) and have no such variant.
// 16-bit sequences of up to 64 rows on average take workgroups of 128 rows however many there are, unless they take 32
// (forward and backward of sequences of 64 / 32 / 8 positions, 4096 in all, 8 heads of 128, 128 against 64 rows:
// 59 and 65, 71 and 94, 211 and 299 us; 12 heads of 64: the same).
static bool attn_brief(const bgx_attention_shape* a) {
  return a->dtype != BGX_F32 && a->rows <= AT_SHORT * (int64_t)a->n_seqs;
}

// What the kernels of a call are: AT_LONG where the host can tell that no sequence is short, AT_BRIEF for that and a second one
// (in workgroups of 128 rows), AT_MIXED for one that has both.
static AttnKind attn_kind(const bgx_attention_shape* a) {
  const bool one_width = a->plan_dev == nullptr && a->cu_seqlens_dev == nullptr && a->lengths_dev == nullptr;
  if (one_width && !attn_brief(a)) return AT_LONG;
  return a->head_dim > 64 && !attn_brief(a) ? AT_BRIEF : AT_MIXED;
}

// The launch for short sequences: in the batch layout the first tile of every sequence, else the list of all tiles.
static AttnArgs attn_brief_args(const AttnArgs& A, unsigned grid, unsigned* few) {
  AttnArgs B = A;
  *few = grid;
  if (A.table == nullptr && A.bounds == nullptr) {
    *few = grid / (unsigned)A.tiles;
    B.tiles = 1;
  }
  return B;
}

enum AttnKernel { ATTN_FORWARD, ATTN_Q, ATTN_KV };
static unsigned attn_grid(AttnArgs& A, const bgx_attention_shape* a, AttnKernel kernel, int* which) {
  const int heads = kernel == ATTN_KV && A.part_k == nullptr ? a->kv_heads : a->heads;
  const int64_t tall = attn_items(a, 0) * heads;
  const bool wide = a->head_dim > 64, full = a->dtype == BGX_F32;
  const int64_t many = full ? (!wide ? 1024 : kernel == ATTN_KV ? INT64_MAX : 512)
                            : (!wide ? 512 : kernel == ATTN_FORWARD ? 160 : 256);
  *which = tall >= many ? 0 : tall >= 160 ? 1 : 2;
  if (*which == 1 && attn_brief(a)) *which = 0;
  for (int i = 0; i < 3; ++i)
    if (switches().attention_rows == AT_TILES[i]) *which = i;
  if (kernel == ATTN_KV && wide && full && *which == 0) *which = 1;
  const int64_t grid = attn_items(a, *which) * heads;
  if (a->plan_dev != nullptr) {
    A.table = (const int4*)a->plan_dev;
    for (int i = 0; i < *which; ++i) A.table += plan_entries(a->rows, a->n_seqs, i);
  }
  A.tiles = (A.S + AT_TILES[*which] - 1) / AT_TILES[*which];
  return grid < (1ll << 31) ? (unsigned)grid : 0;
}

// offsets within a tile are 32-bit
static int attn_check_rows(const bgx_attention_rows* t, int head_dim, int dtype, const char* what) {
  BGX_REQUIRE(t != nullptr && t->data != nullptr, BGX_E_ARG, "%s: null operand", what);
  BGX_REQUIRE(t->tok_stride >= head_dim && t->tok_stride * (int64_t)dtype_size(dtype) <= (1 << 23), BGX_E_SHAPE,
              "%s: %lld elements between positions, supported are head_dim=%d up to 8 MiB", what,
              (long long)t->tok_stride, head_dim);
  return 0;
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

// the tallest variant of each kernel and its threads
template <typename T, int DP>
constexpr int attention_forward_kernel_tall() {
  return 4;
}
template <typename T, int DP>
constexpr int attention_forward_kernel_threads() {
  return AT_THREADS;
}
template <typename T, int DP>
constexpr int attention_backward_q_kernel_tall() {
  return 4;
}
template <typename T, int DP>
constexpr int attention_backward_q_kernel_threads() {
  return AT_THREADS;
}
template <typename T, int DP>
constexpr int attention_backward_kv_kernel_tall() {
  return sizeof(T) == 4 && DP > 64 ? 2 : 4;
}
template <typename T, int DP>
constexpr int attention_backward_kv_kernel_threads() {
  return kv_waves<T, DP, attention_backward_kv_kernel_tall<T, DP>()>() * WAVE;
}

#define BGX_ATTN_ROWS(KERNEL, T, DP, WHICH, GRID, S, A)                    \
  do {                                                                     \
    constexpr int tall = KERNEL##_tall<T, DP>(), threads = KERNEL##_threads<T, DP>(); \
    constexpr bool full = sizeof(T) == 4; /* nothing to decide */          \
    if ((WHICH) == 0 && kind == AT_MIXED)                                  \
      KERNEL<T, DP, tall, full ? AT_ALL : AT_MIXED><<<(GRID), threads, 0, (S)>>>(A); \
    else if ((WHICH) == 0)                                                 \
      KERNEL<T, DP, tall, full ? AT_ALL : AT_LONG><<<(GRID), threads, 0, (S)>>>(A); \
    else if ((WHICH) == 1 && kind != AT_LONG)                              \
      KERNEL<T, DP, 2, full ? AT_ALL : AT_MIXED><<<(GRID), AT_THREADS, 0, (S)>>>(A); \
    else if ((WHICH) == 1)                                                 \
      KERNEL<T, DP, 2, full ? AT_ALL : AT_LONG><<<(GRID), AT_THREADS, 0, (S)>>>(A); \
    else                                                                   \
      KERNEL<T, DP, 1, AT_ALL><<<(GRID), AT_THREADS, 0, (S)>>>(A);         \
    if constexpr (!full && DP > 64)                                        \
      if ((WHICH) == 0 && kind == AT_BRIEF) {                              \
        unsigned few;                                                      \
        const AttnArgs brief = attn_brief_args((A), (GRID), &few);         \
        KERNEL<T, DP, tall, AT_BRIEF><<<few, threads, 0, (S)>>>(brief);    \
      }                                                                    \
  } while (0)
#define BGX_ATTN_WIDTHS(KERNEL, T, D, WHICH, GRID, S, A)      \
  do {                                                        \
    if ((D) <= 32)                                            \
      BGX_ATTN_ROWS(KERNEL, T, 32, WHICH, GRID, S, A);        \
    else if ((D) <= 64)                                       \
      BGX_ATTN_ROWS(KERNEL, T, 64, WHICH, GRID, S, A);        \
    else if ((D) <= 96)                                       \
      BGX_ATTN_ROWS(KERNEL, T, 96, WHICH, GRID, S, A);        \
    else                                                      \
      BGX_ATTN_ROWS(KERNEL, T, 128, WHICH, GRID, S, A);       \
  } while (0)
#define BGX_ATTN_LAUNCH(KERNEL, DTYPE, D, WHICH, GRID, S, A)  \
  do {                                                        \
    if ((DTYPE) == BGX_F32)                                   \
      BGX_ATTN_WIDTHS(KERNEL, float, D, WHICH, GRID, S, A);   \
    else if ((DTYPE) == BGX_F16)                              \
      BGX_ATTN_WIDTHS(KERNEL, f16_t, D, WHICH, GRID, S, A);   \
    else                                                      \
      BGX_ATTN_WIDTHS(KERNEL, bf16_t, D, WHICH, GRID, S, A);  \
    BGX_HIP(hipGetLastError());                               \
  } while (0)

size_t attention_plan_bytes(int64_t rows, int n_seqs) {
  if (rows < 0 || n_seqs < 0) return 0;
  size_t entries = 0;
  for (int i = 0; i < 3; ++i) entries += plan_entries(rows, n_seqs, i);
  return entries * sizeof(int4);
}

int attention_plan_impl(const int32_t* cu, int n_seqs, int64_t rows, void* plan, size_t plan_bytes, void* stream) {
  BGX_REQUIRE(n_seqs >= 0 && rows >= 0 && rows < (1ll << 31) - 4 * AT_TILES[0], BGX_E_ARG, "attention plan: n_seqs=%d rows=%lld",
              n_seqs, (long long)rows);
  BGX_REQUIRE(cu != nullptr || n_seqs == 0, BGX_E_ARG, "attention plan: null cu_seqlens");
  int64_t n[3], all = 0;
  for (int i = 0; i < 3; ++i) all += n[i] = plan_entries(rows, n_seqs, i);
  BGX_REQUIRE(all < (1ll << 31), BGX_E_SHAPE, "attention plan: %lld entries", (long long)all);
  BGX_REQUIRE(plan != nullptr && plan_bytes >= attention_plan_bytes(rows, n_seqs), BGX_E_WORKSPACE,
              "attention plan: %zu bytes, %zu needed", plan_bytes, attention_plan_bytes(rows, n_seqs));
  attention_plan_kernel<<<3, PLAN_THREADS, 0, (hipStream_t)stream>>>(cu, n_seqs, (int)rows, (int4*)plan, (int)n[0],
                                                                    (int)n[1], (int)n[2]);
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
  for (const bgx_attention_rows* t : {q, k, v, o})
    if (int rc = attn_check_rows(t, a->head_dim, a->dtype, "attention")) return rc;
  AttnArgs A = attn_args(a);
  A.q = attn_view(q);
  A.k = attn_view(k);
  A.v = attn_view(v);
  A.o = attn_view(o);
  attn_saved(A, a, saved);
  int which;
  const AttnKind kind = attn_kind(a);
  const unsigned grid = attn_grid(A, a, ATTN_FORWARD, &which);
  BGX_REQUIRE(grid > 0, BGX_E_SHAPE, "attention: %lld rows of %d heads", (long long)a->rows, a->heads);
  BGX_ATTN_LAUNCH(attention_forward_kernel, a->dtype, a->head_dim, which, grid, (hipStream_t)stream, A);
  return 0;
}

// Where few key/value heads and rows leave too few workgroups that walk all query heads of a group one after the
// other, every query head gets workgroups of its own and the heads' parts are added by a kernel behind: 8 bytes of
// parts per query element, written and read once.
constexpr int64_t ATTN_PARTS_MAX = 512ll << 20;
static int64_t attn_part_bytes(const bgx_attention_shape* a) {
  if (a->kv_heads < 1 || a->heads <= a->kv_heads || attn_items(a, 0) * a->kv_heads >= 384) return 0;
  const int64_t bytes = a->rows * a->heads * a->head_dim * (int64_t)sizeof(float) * 2;
  return bytes <= ATTN_PARTS_MAX ? bytes : 0;
}

static int64_t attn_stat_bytes(const bgx_attention_shape* a) {
  const int64_t n = a->rows * a->heads * (int64_t)sizeof(float) * (a->dtype == BGX_F16 ? 2 : 1);
  return (n + 15) / 16 * 16;
}

size_t attention_backward_workspace_bytes(const bgx_attention_shape* a) {
  if (a == nullptr || a->rows <= 0 || a->heads <= 0) return 0;
  return (size_t)(attn_stat_bytes(a) + attn_part_bytes(a));
}

int attention_backward_impl(const bgx_attention_shape* a, const bgx_attention_rows* q, const bgx_attention_rows* k,
                            const bgx_attention_rows* v, const bgx_attention_rows* o, const void* saved,
                            const bgx_attention_rows* grad_o, const bgx_attention_rows* dq, const bgx_attention_rows* dk,
                            const bgx_attention_rows* dv, void* ws, size_t ws_bytes, void* stream) {
  if (int rc = attn_check(a, "attention backward")) return rc;
  if (a->rows == 0) return 0;
  for (const bgx_attention_rows* t : {q, k, v, o, grad_o, dq, dk, dv})
    if (int rc = attn_check_rows(t, a->head_dim, a->dtype, "attention backward")) return rc;
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
  BGX_REQUIRE((uintptr_t)ws % 16 == 0, BGX_E_ALIGN, "attention backward: workspace not aligned to 16 bytes");
  hipStream_t s = (hipStream_t)stream;
  int which;
  const AttnKind kind = attn_kind(a);
  unsigned grid = attn_grid(A, a, ATTN_Q, &which);
  BGX_REQUIRE(grid > 0, BGX_E_SHAPE, "attention backward: %lld rows of %d heads", (long long)a->rows, a->heads);
  BGX_ATTN_LAUNCH(attention_backward_q_kernel, a->dtype, a->head_dim, which, grid, s, A);
  const int64_t parts = attn_part_bytes(a);
  if (parts > 0) {
    A.part_k = (float*)((char*)ws + attn_stat_bytes(a));
    A.part_v = A.part_k + parts / 2 / (int64_t)sizeof(float);
  }
  grid = attn_grid(A, a, ATTN_KV, &which);
  BGX_REQUIRE(grid > 0, BGX_E_SHAPE, "attention backward: %lld rows of %d heads", (long long)a->rows, a->heads);
  BGX_ATTN_LAUNCH(attention_backward_kv_kernel, a->dtype, a->head_dim, which, grid, s, A);
  if (parts > 0) {
    const dim3 join((unsigned)((a->rows * a->kv_heads * (a->head_dim / 4) + 255) / 256), 2);
    if (a->dtype == BGX_F32)
      attention_backward_join_kernel<float><<<join, 256, 0, s>>>(A);
    else if (a->dtype == BGX_F16)
      attention_backward_join_kernel<f16_t><<<join, 256, 0, s>>>(A);
    else
      attention_backward_join_kernel<bf16_t><<<join, 256, 0, s>>>(A);
    BGX_HIP(hipGetLastError());
  }
  return 0;
}

}  // namespace bgx
