// expert_products.hip -- matrix products on rows sorted by expert (ragged
// groups), 16-bit operands with their gradients and int8 operands with a scale
// for each row and output channel, on the matrix cores of gfx950.
//
//   y[r] = W[e] x[r]      dx[r] = W[e]^T dy[r]      dW[e] = sum_r dy[r] x[r]^T
#pragma clang fp contract(off)
#include <type_traits>

#include "expert_products.hpp"
#include "mi_moe_device.hpp"

namespace mimoe {

namespace {

constexpr int kThreads = 512, kWaves = 8;
constexpr int kTile = 256;          // output columns of a tile, and most rows
// A step of the products' index: a cache line of a row, or 64 rows across it.
// (Loads of 64 bytes of a row make twice the requests to the L2, and those
// bound the loop: bf16 8192 x 8192 x 4096 444 us, 402 with whole lines.)
constexpr int kStepBytes = 128;
constexpr int kStepRows = 64;
constexpr int kLds = 163840;        // all of a compute unit's
constexpr uint32_t kOutside = 0x80000000u;     // an offset beyond any buffer: loads give zero

typedef __attribute__((address_space(3))) unsigned char lds_byte;
typedef short s16x4_t __attribute__((ext_vector_type(4)));

// Operand types.  A 16-byte register of each holds what one matrix
// instruction takes of a lane: 8 values of 16 bits or 16 of 8, at the same
// place of the row, so all three share the LDS layout.
struct F16 { typedef f32x4_t acc; };
struct BF16 { typedef f32x4_t acc; };
struct I8 { typedef i32x4_t acc; };
__device__ __forceinline__ void mma(F16, const u32x4_t& a, const u32x4_t& b, f32x4_t& c) {
  c = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
}
__device__ __forceinline__ void mma(BF16, const u32x4_t& a, const u32x4_t& b, f32x4_t& c) {
  c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}
__device__ __forceinline__ void mma(I8, const u32x4_t& a, const u32x4_t& b, i32x4_t& c) {
  c = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4_t, a), __builtin_bit_cast(i32x4_t, b), c, 0, 0, 0);
}

__device__ __forceinline__ uint32_t uni(uint32_t v) { return __builtin_amdgcn_readfirstlane(v); }

// 64 lanes * 16 B from a buffer (zeros past its end) to LDS at `lds` on.  The
// load has no register to write, so nothing but the counter tells that it is
// done: wait_loads_meet.
__device__ __forceinline__ void load_to_lds(__amdgpu_buffer_rsrc_t buf, uint32_t off, uint32_t lds) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(buf, (__attribute__((address_space(3))) void*)(uintptr_t)lds, 16, (int)off, 0, 0, 0);
}
// All but the last N loads to LDS of this wave are done, and all its LDS
// reads; then all waves meet.
template <int N>
__device__ __forceinline__ void wait_loads_meet() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}
__device__ __forceinline__ void meet() { asm volatile("s_barrier" ::: "memory"); }

// Every load and store of a tile goes through a buffer: what lies past its
// end, or at kOutside, reads as zero and is not written.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer_of(const void* p, int64_t bytes) {
  const uint32_t n = bytes < 0 ? 0u : bytes > 0x7fffffff ? 0x7fffffffu : (uint32_t)bytes;
  return __builtin_amdgcn_make_buffer_rsrc((void*)p, (short)0, (int)uni(n), 0x00020000);
}

// One operand's share of a tile.  COLS false: DIM rows with the products'
// index along the row ([row][128 B] in LDS, the 16-byte pieces of a row
// permuted by the row, so that rows read at one place lie in different
// banks).  COLS true: the products' index across rows of 16-bit values ([64
// rows][2 DIM B], the 32-byte chunks of a row permuted by the row, so that
// the 8 rows of half a transposed read do).  NSUB: subtiles of a wave.
template <bool COLS, int DIM, int NSUB>
struct Operand {
  static constexpr int kIssues = (DIM + 63) / 64;   // loads of a wave a step
  static constexpr int kBytes = kIssues * 8192;
  static constexpr int kReads = COLS ? NSUB : 2;    // LDS addresses of a wave
  // loads: the next step's
  const unsigned char* base;
  uint32_t size;       // bytes of it that belong to the tile
  uint32_t off[kIssues];
  int left;            // steps (COLS: rows) from there to the end
  uint32_t ld;
  int ragged;          // the last step's 16-byte pieces (0: all eight); !COLS
  // reads
  uint32_t at[kReads];

  // b: the tile's first element; n: its rows (COLS: columns); len: length of
  // the products' index in bytes of a row (COLS: in rows); sub: the wave's
  // first subtile; lds: where the ring begins for this operand.
  __device__ __forceinline__ void set(const unsigned char* b, int n, uint32_t ld_, int len, int sub, uint32_t lds) {
    base = b;
    ld = ld_;
    const int t = threadIdx.x, lane = t & 63, q = lane >> 4, r = lane & 15;
    if constexpr (COLS) {
      static_assert(DIM == 256 || DIM == 128, "a row of 32 or 16 pieces");
      constexpr int kPieces = DIM / 8, kRows = kThreads / kPieces;   // of a row; rows of an issue
      const int k = t / kPieces, piece = t % kPieces;
#pragma unroll
      for (int i = 0; i < kIssues; ++i) {
        const int row = k + kRows * i, c = piece ^ (swizzle(row) << 1);
        off[i] = 8 * c < n ? (uint32_t)row * ld + 16u * c : kOutside;
      }
      left = len;
      const int kr = 8 * q + (r >> 2);
#pragma unroll
      for (int i = 0; i < NSUB; ++i) at[i] = lds + kr * (2 * DIM) + (((sub + i) ^ swizzle(kr)) << 5) + ((r & 3) << 3);
    } else {
#pragma unroll
      for (int i = 0; i < kIssues; ++i) {
        const int row = 64 * i + (t >> 3);
        off[i] = row < min(n, DIM) ? (uint32_t)row * ld + 16u * piece_of(t) : kOutside;
      }
      left = (len + kStepBytes - 1) / kStepBytes;
      ragged = (len % kStepBytes) >> 4;
#pragma unroll
      for (int h = 0; h < 2; ++h) at[h] = lds + (16 * sub + r) * kStepBytes + (((4 * h + q) ^ (r & 7)) << 4);
    }
    limit();
  }
  static __device__ __forceinline__ int swizzle(int k) { return (k & 3) | ((k >> 1) & 4); }
  static __device__ __forceinline__ int piece_of(int t) { return (t & 7) ^ ((t >> 3) & 7); }

  // What the next step's loads may read: nothing past the last step.
  __device__ __forceinline__ void limit() {
    if constexpr (COLS) {
      size = (uint32_t)max(0, min(left, kStepRows)) * ld;
    } else {
      size = left > 0 ? 0x7fffffffu : 0u;
      if (left == 1 && ragged) {   // uniform, once
#pragma unroll
        for (int i = 0; i < kIssues; ++i) off[i] = piece_of(threadIdx.x) < ragged ? off[i] : kOutside;
      }
    }
  }
  __device__ __forceinline__ void advance() {
    base += COLS ? (uint64_t)kStepRows * ld : (uint64_t)kStepBytes;
    left -= COLS ? kStepRows : 1;
    limit();
  }
  // Loads of a step to LDS at `dst`, this wave's first kilobyte of it.
  __device__ __forceinline__ void load(uint32_t dst) const {
    const __amdgpu_buffer_rsrc_t buf = __builtin_amdgcn_make_buffer_rsrc((void*)base, (short)0, (int)size, 0x00020000);
#pragma unroll
    for (int i = 0; i < kIssues; ++i) load_to_lds(buf, off[i], dst + i * 8192);
  }
  // What the matrix instruction takes of the wave's subtile i (16 rows, or
  // columns), half h of the step.
  __device__ __forceinline__ u32x4_t get(int i, int h) const {
    if constexpr (COLS) {
      const uint32_t p = at[i] + h * 32 * (2 * DIM);
      const s16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4_t*)(uintptr_t)p);
      const s16x4_t hi =
          __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4_t*)(uintptr_t)(p + 4 * (2 * DIM)));
      const u32x2_t a = __builtin_bit_cast(u32x2_t, lo), b = __builtin_bit_cast(u32x2_t, hi);
      return u32x4_t{a.x, a.y, b.x, b.y};
    } else {
      return *(const __attribute__((address_space(3))) u32x4_t*)(uintptr_t)(at[h] + i * 16 * kStepBytes);
    }
  }
  __device__ __forceinline__ void move(uint32_t d) {
#pragma unroll
    for (int i = 0; i < kReads; ++i) at[i] += d;
  }
};

// acc[i][u * NU + j] += the wave's subtile i of P times its subtile j of half
// u of Q, over all steps.
//
// The steps pass through a ring of RING LDS buffers.  The two waves of a SIMD
// take turns: while one reads its operands from LDS and starts loads, the
// other runs its matrix instructions (`late` waves are one turn behind).
//   turn 4 s      early: read P, Q0 of step s     late: products with Q1, step s - 1
//   turn 4 s + 1  early: products with Q0         late: read P, Q0 of step s
//   turn 4 s + 2  early: read Q1                  late: products with Q0
//   turn 4 s + 3  early: products with Q1         late: read Q1
// What has been read is in registers, so P and Q0 of step s + RING are loaded
// into the places of step s from turn 4 s + 2 on, with the reads of Q1, and Q1
// of step s + RING from turn 4 s + 4 on, with the next reads of P and Q0.
// Every wave ends its reads by waiting until all but its last (RING - 1) steps'
// worth of loads are done: what is read two turns later is then in LDS.
// Addresses are moved on among the matrix instructions, whose issue leaves room.
template <class OP, class OQ>
struct Ring {
  static constexpr int kStage = OP::kBytes + 2 * OQ::kBytes, kLoads = OP::kIssues + 2 * OQ::kIssues;
  static constexpr int kSize = kLds / kStage;
  static_assert(kSize >= 2, "a step ahead");
};
template <class T, class OP, class OQ, int NP, int NQ>
__device__ __forceinline__ void products(OP& P, OQ& Q0, OQ& Q1, uint32_t lds, int steps, bool late, typename T::acc (&acc)[NP][NQ]) {
  constexpr int NU = NQ / 2, STAGE = Ring<OP, OQ>::kStage, RING = Ring<OP, OQ>::kSize, AHEAD = (RING - 1) * Ring<OP, OQ>::kLoads;
  const uint32_t mine = lds + uni(threadIdx.x >> 6) * 1024;
#pragma unroll
  for (int i = 0; i < NP; ++i)
#pragma unroll
    for (int j = 0; j < NQ; ++j) acc[i][j] = typename T::acc{0, 0, 0, 0};
#pragma unroll
  for (int s = 0; s < RING; ++s) {
    P.load(mine + s * STAGE);
    Q0.load(mine + s * STAGE + OP::kBytes);
    P.advance();
    Q0.advance();
    if (s < RING - 1) {
      Q1.load(mine + s * STAGE + OP::kBytes + OQ::kBytes);
      Q1.advance();
    }
  }
  wait_loads_meet<AHEAD>();
  if (late) meet();
  uint32_t cur = 0, prev = (RING - 1) * STAGE;
  u32x4_t p[NP][2], q[NU][2];
  auto turn = [&](int u) {
    __builtin_amdgcn_sched_barrier(0);
    wait_loads_meet<AHEAD>();
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < NP; ++i)
#pragma unroll
        for (int j = 0; j < NU; ++j) mma(T{}, p[i][h], q[j][h], acc[i][u * NU + j]);
  };
  auto over = [&] {
    __builtin_amdgcn_s_setprio(0);
    __builtin_amdgcn_sched_barrier(0);
    meet();
    __builtin_amdgcn_sched_barrier(0);
  };
  for (int s = 0; s < steps; ++s) {
    const uint32_t d = cur == (RING - 1) * STAGE ? (uint32_t)-(RING - 1) * STAGE : (uint32_t)STAGE;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int i = 0; i < NP; ++i) p[i][h] = P.get(i, h);
#pragma unroll
      for (int j = 0; j < NU; ++j) q[j][h] = Q0.get(j, h);
    }
    Q1.load(mine + prev + OP::kBytes + OQ::kBytes);
    turn(0);
    Q1.advance();
    P.move(d);
    Q0.move(d);
    over();
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int j = 0; j < NU; ++j) q[j][h] = Q1.get(j, h);
    P.load(mine + cur);
    Q0.load(mine + cur + OP::kBytes);
    turn(1);
    P.advance();
    Q0.advance();
    Q1.move(d);
    prev = cur;
    cur += d;
    over();
  }
  if (!late) meet();
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // no load to LDS outlives the workgroup
}

// ------------------------------------------------------------ work items
// Groups of rows: 0 the rows before the first expert's, 1 .. E the experts,
// E + 1 the rows behind the last's.  starts is read as its running maximum
// within [0, M], so that no value of it leads outside the tensors.
struct Item {
  int e, row0, rows;   // e < 0: rows of no expert
};

// Item `index` of all groups' items of at most `most` rows; a group's rows
// are split evenly, in multiples of `grain`.  False: past the last item;
// `total` is their number.
__device__ __forceinline__ int items_of(int rows, int most) { return (rows + most - 1) / most; }

struct Groups {
  static constexpr int kPer = (kGroupMaxE + 2 + kWave - 1) / kWave;
  int begin[kPer + 1];   // first rows of this lane's groups, and of the next lane's first
  int before;            // items of the lanes before this one
  int total;

  __device__ __forceinline__ void read(const int32_t* starts, int E, int M, int most) {
    const int lane = threadIdx.x & 63;
    int v[kPer];   // where group g ends
    int m = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int g = lane * kPer + i;
      int s = starts[g <= E ? g : E];
      s = g <= E ? s : M;
      s = s < 0 ? 0 : s > M ? M : s;
      m = m > s ? m : s;
      v[i] = m;
    }
#pragma unroll
    for (int d = 1; d < kWave; d <<= 1) {
      const int o = __shfl_up(m, d);
      if (lane >= d) m = m > o ? m : o;
    }
    int first = __shfl_up(m, 1);
    if (lane == 0) first = 0;
    int n = 0;
    begin[0] = first;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      begin[i + 1] = v[i] > first ? v[i] : first;
      n += items_of(begin[i + 1] - begin[i], most);
    }
    int sum = n;
#pragma unroll
    for (int d = 1; d < kWave; d <<= 1) {
      const int o = __shfl_up(sum, d);
      if (lane >= d) sum += o;
    }
    before = sum - n;
    total = __builtin_amdgcn_readlane(sum, 63);
  }
  __device__ __forceinline__ Item find(int index, int E, int most, int grain) const {
    const int src = 63 - __builtin_clzll(__ballot(before <= index));   // the last lane whose items begin at or before it
    int at = before, g = 0, k = 0, n = 1, b = 0, e = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int c = items_of(begin[i + 1] - begin[i], most);
      if (index >= at && index < at + c) {
        g = (threadIdx.x & 63) * kPer + i;
        k = index - at;
        n = c;
        b = begin[i];
        e = begin[i + 1];
      }
      at += c;
    }
    g = __builtin_amdgcn_readlane(g, src);
    k = __builtin_amdgcn_readlane(k, src);
    n = __builtin_amdgcn_readlane(n, src);
    b = __builtin_amdgcn_readlane(b, src);
    e = __builtin_amdgcn_readlane(e, src);
    const int size = ((e - b + n - 1) / n + grain - 1) / grain * grain;
    const int row0 = b + k * size;
    return Item{g == 0 || g > E ? -1 : g - 1, row0, max(0, min(size, e - row0))};
  }
};

// Items of one launch: each group adds less than one whole item.
__host__ inline int64_t items_max(int64_t M, int64_t E, int most) { return M / most + (M < E + 2 ? M : E + 2); }

// Place of workgroup b among `items` items and `blocks` blocks of columns.
// The list goes through 8 blocks of columns for every item; the XCDs take
// kRun places of it in turn, so that the workgroups that share an L2 at a time
// share rows and weights, and experts of unequal sizes spread over all XCDs.
constexpr int kRun = 8;
__device__ __forceinline__ bool place(int b, int items, int blocks, int& item, int& block) {
  const int j = b >> 3;
  int l = ((j / kRun) * 8 + (b & 7)) * kRun + j % kRun;
  if (l >= items * blocks) return false;
  const int full = items * (blocks & ~7);
  int w = 8, b0 = 0;
  if (l < full) {
    b0 = l / (items * 8) * 8;
    l -= b0 * items;
  } else {
    w = blocks & 7;
    b0 = blocks & ~7;
    l -= full;
  }
  item = l / w;
  block = b0 + l - item * w;
  return true;
}

// ------------------------------------------------------------ stores
template <int OUT>
constexpr int kOutBytes = OUT == 2 ? 4 : 2;

// Four values of a row at byte `off`, `n` of them within it.  vec: rows are
// whole pieces of four.
template <int OUT>
__device__ __forceinline__ void store4(__amdgpu_buffer_rsrc_t y, uint32_t off, const float (&v)[4], int n, bool vec) {
  if constexpr (OUT == 2) {
    if (vec) {   // uniform
      const u32x4_t w = {__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])};
      __builtin_amdgcn_raw_buffer_store_b128(w, y, (int)(n > 0 ? off : kOutside), 0, 0);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(v[i]), y, (int)(i < n ? off + 4 * i : kOutside), 0, 0);
    }
  } else {
    const uint16_t h[4] = {from_f32<OUT>(v[0]), from_f32<OUT>(v[1]), from_f32<OUT>(v[2]), from_f32<OUT>(v[3])};
    if (vec) {
      const u32x2_t w = {h[0] | (uint32_t)h[1] << 16, h[2] | (uint32_t)h[3] << 16};
      __builtin_amdgcn_raw_buffer_store_b64(w, y, (int)(n > 0 ? off : kOutside), 0, 0);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) __builtin_amdgcn_raw_buffer_store_b16(h[i], y, (int)(i < n ? off + 2 * i : kOutside), 0, 0);
    }
  }
}
template <int OUT>
__device__ __forceinline__ __amdgpu_buffer_rsrc_t out_buffer(void* y, int64_t at) {
  return buffer_of((unsigned char*)y + at * kOutBytes<OUT>, 0x7fffffff);
}
template <int OUT>
__device__ __forceinline__ bool out_vec(const void* y, int64_t ldy) { return (ldy & 3) == 0 && ((uintptr_t)y & 15) == 0; }

// `rows` rows of n <= 256 columns become zero.
template <int OUT>
__device__ __forceinline__ void zero_rows(__amdgpu_buffer_rsrc_t y, uint32_t ld, int rows, int n, bool vec) {
  for (int i = threadIdx.x; i < rows * 64; i += kThreads) {
    const int c = 4 * (i & 63);
    const float z[4] = {0, 0, 0, 0};
    store4<OUT>(y, (uint32_t)(i >> 6) * ld + c * kOutBytes<OUT>, z, n - c, vec);
  }
}

template <class T, bool WCOLS, int OUT, int NQ>
__device__ __forceinline__ void row_item(const RowProductArgs& a, unsigned char* smem, const Item& it, int p0) {
  constexpr int kElem = std::is_same<T, I8>::value ? 1 : 2;
  const int wave = uni(threadIdx.x >> 6), wp = wave & 3, wq = wave >> 2, lane = threadIdx.x & 63;
  const int np = min(kTile, a.P - p0);
  typedef Operand<WCOLS, kTile, 4> OpW;
  typedef Operand<false, 16 * NQ, NQ / 2> OpX;   // half of the rows
  OpW W;
  OpX X0, X1;
  const unsigned char *w = a.w + (int64_t)it.e * a.w_expert, *x = a.x + (int64_t)it.row0 * a.ldx;
  const int len = a.K * kElem;
  const uint32_t lds = (uint32_t)(uintptr_t)(lds_byte*)smem;
  W.set(w + (int64_t)p0 * (WCOLS ? kElem : a.ldw), np, a.ldw, WCOLS ? a.K : len, 4 * wp, lds);
  X0.set(x, it.rows, a.ldx, len, NQ / 2 * wq, lds + OpW::kBytes);
  X1.set(x + (int64_t)(16 * NQ) * a.ldx, it.rows - 16 * NQ, a.ldx, len, NQ / 2 * wq, lds + OpW::kBytes + OpX::kBytes);
  typename T::acc acc[4][NQ];
  products<T>(W, X0, X1, lds, (len + kStepBytes - 1) / kStepBytes, wq != 0, acc);
  const __amdgpu_buffer_rsrc_t y = out_buffer<OUT>(a.y, (int64_t)it.row0 * a.ldy + p0);
  const bool vec = out_vec<OUT>(a.y, a.ldy);
  const int r = lane & 15, c0 = 64 * wp + 4 * (lane >> 4);
  float ws[4][4], bias[4][4];
  if constexpr (kElem == 1) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int p = min(p0 + c0 + 16 * i + k, a.P - 1);
        ws[i][k] = a.ws[(int64_t)it.e * a.P + p];
        bias[i][k] = a.bias ? a.bias[p] : 0.0f;
      }
  }
#pragma unroll
  for (int j = 0; j < NQ; ++j) {
    const int row = 16 * (j / (NQ / 2) * NQ + NQ / 2 * wq + j % (NQ / 2)) + r;
    const bool in = row < it.rows;
    const uint32_t off = (uint32_t)row * (uint32_t)(a.ldy * kOutBytes<OUT>);
    float xs = 1.0f;
    if constexpr (kElem == 1) xs = a.xs[it.row0 + (in ? row : 0)];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int c = c0 + 16 * i;
      float v[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        v[k] = (float)acc[i][j][k];
        if constexpr (kElem == 1) v[k] = v[k] * ws[i][k] * xs + bias[i][k];
      }
      store4<OUT>(y, off + c * kOutBytes<OUT>, v, in ? np - c : 0, vec);
    }
  }
}

template <class T, bool WCOLS, int OUT>
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(2))) void row_product_kernel(RowProductArgs a) {
  __shared__ __align__(16) unsigned char smem[kLds];
  const int blocks = (a.P + kTile - 1) / kTile;
  int item, block;
  Item it;
  if (a.starts) {
    Groups g;
    g.read(a.starts, a.E, a.M, kTile);
    if (!place(blockIdx.x, g.total, blocks, item, block)) return;
    it = g.find(item, a.E, kTile, 32);
  } else {
    if (!place(blockIdx.x, items_of(a.M, kTile), blocks, item, block)) return;
    it = Item{0, item * kTile, min(kTile, a.M - item * kTile)};
  }
  const int p0 = block * kTile;
  if (it.rows <= 0) return;
  if (it.e < 0) {
    zero_rows<OUT>(out_buffer<OUT>(a.y, (int64_t)it.row0 * a.ldy + p0), (uint32_t)(a.ldy * kOutBytes<OUT>), it.rows,
                   min(kTile, a.P - p0), out_vec<OUT>(a.y, a.ldy));
    return;
  }
  if (it.rows <= 64) row_item<T, WCOLS, OUT, 2>(a, smem, it, p0);
  else if (it.rows <= 128) row_item<T, WCOLS, OUT, 4>(a, smem, it, p0);
  else if (it.rows <= 192) row_item<T, WCOLS, OUT, 6>(a, smem, it, p0);
  else row_item<T, WCOLS, OUT, 8>(a, smem, it, p0);
}

template <class T, int OUT>
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(2))) void weight_grad_kernel(WeightGradArgs a) {
  __shared__ __align__(16) unsigned char smem[kLds];
  const int bk = (a.K + kTile - 1) / kTile, bn = (a.N + kTile - 1) / kTile;
  int item, block;
  if (!place(blockIdx.x, a.E * bn, bk, item, block)) return;
  const int e = item / bn, n0 = (item - e * bn) * kTile, k0 = block * kTile;
  // the expert's rows: starts as its running maximum within [0, M]
  int b = 0;
  for (int i = threadIdx.x & 63; i <= e; i += 64) b = max(b, a.starts[i]);
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) b = max(b, __shfl_xor(b, d));
  b = uni(min(b, a.M));
  const int end = uni(max(b, min(a.starts[e + 1], a.M))), rows = end - b;
  const int wave = uni(threadIdx.x >> 6), wp = wave & 3, wq = wave >> 2, lane = threadIdx.x & 63;
  typedef Operand<true, kTile, 4> OpX;
  typedef Operand<true, kTile / 2, 4> OpY;   // half of the columns
  OpX X;
  OpY Y0, Y1;
  const uint32_t lds = (uint32_t)(uintptr_t)(lds_byte*)smem;
  const unsigned char *x = a.x + (int64_t)b * a.ldx + (int64_t)k0 * 2, *dy = a.dy + (int64_t)b * a.lddy + (int64_t)n0 * 2;
  X.set(x, min(kTile, a.K - k0), a.ldx, rows, 4 * wp, lds);
  Y0.set(dy, min(kTile, a.N - n0), a.lddy, rows, 4 * wq, lds + OpX::kBytes);
  Y1.set(dy + kTile, a.N - n0 - kTile / 2, a.lddy, rows, 4 * wq, lds + OpX::kBytes + OpY::kBytes);
  f32x4_t acc[4][8];
  products<T>(X, Y0, Y1, lds, (rows + kStepRows - 1) / kStepRows, wq != 0, acc);
  const __amdgpu_buffer_rsrc_t dw = out_buffer<OUT>(a.dw, ((int64_t)e * a.N + n0) * a.K + k0);
  const bool vec = out_vec<OUT>(a.dw, a.K);
  const int r = lane & 15, c0 = 64 * wp + 4 * (lane >> 4);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int row = 16 * (j / 4 * 8 + 4 * wq + j % 4) + r;
    const uint32_t off = (uint32_t)row * (uint32_t)(a.K * kOutBytes<OUT>);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int c = c0 + 16 * i;
      const float v[4] = {acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3]};
      store4<OUT>(dw, off + c * kOutBytes<OUT>, v, row < a.N - n0 ? a.K - k0 - c : 0, vec);
    }
  }
}

unsigned grid_of(int64_t tiles) { return (unsigned)((tiles + 8 * kRun - 1) / (8 * kRun) * (8 * kRun)); }

}  // namespace

hipError_t launch_row_product(const RowProductArgs& a, int dt, int w_cols, int out, hipStream_t st) {
  const int64_t items = a.starts ? items_max(a.M, a.E, kTile) : (a.M + kTile - 1) / kTile;
  const int64_t blocks = (a.P + kTile - 1) / kTile;
  const unsigned grid = grid_of(items * blocks);
  if (dt == 2) {
    if (out == 0) row_product_kernel<I8, false, 0><<<grid, kThreads, 0, st>>>(a);
    else if (out == 1) row_product_kernel<I8, false, 1><<<grid, kThreads, 0, st>>>(a);
    else row_product_kernel<I8, false, 2><<<grid, kThreads, 0, st>>>(a);
  } else if (dt == 1) {
    if (w_cols) row_product_kernel<BF16, true, 1><<<grid, kThreads, 0, st>>>(a);
    else row_product_kernel<BF16, false, 1><<<grid, kThreads, 0, st>>>(a);
  } else {
    if (w_cols) row_product_kernel<F16, true, 0><<<grid, kThreads, 0, st>>>(a);
    else row_product_kernel<F16, false, 0><<<grid, kThreads, 0, st>>>(a);
  }
  return hipGetLastError();
}

hipError_t launch_weight_grad(const WeightGradArgs& a, int dt, hipStream_t st) {
  const int64_t tiles = (int64_t)a.E * ((a.N + kTile - 1) / kTile) * ((a.K + kTile - 1) / kTile);
  const unsigned grid = grid_of(tiles);
  if (dt == 1) weight_grad_kernel<BF16, 1><<<grid, kThreads, 0, st>>>(a);
  else weight_grad_kernel<F16, 0><<<grid, kThreads, 0, st>>>(a);
  return hipGetLastError();
}

}  // namespace mimoe
