// expert_products.hip -- matrix products on rows sorted by expert (ragged
// groups), 16-bit operands with their gradients and int8 operands with a scale
// for each row and output channel, on the matrix cores of gfx950.
//
//   y[r] = W[e] x[r]      dx[r] = W[e]^T dy[r]      dW[e] = sum_r dy[r] x[r]^T
//
// Sums run in fp32 (int32 for int8, exact) in an order that follows from the
// sizes, the expert and the output's column: a row's results are the same bits
// wherever it lies and however many rows the experts have.  Operands are read
// as they lie in memory: rows along the sum as the matrix instruction takes
// them, rows across it through transposed LDS reads, so no product needs a
// transposed copy.
//
// Which kernel: few_rows_kernel for calls of little work, else tiles of 256 x
// 256 outputs down to 128 x 64 (kFewWork, tile_shape).  Measured: bf16 8192 x
// 8192 x 4096 404 us, 1.36 PFLOP/s (the library's 1.49); int8 the same size 232 us,
// 2.37 POP/s (2.2).  The loop alone, its steps in the L2, would take 364 us at
// bf16: the card's power holds its clock at 1.9 to 2.1 GHz by then.
#pragma clang fp contract(off)
#include <type_traits>

#include "expert_products.hpp"
#include "mi_moe_device.hpp"

namespace mimoe {

namespace {

constexpr int kThreads = 512;
constexpr int kTile = 256;          // output columns of a tile, and most rows
// A step of the products' index: a cache line of a row, or 64 rows across it.
// (Loads of 64 bytes of a row make twice the requests to the L2, and those
// bound the loop: bf16 8192 x 8192 x 4096 444 us, 402 with whole lines.)
constexpr int kStepBytes = 128;
constexpr int kStepRows = 64;
constexpr int kLds = 163840 - 4096;   // of the operands; a compute unit's less the table of groups
constexpr uint32_t kOutside = 0x80000000u;     // an offset beyond any buffer: loads give zero

// Compute units, 32 in each of 8 XCDs.  Tile kernels launch a workgroup for each;
// those without a tile end at once.
constexpr int kUnits = 256;
constexpr int kRun = 32;               // place()

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

// The lane, as a value that the compiler does not know: what follows from it
// is computed where it is used, not kept in registers through a tile's products.
__device__ __forceinline__ int lane_here() {
  int l = threadIdx.x & 63;
  asm volatile("" : "+v"(l));
  return l;
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
// the 8 rows of half a transposed read do).  NSUB: subtiles of a wave.  WRAP:
// the sum may begin anywhere in the row and wrap around.
template <bool COLS, int DIM, int NSUB, bool WRAP = false>
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
  int wrap, steps;     // steps to the row's end, and of a row; WRAP
  // reads
  uint32_t at[kReads];

  // What to load: b: the tile's first element; n: its rows (COLS: columns);
  // len: length of the products' index in bytes of a row (COLS: in rows); from:
  // the step to begin with (WRAP, rows of whole steps; else 0).
  __device__ __forceinline__ void source(const unsigned char* b, int n, uint32_t ld_, int len, int from = 0) {
    base = b;
    ld = ld_;
    const int t = (threadIdx.x & ~63) | lane_here();
    if constexpr (COLS) {
      constexpr int kPieces = DIM / 8, kRows = kThreads / kPieces;   // of a row; rows of an issue
      const int k = t / kPieces, piece = t % kPieces;
#pragma unroll
      for (int i = 0; i < kIssues; ++i) {
        const int row = k + kRows * i, c = piece ^ (swizzle(row) << 1);
        off[i] = 8 * c < n ? (uint32_t)row * ld + 16u * c : kOutside;
      }
      left = len;
    } else {
#pragma unroll
      for (int i = 0; i < kIssues; ++i) {
        const int row = 64 * i + (t >> 3);
        off[i] = row < n ? (uint32_t)row * ld + 16u * piece_of(t) : kOutside;
      }
      left = (len + kStepBytes - 1) / kStepBytes;
      ragged = (len % kStepBytes) >> 4;
      if constexpr (WRAP) {
        steps = left;
        wrap = steps - from;
        base += (int64_t)from * kStepBytes;
      }
    }
    limit();
  }
  // Where to read: sub: the wave's first subtile; lds: where the ring begins
  // for this operand.
  __device__ __forceinline__ void reads(int sub, uint32_t lds) {
    const int lane = lane_here(), q = lane >> 4, r = lane & 15;
    if constexpr (COLS) {
      const int kr = 8 * q + (r >> 2);
#pragma unroll
      for (int i = 0; i < kReads; ++i) at[i] = lds + kr * (2 * DIM) + (((sub + i) ^ swizzle(kr)) << 5) + ((r & 3) << 3);
    } else {
#pragma unroll
      for (int h = 0; h < 2; ++h) at[h] = lds + (16 * sub + r) * kStepBytes + (((4 * h + q) ^ (r & 7)) << 4);
    }
  }
  static __device__ __forceinline__ int swizzle(int k) { return ((k & 3) | ((k >> 1) & 4)) & (DIM / 16 - 1); }
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
    if constexpr (WRAP) base -= --wrap == 0 ? (uint64_t)steps * kStepBytes : 0;
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

// A tile's products: acc[i][u * NQ / 2 + j] += the wave's subtile i of P times
// its subtile j of half u of Q, over all steps.
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
//
// start() begins a tile's loads before the tile before it is stored; with FLOW
// the ring runs on from tile to tile, the loads of a tile's last RING steps
// being the next tile's first.  (Short sums gain: dw of 32768 rows of 128
// experts, 4 steps a tile, 423 us, 389 with FLOW.  Long ones lose the registers:
// int8 8192 x 8192 x 4096 236 us, 240 with FLOW.)  Each wave issues at least
// STORES stores between two tiles (`warm`: there was a tile before); the first
// step does not wait for these.
template <class OP, class OQ, int STORES>
struct Ring {
  static constexpr int kStage = OP::kBytes + 2 * OQ::kBytes;
  static constexpr int kSize = kLds / kStage;
  static constexpr int kAhead = (kSize - 1) * (OP::kIssues + 2 * OQ::kIssues);
  static_assert(kSize >= 2 && kAhead + STORES < 64, "a step ahead, within the counter");
  OP P;
  OQ Q0, Q1;
  uint32_t mine;        // this wave's first kilobyte of the ring
  uint32_t cur, prev;   // places of the step at hand and of the one before

  // The first tile's loads, from the ring's first place on.
  __device__ __forceinline__ void start() {
    cur = 0;
    prev = (kSize - 1) * kStage;
#pragma unroll
    for (int s = 0; s < kSize; ++s) {
      P.load(mine + s * kStage);
      Q0.load(mine + s * kStage + OP::kBytes);
      P.advance();
      Q0.advance();
      if (s < kSize - 1) {
        Q1.load(mine + s * kStage + OP::kBytes + OQ::kBytes);
        Q1.advance();
      }
    }
  }
  static __device__ __forceinline__ void wait(bool warm) {
    __builtin_amdgcn_sched_barrier(0);
    if (warm) wait_loads_meet<kAhead + STORES>();
    else wait_loads_meet<kAhead>();
    __builtin_amdgcn_sched_barrier(0);
  }
  // FLOW: steps is at least RING; next0 / next1 set the sources of P and Q0 /
  // of Q1 to the next tile.  Else the ring is left empty.
  template <class T, bool FLOW, int NP, int NQ, class Next0, class Next1>
  __device__ __forceinline__ void products(int steps, bool late, bool warm, typename T::acc (&acc)[NP][NQ], Next0 next0, Next1 next1) {
    constexpr int NU = NQ / 2;
#pragma unroll
    for (int i = 0; i < NP; ++i)
#pragma unroll
      for (int j = 0; j < NQ; ++j) acc[i][j] = typename T::acc{0, 0, 0, 0};
    wait(warm);
    if (late) meet();
    u32x4_t p[NP][2], q[NU][2];
    auto multiply = [&](int u) {
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
    // change: the step whose loads are the next tile's first
    auto step = [&](bool first, auto change) {
      const uint32_t d = cur == (kSize - 1) * kStage ? (uint32_t)-(kSize - 1) * kStage : (uint32_t)kStage;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int i = 0; i < NP; ++i) p[i][h] = P.get(i, h);
#pragma unroll
        for (int j = 0; j < NU; ++j) q[j][h] = Q0.get(j, h);
      }
      Q1.load(mine + prev + OP::kBytes + OQ::kBytes);
      wait(first);
      multiply(0);
      Q1.advance();
      P.move(d);
      Q0.move(d);
      if constexpr (decltype(change)::value) next0();
      over();
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int j = 0; j < NU; ++j) q[j][h] = Q1.get(j, h);
      P.load(mine + cur);
      Q0.load(mine + cur + OP::kBytes);
      wait(first);
      multiply(1);
      P.advance();
      Q0.advance();
      Q1.move(d);
      if constexpr (decltype(change)::value) next1();
      prev = cur;
      cur += d;
      over();
    };
    const int plain = FLOW ? steps - kSize : steps;
    for (int s = 0; s < plain; ++s) step(warm && s == 0, std::false_type{});
    if constexpr (FLOW) {
      step(warm && plain == 0, std::true_type{});
#pragma unroll 1
      for (int s = 1; s < kSize; ++s) step(false, std::false_type{});
    }
    if (!late) meet();
    if constexpr (FLOW) fence();
    else drain();
  }
  // The stores that follow stay behind the loads so far.
  static __device__ __forceinline__ void fence() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  }
  // No load to LDS is under way any more.
  static __device__ __forceinline__ void drain() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }
};

// ------------------------------------------------------------ work items
// Groups of rows: 0 the rows before the first expert's, 1 .. E the experts,
// E + 1 the rows behind the last's.  starts is read as its running maximum
// within [0, M], so that no value of it leads outside the tensors.
struct Item {
  int e, row0, rows;   // e < 0: rows of no expert
};

__device__ __forceinline__ int items_of(int rows, int most) { return (rows + most - 1) / most; }

// The groups' items of at most `most` rows, found by every workgroup for
// itself: no launch before, no list in memory.
struct Groups {
  static constexpr int kPer = (kGroupMaxE + 2 + kWave - 1) / kWave;
  static constexpr int kTable = kWave * kPer + 1;
  int* first;    // LDS: where group g begins; M from the last group's end on
  int before;    // items of the groups of the lanes before this one
  int total;

  // All waves; ends with a barrier.
  __device__ __forceinline__ void read(int* table, const int32_t* starts, int E, int M, int most) {
    const int lane = threadIdx.x & 63;
    int end[kPer];   // of group g
    int m = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int g = lane * kPer + i;
      int s = starts[g <= E ? g : E];
      s = g <= E ? s : M;
      s = s < 0 ? 0 : s > M ? M : s;
      m = m > s ? m : s;
      end[i] = m;
    }
#pragma unroll
    for (int d = 1; d < kWave; d <<= 1) {
      const int o = __shfl_up(m, d);
      if (lane >= d) m = m > o ? m : o;
    }
    int at = __shfl_up(m, 1);
    if (lane == 0) at = 0;
    first = table;
    int n = 0, b = at;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int e = end[i] > at ? end[i] : at;
      if (threadIdx.x < kWave) table[lane * kPer + i] = b;
      n += items_of(e - b, most);
      b = e;
    }
    if (threadIdx.x == kWave - 1) table[kWave * kPer] = b;
    int sum = n;
#pragma unroll
    for (int d = 1; d < kWave; d <<= 1) {
      const int o = __shfl_up(sum, d);
      if (lane >= d) sum += o;
    }
    before = sum - n;
    total = __builtin_amdgcn_readlane(sum, 63);
    __syncthreads();
  }
  // Item `index`: a group's rows are split evenly, in multiples of `grain`.
  __device__ __forceinline__ Item find(int index, int E, int most, int grain) const {
    // the last lane whose items begin at or before index, then the group among its own
    const int owner = 63 - __builtin_clzll(__ballot(before <= index)), g0 = owner * kPer, lane = lane_here();
    const int i = lane < kPer ? lane : kPer - 1, b = first[g0 + i], e = first[g0 + i + 1];
    const int n = lane < kPer ? items_of(e - b, most) : 0;
    int end = n;
#pragma unroll
    for (int d = 1; d < 16; d <<= 1) {
      const int o = __shfl_up(end, d);
      if (lane >= d) end += o;
    }
    end += __builtin_amdgcn_readlane(before, owner);
    const int at = __builtin_ctzll(__ballot(end > index));
    const int k = index - (__builtin_amdgcn_readlane(end, at) - __builtin_amdgcn_readlane(n, at));
    const int rows = __builtin_amdgcn_readlane(e, at) - __builtin_amdgcn_readlane(b, at), g = g0 + at;
    const int size = ((rows + __builtin_amdgcn_readlane(n, at) - 1) / __builtin_amdgcn_readlane(n, at) + grain - 1) / grain * grain;
    return Item{g == 0 || g > E ? -1 : g - 1, __builtin_amdgcn_readlane(b, at) + k * size, max(0, min(size, rows - k * size))};
  }
};
static_assert(Groups::kPer <= 16, "a lane's groups fit 16 lanes");

// Items of one launch: each group adds less than one whole item.
__host__ inline int64_t items_max(int64_t M, int64_t E, int most) { return M / most + (M < E + 2 ? M : E + 2); }

// The n-th place in a list of `tiles` tiles that this workgroup takes.  The
// XCDs take runs of consecutive places in turn (XCD b % 8 runs workgroup b),
// and an XCD's gridDim / 8 workgroups take its places in turn: those that share
// an L2 at a time share rows and weights, and tiles of unequal cost spread over
// all workgroups.  Runs are of equal numbers, about kRun places long, and whole
// groups of `unit` places (those that share rows).  us, runs of 32 / 200: dw of 16384
// rows of 8 skewed experts 512 / 892, bf16 32768 rows of 128 experts 270 / 275.
__device__ __forceinline__ int place(int n, int tiles, int unit) {
  const int each = (tiles + 7) >> 3, rounds = (each + kRun - 1) / kRun, run = ((each + rounds - 1) / rounds + unit - 1) / unit * unit;
  const int j = (blockIdx.x >> 3) + n * (gridDim.x >> 3);
  return ((j / run) * 8 + (blockIdx.x & 7)) * run + j % run;
}
// Place l in the list of `items` items by `blocks` blocks of columns: 8 blocks
// of columns for every item, then the next 8.
__device__ __forceinline__ void tile_at(int l, int items, int blocks, int& item, int& block) {
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
}

// ------------------------------------------------------------ stores
// Two values rounded to 16 bits, to nearest even: one instruction for bf16 (in
// integer operations a 256 x 256 tile's stores take 8000 cycles of its SIMDs).
template <int OUT>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (OUT == 1) return __builtin_bit_cast(uint32_t, bf16x2_t{(__bf16)a, (__bf16)b});
  return __builtin_bit_cast(uint32_t, f16x2_t{(_Float16)a, (_Float16)b});
}
template <int OUT>
__device__ __forceinline__ uint16_t pack1(float a) { return (uint16_t)pack2<OUT>(a, 0.0f); }

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
    const u32x2_t w = {pack2<OUT>(v[0], v[1]), pack2<OUT>(v[2], v[3])};
    if (vec) {
      __builtin_amdgcn_raw_buffer_store_b64(w, y, (int)(n > 0 ? off : kOutside), 0, 0);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        __builtin_amdgcn_raw_buffer_store_b16((uint16_t)(w[i >> 1] >> (16 * (i & 1))), y, (int)(i < n ? off + 2 * i : kOutside), 0, 0);
    }
  }
}
template <int OUT>
__device__ __forceinline__ __amdgpu_buffer_rsrc_t out_buffer(void* y, int64_t at) {
  return buffer_of((unsigned char*)y + at * kOutBytes<OUT>, 0x7fffffff);
}
template <int OUT>
__device__ __forceinline__ bool out_vec(const void* y, int64_t ldy) { return (ldy * kOutBytes<OUT> & 15) == 0 && ((uintptr_t)y & 15) == 0; }

// `rows` rows of n <= 256 columns become zero.
template <int OUT>
__device__ __forceinline__ void zero_rows(__amdgpu_buffer_rsrc_t y, uint32_t ld, int rows, int n, bool vec) {
  for (int i = threadIdx.x; i < rows * 64; i += kThreads) {
    const int c = 4 * (i & 63);
    const float z[4] = {0, 0, 0, 0};
    store4<OUT>(y, (uint32_t)(i >> 6) * ld + c * kOutBytes<OUT>, z, n - c, vec);
  }
}

// An int8 product's output, sum * ws * xs + bias.  fp32 outputs: in 64 bits (the
// scales' product is exact), rounded once; in fp32 throughout each operation
// would round, 1.4 times the error (mean, sums of 2048 products), and the time is
// the same (8192 x 8192 x 4096 260 us): the stores take longer.  16-bit outputs:
// in fp32, four roundings of 2^-24 beside the last one of 2^-11 or 2^-8; 64 bits
// would cost a tile of 256 x 256 its registers (bf16 8192 x 8192 x 4096 227 us, 260
// so).  A sum times a scale beyond kWide may leave the range of fp32 where the
// output does not: then the other scale comes first (what it makes smaller than
// fp32's normal values is an exact multiple of the scale).
constexpr float kWide = 0x1p96f;
template <int OUT>
__device__ __forceinline__ float scaled(int32_t sum, float ws, float xs, float bias, bool wide) {
  if constexpr (OUT == 2) return (float)__builtin_fma((double)sum, (double)ws * (double)xs, (double)bias);
  const bool swap = wide && __builtin_fabsf(ws) > kWide;
  return (float)sum * (swap ? xs : ws) * (swap ? ws : xs) + bias;
}

// The values of a wave's subtiles as they leave a tile's products: lane (r, q)
// has columns 4 q .. 4 q + 3 of subtile i in row r of subtile j.  16-bit
// values change places between lane rows 2 k and 2 k + 1, so that a lane
// stores 16 bytes and four lanes 64 of a row.
template <int OUT, int NP, int NQ, class Value>
__device__ __forceinline__ void store_tile(__amdgpu_buffer_rsrc_t y, uint32_t ld, int rows, int cols, bool vec, int wp, int wq,
                                           Value value) {
  const int lane = lane_here(), r = lane & 15, q = lane >> 4;
#pragma unroll
  for (int j = 0; j < NQ; ++j) {
    const int row = 16 * (j / (NQ / 2) * NQ + NQ / 2 * wq + j % (NQ / 2)) + r;
    const bool in = row < rows;
    if (OUT == 2 || NP == 1 || !vec) {   // uniform
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        const int c = 16 * NP * wp + 16 * i + 4 * q;
        float v[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = value(i, j, k);
        store4<OUT>(y, (uint32_t)row * ld + c * kOutBytes<OUT>, v, in ? cols - c : 0, vec);
      }
    } else {
#pragma unroll
      for (int i = 0; i + 1 < NP; i += 2) {
        uint32_t w[2][2];
#pragma unroll
        for (int o = 0; o < 2; ++o)
#pragma unroll
          for (int k = 0; k < 2; ++k)
            w[o][k] = pack2<OUT & 1>(value(i + o, j, 2 * k), value(i + o, j, 2 * k + 1));
        const auto s0 = __builtin_amdgcn_permlane16_swap(w[0][0], w[1][0], false, false);
        const auto s1 = __builtin_amdgcn_permlane16_swap(w[0][1], w[1][1], false, false);
        const int c = 16 * NP * wp + 16 * (i + (q & 1)) + 8 * (q >> 1);
        const u32x4_t v = {s0[0], s1[0], s0[1], s1[1]};
        __builtin_amdgcn_raw_buffer_store_b128(v, y, (int)(in && c < cols ? (uint32_t)row * ld + 2 * c : kOutside), 0, 0);
      }
    }
  }
}

// ------------------------------------------------------------ rows
// Items of up to 64 and 128 rows (SMALL) keep three steps of 256 columns in LDS
// (128 columns: four, 64: six), those of up to 192 and 256 rows two (three, three).
// WRAP: sums begin at a step of the row that the expert and the block of columns
// decide, see wrap_sums().
template <class T, bool WCOLS, int OUT, int NP, bool WRAP>
struct Rows {
  static constexpr int kElem = std::is_same<T, I8>::value ? 1 : 2, kCols = 64 * NP;
  using OpW = Operand<WCOLS, kCols, NP, WRAP>;
  template <bool SMALL>
  using OpX = Operand<false, SMALL ? 64 : 128, 0, WRAP>;   // half of the rows
  const RowProductArgs& a;
  Groups groups;
  uint32_t lds;
  int wp, wq, n, blocks;
  // the tile at hand
  Item it;
  int p0;
  bool live;

  __device__ __forceinline__ void next() {
    const int items = a.starts ? groups.total : items_of(a.M, a.most), tiles = items * blocks;
    const int l = place(n++, tiles, tiles < kUnits ? 1 : min(blocks, 8));
    live = l < tiles;
    if (!live) return;
    int item, block;
    tile_at(l, items, blocks, item, block);
    it = a.starts ? groups.find(item, a.E, a.most, 32) : Item{0, item * a.most, min(a.most, a.M - item * a.most)};
    p0 = block * kCols;
  }
  // rows of half an item as its products take them
  static __device__ __forceinline__ int half(int rows) { return rows <= 64 ? 32 : rows <= 128 ? 64 : rows <= 192 ? 96 : 128; }

  template <bool SMALL, class R>
  __device__ __forceinline__ void start(R& ring) const {
    constexpr int kW = OpW::kBytes, kX = OpX<SMALL>::kBytes;
    const unsigned char *w = a.w + (int64_t)it.e * a.w_expert, *x = a.x + (int64_t)it.row0 * a.ldx;
    const int len = a.K * kElem, h = half(it.rows);
    const int from = WRAP ? (it.e * blocks + p0 / kCols) % (len / kStepBytes) : 0;
    ring.P.source(w + (int64_t)p0 * (WCOLS ? kElem : a.ldw), min(kCols, a.P - p0), a.ldw, WCOLS ? a.K : len, from);
    ring.Q0.source(x, min(it.rows, h), a.ldx, len, from);
    ring.Q1.source(x + (int64_t)h * a.ldx, it.rows - h, a.ldx, len, from);
    ring.P.reads(NP * wp, lds);
    ring.Q0.reads(h / 32 * wq, lds + kW);
    ring.Q1.reads(h / 32 * wq, lds + kW + kX);
    ring.start();
  }

  // The tile at hand, whose loads have begun; begins those of the next one if
  // it is of the same kind (returns whether).
  template <bool SMALL, int NQ, class R>
  __device__ __forceinline__ bool tile(R& ring, bool warm) {
    const Item done = it;
    const int d0 = p0, cols = min(kCols, a.P - p0);
    typename T::acc acc[NP][NQ];
    ring.template products<T, false>((a.K * kElem + kStepBytes - 1) / kStepBytes, wq != 0, warm, acc, [] {}, [] {});
    const int lane = lane_here(), r = lane & 15, q = lane >> 4;
    float ws[NP][4], bias[NP][4], xs[NQ];
    if constexpr (kElem == 1) {
#pragma unroll
      for (int i = 0; i < NP; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int p = min(d0 + 16 * NP * wp + 16 * i + 4 * q + k, a.P - 1);
          ws[i][k] = a.ws[(int64_t)done.e * a.P + p];
          bias[i][k] = a.bias ? a.bias[p] : 0.0f;
        }
#pragma unroll
      for (int j = 0; j < NQ; ++j)
        xs[j] = a.xs[done.row0 + min(16 * (j / (NQ / 2) * NQ + NQ / 2 * wq + j % (NQ / 2)) + r, done.rows - 1)];
    }
    next();
    const bool same = live && it.e >= 0 && it.rows > 0 && (it.rows <= 128) == SMALL;
    if (same) {
      start<SMALL>(ring);
      ring.fence();
    }
    auto store = [&](auto wide) {
      store_tile<OUT, NP, NQ>(out_buffer<OUT>(a.y, (int64_t)done.row0 * a.ldy + d0), (uint32_t)(a.ldy * kOutBytes<OUT>), done.rows, cols,
                              out_vec<OUT>(a.y, a.ldy), wp, wq, [&](int i, int j, int k) {
                                if constexpr (kElem == 1)
                                  return scaled<OUT>(acc[i][j][k], ws[i][k], xs[j], bias[i][k], decltype(wide)::value);
                                else return acc[i][j][k];
                              });
    };
    if constexpr (kElem == 1 && OUT != 2) {
      bool wide = false;
#pragma unroll
      for (int i = 0; i < NP; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) wide |= !(__builtin_fabsf(ws[i][k]) <= kWide);
      if (__builtin_amdgcn_ballot_w64(wide)) store(std::true_type{});
      else store(std::false_type{});
    } else {
      store(std::false_type{});
    }
    return same;
  }
  template <bool SMALL>
  __device__ __forceinline__ void tiles() {
    // stores of the smaller kind of tile
    Ring<OpW, OpX<SMALL>, (SMALL ? 2 : 6) * (OUT == 2 || NP == 1 ? NP : NP / 2)> ring;
    ring.mine = lds + uni(threadIdx.x >> 6) * 1024;
    start<SMALL>(ring);
    for (bool warm = false, same = true; same; warm = true) {
      if (SMALL) same = it.rows <= 64 ? tile<SMALL, 2>(ring, warm) : tile<SMALL, 4>(ring, warm);
      else same = it.rows <= 192 ? tile<SMALL, 6>(ring, warm) : tile<SMALL, 8>(ring, warm);
    }
    __syncthreads();   // the ring may be another's
  }
};

// Tiles of up to 256 rows by 64 NP columns: 8 waves, two rows of four.  256
// rows an expert put the weights' bytes and the products in balance: bf16 32768
// rows of 128 experts, N=1536 K=2048: 270 us, 3.8 TB/s of what it has to move and
// 0.76 PFLOP/s (without loads 177 us; with loads of the L2 alone 198); its dx 285.
// 16384 rows of 8 skewed experts, 4096 x 4096: 470 us, 1.17 PFLOP/s; dx 490.  Rows
// that are no whole cache lines (K=1440) make 1.5 times the requests to the L2:
// 30000 rows of 64 experts, N=4096: 431 us, 0.82 PFLOP/s.
template <class T, bool WCOLS, int OUT, int NP, bool WRAP>
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(2))) void row_product_kernel(RowProductArgs a) {
  __shared__ __align__(16) unsigned char smem[kLds];
  __shared__ int table[Groups::kTable];
  const int wave = uni(threadIdx.x >> 6);
  Rows<T, WCOLS, OUT, NP, WRAP> rows{a};
  rows.lds = (uint32_t)(uintptr_t)(lds_byte*)smem;
  rows.wp = wave & 3;
  rows.wq = wave >> 2;
  rows.n = 0;
  rows.blocks = (a.P + rows.kCols - 1) / rows.kCols;
  if (a.starts) rows.groups.read(table, a.starts, a.E, a.M, a.most);
  rows.next();
  while (rows.live) {
    const Item& it = rows.it;
    if (it.e < 0 || it.rows <= 0) {
      zero_rows<OUT>(out_buffer<OUT>(a.y, (int64_t)it.row0 * a.ldy + rows.p0), (uint32_t)(a.ldy * kOutBytes<OUT>), it.rows,
                     min(rows.kCols, a.P - rows.p0), out_vec<OUT>(a.y, a.ldy));
      rows.next();
    } else if (it.rows <= 128) {
      rows.template tiles<true>();
    } else {
      rows.template tiles<false>();
    }
  }
}

// ------------------------------------------------------------ few rows
// Products of few rows (a decode call, some rows an expert) are bound by the
// weights' bytes, or by latency.  A workgroup takes 16 columns of an item of up
// to 64 rows; its 4 waves split the products' index, load what the matrix
// instruction takes straight to registers, many loads at once, and add up
// through LDS (in the order of the waves).  bf16, one token's 8 of 128 experts
// 1536 x 2048, 50 MB: 11.6 us, 4.3 TB/s; int8 450 rows of 128 experts 1024 x 2048,
// 268 MB: 60 us, 4.5 TB/s (a copy: 4.9); int8 one row 4096 x 2048: 3.8 us.
constexpr int kFewThreads = 256, kFewRows = 64, kFewCols = 16;

template <class T, int OUT, int MT>
__device__ __forceinline__ void few_item(const RowProductArgs& a, float* sums, const Item& it, int p0) {
  constexpr int kElem = std::is_same<T, I8>::value ? 1 : 2, kBatch = MT == 1 ? 8 : 4;
  const int lane = threadIdx.x & 63, wave = uni(threadIdx.x >> 6), r = lane & 15, q = lane >> 4;
  const int len = a.K * kElem, chunks = (len + 63) >> 6, per = (chunks + 3) >> 2, c0 = wave * per, c1 = min(chunks, c0 + per);
  const __amdgpu_buffer_rsrc_t wb = buffer_of(a.w + (int64_t)it.e * a.w_expert + (int64_t)p0 * a.ldw, 0x7fffffff);
  const __amdgpu_buffer_rsrc_t xb = buffer_of(a.x + (int64_t)it.row0 * a.ldx, 0x7fffffff);
  const uint32_t wo = p0 + r < a.P ? r * a.ldw : kOutside;
  uint32_t xo[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) xo[m] = 16 * m + r < it.rows ? (16 * m + r) * a.ldx : kOutside;
  typename T::acc acc[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) acc[m] = typename T::acc{0, 0, 0, 0};
  for (int c = c0; c < c1; c += kBatch) {
    u32x4_t w[kBatch], x[kBatch][MT];
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const uint32_t at = 64 * (c + u) + 16 * q;
      const bool in = c + u < c1 && at < (uint32_t)len;
      w[u] = __builtin_amdgcn_raw_buffer_load_b128(wb, (int)(in && wo != kOutside ? wo + at : kOutside), 0, 0);
#pragma unroll
      for (int m = 0; m < MT; ++m)
        x[u][m] = __builtin_amdgcn_raw_buffer_load_b128(xb, (int)(in && xo[m] != kOutside ? xo[m] + at : kOutside), 0, 0);
    }
#pragma unroll
    for (int u = 0; u < kBatch; ++u)
#pragma unroll
      for (int m = 0; m < MT; ++m) mma(T{}, w[u], x[u][m], acc[m]);
  }
  typedef typename T::acc acc_t;
  acc_t* part = reinterpret_cast<acc_t*>(sums);
#pragma unroll
  for (int m = 0; m < MT; ++m) part[(wave * MT + m) * kWave + lane] = acc[m];
  __syncthreads();
  // a thread an output: column t % 16 of rows t / 16, + 16, ..
  const int n = threadIdx.x & 15, row = threadIdx.x >> 4;
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    auto v = part[m * kWave + (n >> 2) * 16 + row][n & 3];
#pragma unroll
    for (int k = 1; k < 4; ++k) v += part[(k * MT + m) * kWave + (n >> 2) * 16 + row][n & 3];
    const int mr = 16 * m + row, p = p0 + n;
    if (mr < it.rows && p < a.P) {
      float f;
      if constexpr (kElem == 1) f = scaled<OUT>(v, a.ws[(int64_t)it.e * a.P + p], a.xs[it.row0 + mr], a.bias ? a.bias[p] : 0.0f, true);
      else f = v;
      const int64_t at = (int64_t)(it.row0 + mr) * a.ldy + p;
      if constexpr (OUT == 2) reinterpret_cast<float*>(a.y)[at] = f;
      else reinterpret_cast<uint16_t*>(a.y)[at] = pack1<OUT>(f);
    }
  }
  __syncthreads();   // the sums may be written again
}

template <class T, int OUT>
__global__ __launch_bounds__(kFewThreads) __attribute__((amdgpu_waves_per_eu(4))) void few_rows_kernel(RowProductArgs a) {
  __shared__ __align__(16) float sums[4 * 4 * kWave * 4];
  __shared__ int table[Groups::kTable];
  Groups groups;
  if (a.starts) groups.read(table, a.starts, a.E, a.M, kFewRows);
  const int items = a.starts ? groups.total : items_of(a.M, kFewRows), blocks = (a.P + kFewCols - 1) / kFewCols;
  for (int64_t l = blockIdx.x; l < (int64_t)items * blocks; l += gridDim.x) {
    const int item = (int)(l / blocks), p0 = (int)(l - (int64_t)item * blocks) * kFewCols;
    const Item it = a.starts ? groups.find(item, a.E, kFewRows, 16) : Item{0, item * kFewRows, min(kFewRows, a.M - item * kFewRows)};
    if (it.e < 0) {
      const int n = threadIdx.x & 15, p = p0 + n;
      for (int row = threadIdx.x >> 4; row < it.rows; row += 16) {
        const int64_t at = (int64_t)(it.row0 + row) * a.ldy + p;
        if (p < a.P) {
          if constexpr (OUT == 2) reinterpret_cast<float*>(a.y)[at] = 0.0f;
          else reinterpret_cast<uint16_t*>(a.y)[at] = 0;
        }
      }
    } else if (it.rows <= 16) {
      few_item<T, OUT, 1>(a, sums, it, p0);
    } else if (it.rows <= 32) {
      few_item<T, OUT, 2>(a, sums, it, p0);
    } else {
      few_item<T, OUT, 4>(a, sums, it, p0);
    }
  }
}

// ------------------------------------------------------------ weight gradient
// Both operands lie across the sum.  Tiles of 256 x 256 of dw, stored once: no
// sum is split, so none is added up in memory.  Experts of 256 rows are bound
// by the stores, which no product of the same tile overlaps: 32768 rows of 128
// experts, 1536 x 2048, 805 MB of dw: 389 us (the stores alone 131, loads and
// products without them 264; two workgroups of 4 waves a compute unit, so that
// one stores while the other multiplies, took 454).  16384 rows of 8 experts 4096 x 4096:
// 500 us, 1.1 PFLOP/s.
template <class T, int OUT>
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(2))) void weight_grad_kernel(WeightGradArgs a) {
  __shared__ __align__(16) unsigned char smem[kLds];
  __shared__ int table[Groups::kTable];
  typedef Operand<true, kTile, 4> OpX;
  typedef Operand<true, kTile / 2, 4> OpY;   // half of the columns of dy
  const int wave = uni(threadIdx.x >> 6), wp = wave & 3, wq = wave >> 2;
  const uint32_t lds = (uint32_t)(uintptr_t)(lds_byte*)smem;
  const int bk = (a.K + kTile - 1) / kTile, bn = (a.N + kTile - 1) / kTile;
  Groups groups;
  groups.read(table, a.starts, a.E, a.M, kTile);
  Ring<OpX, OpY, 16> ring;
  ring.mine = lds + wave * 1024;
  int n = 0, e, n0, k0, rows;
  const unsigned char* dy;
  auto next = [&]() -> bool {
    const int each = bn * bk, l = place(n++, a.E * each, 1);
    if (l >= a.E * each) return false;
    e = l / each;   // one expert after the other: tiles of one cost
    int item, block;
    tile_at(l - e * each, bn, bk, item, block);
    n0 = item * kTile;
    k0 = block * kTile;
    rows = uni(table[e + 2]) - uni(table[e + 1]);
    return true;
  };
  auto source0 = [&] {
    const int64_t b = uni(table[e + 1]);
    dy = a.dy + b * a.lddy + (int64_t)n0 * 2;
    ring.P.source(a.x + b * a.ldx + (int64_t)k0 * 2, min(kTile, a.K - k0), a.ldx, rows);
    ring.Q0.source(dy, min(kTile / 2, a.N - n0), a.lddy, rows);
  };
  auto source1 = [&] { ring.Q1.source(dy + kTile, a.N - n0 - kTile / 2, a.lddy, rows); };
  bool more = next();
  if (!more) return;
  ring.P.reads(4 * wp, lds);
  ring.Q0.reads(4 * wq, lds + OpX::kBytes);
  ring.Q1.reads(4 * wq, lds + OpX::kBytes + OpY::kBytes);
  source0();
  source1();
  ring.start();
  for (bool warm = false; more; warm = true) {
    f32x4_t acc[4][8];
    const int de = e, dn = n0, dk = k0;
    // at least as many steps as the ring has places: sums of no or few rows go on with zeros
    ring.template products<T, true>(
        max((rows + kStepRows - 1) / kStepRows, ring.kSize), wq != 0, warm, acc,
        [&] {
          more = next();
          if (more) source0();
        },
        [&] {
          if (more) source1();
        });
    store_tile<OUT, 4, 8>(out_buffer<OUT>(a.dw, ((int64_t)de * a.N + dn) * a.K + dk), (uint32_t)(a.K * kOutBytes<OUT>), a.N - dn, a.K - dk,
                          out_vec<OUT>(a.dw, a.K), wp, wq, [&](int i, int j, int k) { return acc[i][j][k]; });
  }
  ring.drain();   // no load to LDS outlives the workgroup
}

// Up to this much work (rows * columns * bytes of a weight row) the few-rows
// kernel runs: it reads the weights at the rate of a copy, but the rows again
// for every 16 columns.  us, few / tiles: int8, one weight 4096 x 4096: 16 rows
// 6.7 / 16, 64 rows (1.1e9) 14 / 17, 128 rows (2.1e9) 22 / 21; 8192 x 8192: 16 rows
// (1.1e9) 20 / 28, 32 rows (2.1e9) 28 / 28; bf16, 128 experts 1536 x 2048: 128 rows
// (0.8e9) 109 / 118, 512 rows (3.2e9) 178 / 181, 1024 rows 203 / 184; 8 experts 4096 x
// 4096: 64 rows (2.1e9) 67 / 68, 256 rows 118 / 70.
constexpr int64_t kFewWork = 3 << 29;

// Rows and columns of a tile: 256 x 256, which moves least through the L2 and
// LDS for a product, unless that leaves compute units without a tile; then the
// shape with most tiles that still has a unit for each.  Narrow and low tiles
// keep more steps in LDS, which hides more of the memory's latency.  us at 256 x
// 256 / 256 x 128 / 128 x 128 / 256 x 64 / 128 x 64, int8 4096 x 4096: 256 rows 49 / 28 / 22 / 25 /
// 21 (the last has 128 tiles), 1024 rows 51 / 31 / 25 / 29 / 41 (128 x 128 has 256), 2048 rows
// 55 / 40 / 50 / 59 / 78 (256 x 128 has 256).
struct Shape {
  int rows, np;
};
Shape tile_shape(const RowProductArgs& a) {
  constexpr Shape shapes[] = {{256, 4}, {256, 2}, {128, 2}, {256, 1}, {128, 1}};
  Shape best = shapes[0];
  int64_t most = 0;
  for (const Shape& s : shapes) {
    // experts of few rows are an item each; others leave half an item over on average
    const int64_t groups = a.M < a.E ? a.M : a.E, whole = a.M / s.rows;
    const int64_t items = !a.starts ? (a.M + s.rows - 1) / s.rows : groups > whole + groups / 2 ? groups : whole + groups / 2;
    const int64_t tiles = items * ((a.P + 64 * s.np - 1) / (64 * s.np));
    if (tiles <= kUnits && tiles > most) {
      most = tiles;
      best = s;
    }
  }
  return best;
}

template <class T, int OUT>
void few_rows(const RowProductArgs& a, hipStream_t st) {
  const int64_t items = a.starts ? items_max(a.M, a.E, kFewRows) : (a.M + kFewRows - 1) / kFewRows;
  const int64_t tiles = items * ((a.P + kFewCols - 1) / kFewCols);
  few_rows_kernel<T, OUT><<<(unsigned)(tiles < 4 * kUnits ? tiles : 4 * kUnits), kFewThreads, 0, st>>>(a);
}

// Experts of few rows read the weights at the rate of the memory.  Where rows
// are a power of two long, all workgroups at one place of theirs would put
// their reads on few of its channels, so tiles begin their sums at different
// steps.  Which one follows from the expert and the block of columns, and
// whether from the sizes, for tiles of any number of rows, so that no sum's
// order depends on starts.  bf16, us without / so: 128 experts 1536 x 2048, 512
// rows 189 / 162, 4096 rows 200 / 171, 24576 rows 270 / 238; 8 experts 4096 x 4096,
// 256 rows 70 / 59; skewed 160 to 224 rows an expert 1 to 3% slower, and so
// from 256 rows an expert on.  int8, half as many steps: within 1.5% either way, not
// done; nor in tiles of 64 columns, taken where compute units are left over.
template <int NP, bool WCOLS, class T>
constexpr bool kMayWrap = !WCOLS && !std::is_same<T, I8>::value && NP >= 2;
bool wrap_sums(const RowProductArgs& a) { return a.starts && a.M < (int64_t)kTile * a.E && a.K * 2 % kStepBytes == 0; }

template <class T, bool WCOLS, int OUT, int NP>
void tiles(const RowProductArgs& a, hipStream_t st) {
  if constexpr (kMayWrap<NP, WCOLS, T>) {
    if (wrap_sums(a)) {
      row_product_kernel<T, WCOLS, OUT, NP, true><<<kUnits, kThreads, 0, st>>>(a);
      return;
    }
  }
  row_product_kernel<T, WCOLS, OUT, NP, false><<<kUnits, kThreads, 0, st>>>(a);
}

template <class T, bool WCOLS, int OUT>
void row_product(const RowProductArgs& a, hipStream_t st) {
  if constexpr (!WCOLS) {
    if ((int64_t)a.M * a.P * a.K <= kFewWork / (std::is_same<T, I8>::value ? 1 : 2)) return few_rows<T, OUT>(a, st);
  }
  const Shape s = tile_shape(a);
  RowProductArgs b = a;
  b.most = s.rows;
  if (s.np == 1) tiles<T, WCOLS, OUT, 1>(b, st);
  else if (s.np == 2) tiles<T, WCOLS, OUT, 2>(b, st);
  else tiles<T, WCOLS, OUT, 4>(b, st);
}

}  // namespace

hipError_t launch_row_product(const RowProductArgs& a, int dt, int w_cols, int out, hipStream_t st) {
  if (dt == 2) {
    if (out == 0) row_product<I8, false, 0>(a, st);
    else if (out == 1) row_product<I8, false, 1>(a, st);
    else row_product<I8, false, 2>(a, st);
  } else if (dt == 1) {
    if (w_cols) row_product<BF16, true, 1>(a, st);
    else row_product<BF16, false, 1>(a, st);
  } else {
    if (w_cols) row_product<F16, true, 0>(a, st);
    else row_product<F16, false, 0>(a, st);
  }
  return hipGetLastError();
}

hipError_t launch_weight_grad(const WeightGradArgs& a, int dt, hipStream_t st) {
  if (dt == 1) weight_grad_kernel<BF16, 1><<<kUnits, kThreads, 0, st>>>(a);
  else weight_grad_kernel<F16, 0><<<kUnits, kThreads, 0, st>>>(a);
  return hipGetLastError();
}

}  // namespace mimoe
