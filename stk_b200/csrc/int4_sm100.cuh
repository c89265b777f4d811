// Matrix-vector products with the experts' 4-bit weights: y[s] = W_e x[s / x_div] for every slot s that chose expert
// e, W = (code - zero) * scale with a scale (and a zero point, 8 where there is none) for each output row and group of
// 32, 64 or 128 inputs.
//
// The bytes of the chosen experts' weights are the floor: a weight is half a byte, so at 6.5 TB/s an SM has to take in 46
// weights a clock, more than it could convert and multiply on the CUDA cores in 32 bits (three instructions a weight).
// So the products run as mma.m16n8k16: 16 output rows x 16 inputs of weights against 8 slots, sums in 32 bits.  The A
// operand is code - zero: putting an exponent above the code's four bits makes 16 + code, a 16-bit float (one shift and one
// logical instruction for two weights), and a packed subtraction takes 16 + zero away (one more); both are exact.  The
// scale multiplies a group's sum.  So the only roundings are those of sums of (code - zero) x and of scaled group sums, in 32
// bits, and that of the result: the error goes by sum |w x|, and an input whose code is the zero point adds exactly nothing.
// (Summing (16 + code) x and taking (16 + zero) sum x away from the sum instead is cheaper by the subtractions and dearer by
// a table of input sums, and its error goes by sum (32 + code + zero) |scale x|, which outliers among the inputs make
// large.)  An infinity among the inputs makes its results infinite, or NaN where its weight is 0; so do finite ones whose sum
// of (code - zero) x over a group is beyond the range of 32 bits (bf16 inputs above 1e35).
//
// Layout (made once, by the host): a record holds 32 output rows (two strips of 16) x 128 inputs, in the order in which
// the kernel reads them.  First the codes, strip by strip, 64 inputs at a time, 512 bytes in the order in which the lanes
// of a warp hold the A operand: lane (g, t) = (lane / 4, lane % 4) has 16 bytes, word 2h + s of them the weights of rows
// g and g + 8 for the inputs 32h + 8t + 4s + {0, 1, 2, 3}; nibble 4b + 2p + r: row g + 8r, input 2p + b of the four.  (The
// order of the inputs inside a product is free, so a lane's share of x is 16 contiguous bytes.)  A word is turned left by
// 3 bits (bf16) or 6 (fp16), so that its first two codes lie where a 16-bit float has its last exact bits.  Then the
// scales [group of the record][strip][g][r], then the zero points in the same order, a byte each.  What is beyond the
// last row or input is code 0, scale 0, zero point 0, and not added up.
//
// One CTA of 16 warps per SM takes an equal share of the records' rows (of every expert and tile of up to 16 of its
// slots), several of them at a time: an item is 1, 2, 4, 8 or 16 of them, as many as are left, so that shares stay equal
// to a record's rows; 16 / that many warps cut each row along the inputs, and their sums are joined in shared memory, in
// order.  Each warp streams its records through a ring of its own, by bulk copies that one lane starts; the copies run
// ahead across the items.
//
// 32 slots on 8 experts of 4096 inputs x 14336 outputs, bf16, group 128 (242 MB, 37 us of HBM time): 64 - 70 us; the copies
// alone take 41.  20.6 instructions for a word of 8 codes a lane, 9.5 of them on the integer pipe (59 % busy) and 4 the
// subtractions (58 - 62 us with a table of input sums in their place, which is not exact); 0.64 instructions a clock and scheduler,
// mma.sync 25 % busy: no one unit is full, the schedulers and the integer pipe together are nearest to it.  Measured and no
// better: two rows of records per warp sharing their loads of x, 24 warps of 80 registers, a ring of 4, shifts by
// multiplication, the subtraction as a packed multiply-add.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include <atomic>

#include "../../include/stk_b200.h"
#include "bsmm_sm100.cuh"
#include "gate_sm100.cuh"
#include "sm100_ptx.cuh"
#include "status.cuh"

namespace stk {

constexpr int kInt4Warps = 16;
constexpr int kInt4Threads = 32 * kInt4Warps;
constexpr int kInt4Strips = 2;                      // strips of a record
constexpr int kInt4Rows = 16 * kInt4Strips;         // output rows of a record
constexpr int kInt4Inputs = 128;                    // inputs of a record
constexpr int kInt4Stages = 2;                      // records of a warp's ring
constexpr int kInt4MaxExperts = 1024;
constexpr int kInt4MaxSlots = 256;                  // of one launch
constexpr int kInt4MaxGroups = 512;                 // of the inputs
constexpr int kInt4MaxTiles = 2;                    // products of 8 slots per item
constexpr int kInt4MaxEntries = kInt4MaxSlots;      // (expert, tile) pairs: each holds a slot at least

template <int kGroup>
struct Int4RecordBase {
  static constexpr int kGroups = kInt4Inputs / kGroup;
  uint4 words[kInt4Strips][2][32];
  uint32_t scales[kGroups][kInt4Strips][8];         // rows g and g + 8
};
template <int kGroup, bool kZeros>
struct Int4Record : Int4RecordBase<kGroup> {};
template <int kGroup>
struct Int4Record<kGroup, true> : Int4RecordBase<kGroup> {
  uint16_t zeros[Int4RecordBase<kGroup>::kGroups][kInt4Strips][8];
};
struct Int4Args {
  const unsigned char* records;  // [experts][outputs / 32][inputs / 128], rounded up
  const void* x;          // [.., inputs], contiguous
  const int32_t* ids;     // [slots]
  void* out;              // [slots][outputs]: T, or float
  int slots, first_slot;  // slots of this launch; the first one's number
  int x_div, experts, outputs, inputs;
  int min_log;            // log2 of the fewest row groups of an item
  int gelu, out_f32;
};

constexpr int kInt4MaxLog = 4;                      // log2 of the most rows of records of an item: a warp each

// The items of a CTA, one after the other: rows of records [block, block + n) of an entry, n <= 2^log, 16 >> log warps each.
struct Int4Item {
  int left;                // rows of records of the CTA's share from this item on
  int entry, block, n, log;
  int c0, c1, row;         // the warp's part: these records of this row (from `block` on)
  __device__ __forceinline__ void settle(const Int4Args& a, int blocks, int units, int warp) {
    n = min(left, blocks - block);
    log = kInt4MaxLog;
    static_assert(kInt4Warps == 1 << kInt4MaxLog, "");
    while (log > a.min_log && (1 << log) > n) --log;
    n = min(n, 1 << log);
    const int split_log = kInt4MaxLog - log, share = warp & ((1 << split_log) - 1);
    row = warp >> split_log;
    c0 = units * share >> split_log;
    c1 = row < n ? units * (share + 1) >> split_log : c0;
  }
  __device__ __forceinline__ bool next(const Int4Args& a, int blocks, int units, int warp) {
    left -= n;
    block += n;
    if (block == blocks) {
      block = 0;
      ++entry;
    }
    if (left <= 0) return false;
    settle(a, blocks, units, warp);
    return true;
  }
};

// Where a warp's copies have got to.
struct Int4Cursor {
  const unsigned char* record;  // the next one
  int more;                     // of the item still to be copied
  uint32_t head;                // copied so far; the next one goes to stage head % kInt4Stages
  int left, entry, block;       // the items after it
};

template <int kGroup, bool kZeros>
struct Int4Smem {
  Int4Record<kGroup, kZeros> ring[kInt4Warps][kInt4Stages];
  float joined[kInt4Warps][kInt4Strips * kInt4MaxTiles * 4][32];
  uint64_t full[kInt4Warps][kInt4Stages];
  int32_t list[kInt4MaxSlots];                      // slots, expert by expert
  int32_t row[kInt4MaxSlots];                       // their rows of x
  uint16_t entry_expert[kInt4MaxEntries];
  uint16_t entry_first[kInt4MaxEntries];            // in the list
  uint16_t entry_slots[kInt4MaxEntries];
  int32_t counter[kInt4MaxExperts];
  int32_t entries;
  int32_t dropped;
  int32_t stuck;
};

template <typename T> struct Int4Type;
template <> struct Int4Type<__nv_bfloat16> {
  static constexpr uint32_t kMagic = 0x41804180u;  // 16, with steps of 1 from bit 3 on
  static constexpr int kBit = 3;
  static constexpr uint32_t kOffset = 0x41c041c0u;  // 24: the magic number and a zero point of 8
  __device__ static uint32_t minus(uint32_t a, uint32_t b) {
    const __nv_bfloat162 d = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
    return *reinterpret_cast<const uint32_t*>(&d);
  }
  __device__ static float2 pair(uint32_t v) { return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&v)); }
  __device__ static void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
  __device__ static void mma_from(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, const float (&c)[4]) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
  }
};
template <> struct Int4Type<__half> {
  static constexpr uint32_t kMagic = 0x4c004c00u;  // 16, with steps of 1 from bit 6 on
  static constexpr int kBit = 6;
  static constexpr uint32_t kOffset = 0x4e004e00u;  // 24
  __device__ static uint32_t minus(uint32_t a, uint32_t b) {
    const __half2 d = __hsub2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&d);
  }
  __device__ static float2 pair(uint32_t v) { return __half22float2(*reinterpret_cast<const __half2*>(&v)); }
  __device__ static void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
  __device__ static void mma_from(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, const float (&c)[4]) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
  }
};

// code - zero for the 8 codes of a word, as the A operand of one product; lo and hi are 16 + zero of rows g and g + 8.  mask
// and magic are registers (int4_constant): one logical instruction takes one immediate, and with two constants known to it
// the compiler makes two of it (14 instead of 7 integer instructions a word).
template <typename T>
__device__ __forceinline__ void int4_decode(uint32_t w, uint32_t mask, uint32_t magic, uint32_t lo, uint32_t hi,
                                            uint32_t (&a)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t v;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(v) : "r"(__funnelshift_r(w, w, 4 * i)), "r"(mask), "r"(magic));
    a[i] = Int4Type<T>::minus(v, i % 2 ? hi : lo);
  }
}
__device__ __forceinline__ uint32_t int4_constant(uint32_t v) {
  uint32_t r;
  asm volatile("mov.b32 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

// x Phi(x) = x erfc(-x / sqrt 2) / 2, for a few outputs each: to (x^2 + 8) 2^-23, relative, in the tail too (from the rounded
// argument's x^2 2^-23 and erfcf's own error).  Below -16 it is beneath 32 bits, and -infinity gives -0 as in the products'
// epilogues, whose shorter form has a constant tail below -8.  A NaN stays one.
__device__ __forceinline__ float int4_gelu(float x) { return x < -16.0f ? -0.0f : 0.5f * x * erfcf(-0.70710678f * x); }

__device__ __forceinline__ void int4_copy(uint32_t to, const void* from, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
               ::"r"(to), "l"(from), "r"(bytes), "r"(bar) : "memory");
}

// To the first record of the next item in which the warp has a part.
template <int kGroup, bool kZeros>
__device__ __forceinline__ void int4_point(const Int4Args& a, const Int4Smem<kGroup, kZeros>& sm, int blocks, int units,
                                           int warp, Int4Cursor& c) {
  Int4Item item;
  while (c.left > 0) {
    item.left = c.left;
    item.block = c.block;
    item.settle(a, blocks, units, warp);
    const int64_t row = static_cast<int64_t>(sm.entry_expert[c.entry]) * blocks + c.block + item.row;
    c.left -= item.n;
    c.block += item.n;
    if (c.block == blocks) {
      c.block = 0;
      ++c.entry;
    }
    if (item.c0 >= item.c1) continue;
    c.record = a.records + (row * units + item.c0) * static_cast<int64_t>(sizeof(Int4Record<kGroup, kZeros>));
    c.more = item.c1 - item.c0;
    return;
  }
}

// Starts the next copy; every lane has read the stage that it goes to.
template <int kGroup, bool kZeros>
__device__ __forceinline__ void int4_fetch(const Int4Args& a, Int4Smem<kGroup, kZeros>& sm, int blocks, int units, int warp,
                                           int lane, Int4Cursor& c) {
  constexpr uint32_t kBytes = sizeof(Int4Record<kGroup, kZeros>);
  static_assert(kBytes % 16 == 0 && kBytes == 2048 + kInt4Inputs / kGroup * kInt4Rows * (kZeros ? 3 : 2), "bulk copies");
  if (c.more == 0) return;
  if (lane == 0) {
    const uint32_t bar = smem_u32(&sm.full[warp][c.head % kInt4Stages]);
    mbar_arrive_expect_tx(bar, kBytes);
    int4_copy(smem_u32(&sm.ring[warp][c.head % kInt4Stages]), c.record, kBytes, bar);
  }
  ++c.head;
  c.record += kBytes;
  if (--c.more == 0) int4_point<kGroup, kZeros>(a, sm, blocks, units, warp, c);
}

// x of the entry's slots as the lanes hold the B operand: 8 inputs of slot 8 n + g.
template <typename T, int NT, int kGroup, bool kZeros>
struct Int4Inputs {
  const T* x[NT];
  __device__ __forceinline__ Int4Inputs(const Int4Args& a, const Int4Smem<kGroup, kZeros>& sm, int first, int slots, int c,
                                        int lane) {
#pragma unroll
    for (int n = 0; n < NT; ++n)
      // (columns beyond the slots repeat the last one: a column of a product does not reach the others)
      x[n] = static_cast<const T*>(a.x) + static_cast<int64_t>(sm.row[first + min(8 * n + lane / 4, slots - 1)]) * a.inputs +
             c * kInt4Inputs + 8 * (lane % 4);
  }
  __device__ __forceinline__ void next() {
#pragma unroll
    for (int n = 0; n < NT; ++n) x[n] += kInt4Inputs;
  }
  // A quarter, of 32 inputs, of record c, which x is at.  (One beyond the inputs is not added up: any of the row's values
  // will do.  A choice between loaded values and zeros would wait for the load where it stands.)
  __device__ __forceinline__ void load(const Int4Args& a, int c, int quarter, uint4 (&to)[NT]) const {
    const int at = kGroup == 128 || c * kInt4Inputs + quarter * 32 < a.inputs ? 4 * quarter : 0;
#pragma unroll
    for (int n = 0; n < NT; ++n) to[n] = load_written(reinterpret_cast<const uint4*>(x[n]) + at);
  }
};

// (Out of line: what it needs registers for is not the main loop's.)
__device__ __noinline__ bool int4_wait(uint32_t bar, uint32_t parity, volatile int* stuck) {
  return mbar_wait(bar, parity, stuck);
}

// After a wait has run out: the warp's last copies, which may still land in its ring, are waited for, with a limit as well, so
// that the block's shared memory is not handed on while they do.  head: how many it has started.
__device__ __noinline__ void int4_drain(uint32_t bars, uint32_t head) {
  volatile int given_up = 0;
  for (uint32_t i = head > kInt4Stages ? head - kInt4Stages : 0; i < head; ++i)
    mbar_wait(bars + 8 * (i % kInt4Stages), i / kInt4Stages & 1u, &given_up);
}

// The warp's part of an item: records [c0, c1), from the ring's stage tail % kInt4Stages on; NT tiles of 8 slots.
// before: the last item's log.
template <typename T, int NT, int kGroup, bool kZeros>
__device__ __forceinline__ void int4_item(const Int4Args& a, Int4Smem<kGroup, kZeros>& sm, const Int4Item& item, int blocks,
                                          int units, int warp, int lane, uint32_t& tail, int& before, Int4Cursor& cursor) {
  const int g = lane >> 2, t = lane & 3, c0 = item.c0, c1 = item.c1;
  const int first = sm.entry_first[item.entry], slots = sm.entry_slots[item.entry];
  Int4Inputs<T, NT, kGroup, kZeros> in(a, sm, first, slots, c0, lane);
  float acc[kInt4Strips][NT][4], part[kInt4Strips][NT][4];
#pragma unroll
  for (int r = 0; r < kInt4Strips; ++r)
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[r][n][i] = 0.0f;
  const uint32_t mask = int4_constant(0x000f000fu << Int4Type<T>::kBit), magic = int4_constant(Int4Type<T>::kMagic);
  uint32_t lo[kInt4Strips], hi[kInt4Strips];         // 16 + zero, twice
#pragma unroll
  for (int r = 0; r < kInt4Strips; ++r) lo[r] = hi[r] = Int4Type<T>::kOffset;
  // x runs kAhead quarters (of 32 inputs) ahead, across the records
  constexpr int kAhead = NT == 1 ? 4 : 2;
  uint4 xq[kAhead][NT];
  if (c0 < c1) {
#pragma unroll
    for (int h = 0; h < kAhead; ++h) in.load(a, c0, h, xq[h]);
  }
  for (int c = c0; c < c1; ++c) {
    const uint32_t from = tail % kInt4Stages;
    const Int4Record<kGroup, kZeros>& st = sm.ring[warp][from];
    const uint32_t bar = smem_u32(&sm.full[warp][from]), parity = tail / kInt4Stages & 1u;
    if (!mbar_try_wait(bar, parity) && !int4_wait(bar, parity, &sm.stuck)) {
      report_status(STK_ERR_DEVICE_TIMEOUT);
      cursor.more = cursor.left = 0;                 // no further copies
    }
    uint4 q[kInt4Strips];
#pragma unroll
    for (int h = 0; h < 4; ++h) {                    // quarters
      constexpr int kPer = kGroup / 32;
      if (h % 2 == 0) {
#pragma unroll
        for (int r = 0; r < kInt4Strips; ++r) q[r] = st.words[r][h / 2][lane];
      }
      if constexpr (kZeros) {
        if (h % kPer == 0) {                         // a new group
          constexpr uint32_t kTwice = 0x00010001u << Int4Type<T>::kBit;
#pragma unroll
          for (int r = 0; r < kInt4Strips; ++r) {
            const uint32_t z = st.zeros[h / kPer][r][g];
            lo[r] = (z & 0xffu) * kTwice + magic;
            hi[r] = (z >> 8) * kTwice + magic;
          }
        }
      }
#pragma unroll
      for (int u = 0; u < 2; ++u) {
#pragma unroll
        for (int r = 0; r < kInt4Strips; ++r) {
          uint32_t w[4];
          int4_decode<T>(h % 2 ? (u ? q[r].w : q[r].z) : (u ? q[r].y : q[r].x), mask, magic, lo[r], hi[r], w);
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            const uint4& v = xq[h % kAhead][n];
            if (h % kPer == 0 && u == 0) {
              const float zero[4] = {0.0f, 0.0f, 0.0f, 0.0f};
              Int4Type<T>::mma_from(part[r][n], w, v.x, v.y, zero);
            } else {
              Int4Type<T>::mma(part[r][n], w, u ? v.z : v.x, u ? v.w : v.y);
            }
          }
        }
      }
      if (h == 4 - kAhead) in.next();
      if (h + kAhead < 4) in.load(a, c, h + kAhead, xq[h % kAhead]);
      else if (c + 1 < c1) in.load(a, c + 1, h + kAhead - 4, xq[h % kAhead]);
      // the end of a group (one beyond the inputs is left out: its x is another quarter's, and infinite if that is)
      if (h % kPer == kPer - 1 && (kGroup == 128 || c * kInt4Inputs + h / kPer * kGroup < a.inputs)) {
#pragma unroll
        for (int r = 0; r < kInt4Strips; ++r) {
          const float2 scale = Int4Type<T>::pair(st.scales[h / kPer][r][g]);
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[r][n][i] = fmaf(i < 2 ? scale.x : scale.y, part[r][n][i], acc[r][n][i]);
        }
      }
    }
    ++tail;
    __syncwarp();                                    // the record is read: the copies run on into its stage
    int4_fetch<kGroup, kZeros>(a, sm, blocks, units, warp, lane, cursor);
  }
  // The sums of a row's warps are added up, in order, each warp taking its share of the values, between barriers of the
  // row's warps (before the first of them they read the last item's sums; where rows get fewer warps, those were a larger
  // group's, and the barrier is the whole CTA's).  Groups of each size have barriers of their own (0 for one group, 1 - 2,
  // 3 - 6, 7 - 14): some warps may be an item ahead, in groups of another size.
  constexpr int kValues = kInt4Strips * NT * 4;
  const int split_log = kInt4MaxLog - item.log, split = 1 << split_log;
  const auto meet = [&] {
    if (split_log == 0) __syncwarp();
    else asm volatile("bar.sync %0, %1;" ::"r"((1 << item.log) - 1 + item.row), "r"(32 * split) : "memory");
  };
  if (item.log > before) __syncthreads();
  else meet();
  before = item.log;
  float (*mine)[32] = sm.joined[warp];
#pragma unroll
  for (int r = 0; r < kInt4Strips; ++r)
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) mine[(r * NT + n) * 4 + i][lane] = acc[r][n][i];
  meet();
  if (item.row < item.n) {
    const int row0 = (item.block + item.row) * kInt4Rows + g;
    const float (*group)[kInt4Strips * kInt4MaxTiles * 4][32] = &sm.joined[item.row << split_log];
    for (int v = warp & (split - 1); v < kValues; v += split) {
      const int i = v % 4, n = v / 4 % NT, r = v / 4 / NT;
      const int which = 8 * n + 2 * t + i % 2, row = row0 + r * 16 + i / 2 * 8;
      if (which >= slots || row >= a.outputs) continue;
      float s = 0.0f;
      for (int p = 0; p < split; ++p) s += group[p][v][lane];
      const int64_t at = static_cast<int64_t>(sm.list[first + which] + a.first_slot) * a.outputs + row;
      s = a.gelu ? int4_gelu(s) : s;
      if (a.out_f32) static_cast<float*>(a.out)[at] = s;
      else static_cast<T*>(a.out)[at] = from_f32<T>(s);
    }
  }
}

template <typename T, int kGroup, bool kZeros>
__global__ void __launch_bounds__(kInt4Threads, 1)
int4_matvec_kernel(const Int4Args a) {
  extern __shared__ __align__(16) unsigned char int4_smem[];
  using Smem = Int4Smem<kGroup, kZeros>;
  Smem& sm = *reinterpret_cast<Smem*>(int4_smem);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int32_t* ids = a.ids + a.first_slot;
  // The kernel after this one, if it was launched so, sets up and starts its copies while this one runs out; it waits for
  // this one's results where it first reads x.
  pdl_launch_dependents();

  // the slots, expert by expert, and the (expert, tile) entries of up to 8 * kInt4MaxTiles of them
  for (int e = threadIdx.x; e < a.experts; e += kInt4Threads) sm.counter[e] = 0;
  if (threadIdx.x == 0) sm.dropped = sm.stuck = 0;
  if (threadIdx.x < kInt4Warps * kInt4Stages) mbar_init(smem_u32(&sm.full[0][0] + threadIdx.x), 1);
  fence_barrier_init();
  __syncthreads();
  for (int s = threadIdx.x; s < a.slots; s += kInt4Threads) {
    const int e = ids[s];
    if (e >= 0 && e < a.experts) atomicAdd(&sm.counter[e], 1);
    else sm.dropped = 1;
  }
  __syncthreads();
  if (warp == 0) {
    constexpr int kTile = 8 * kInt4MaxTiles;
    int slots_before = 0, entries_before = 0;
    for (int e0 = 0; e0 < a.experts; e0 += 32) {
      const int e = e0 + lane;
      const int n = e < a.experts ? sm.counter[e] : 0, tiles = (n + kTile - 1) / kTile;
      int slots_up = n, tiles_up = tiles;
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, slots_up, off), v = __shfl_up_sync(0xffffffffu, tiles_up, off);
        if (lane >= off) {
          slots_up += u;
          tiles_up += v;
        }
      }
      int first = slots_before + slots_up - n, entry = entries_before + tiles_up - tiles;
      if (e < a.experts) sm.counter[e] = first;
      for (int left = n; left > 0; left -= kTile, first += kTile, ++entry) {
        sm.entry_expert[entry] = static_cast<uint16_t>(e);
        sm.entry_first[entry] = static_cast<uint16_t>(first);
        sm.entry_slots[entry] = static_cast<uint16_t>(min(left, kTile));
      }
      slots_before += __shfl_sync(0xffffffffu, slots_up, 31);
      entries_before += __shfl_sync(0xffffffffu, tiles_up, 31);
    }
    if (lane == 0) sm.entries = entries_before;
  }
  __syncthreads();
  if (warp == 0) {                                   // in order: every CTA has to cut the same tiles
    for (int s0 = 0; s0 < a.slots; s0 += 32) {
      const int s = s0 + lane, id = s < a.slots ? ids[s] : -1, e = id < a.experts ? id : -1;
      const unsigned same = __match_any_sync(0xffffffffu, e), before = same & ((1u << lane) - 1);
      const int at = e >= 0 ? sm.counter[e] + __popc(before) : 0;
      __syncwarp();
      if (e >= 0) {
        sm.list[at] = s;
        sm.row[at] = (s + a.first_slot) / a.x_div;
        if (before == 0) sm.counter[e] = at + __popc(same);
      }
      __syncwarp();
    }
  }
  __syncthreads();
  if (sm.dropped) {                                  // zeros for the slots without an expert, dealt out to the CTAs
    for (int s = blockIdx.x; s < a.slots; s += gridDim.x) {
      const int e = ids[s];
      if (e >= 0 && e < a.experts) continue;
      if (e >= a.experts && threadIdx.x == 0) report_status(STK_ERR_BAD_DIMS);
      const int64_t at = static_cast<int64_t>(s + a.first_slot) * a.outputs;
      for (int n = threadIdx.x; n < a.outputs; n += kInt4Threads) {
        if (a.out_f32) static_cast<float*>(a.out)[at + n] = 0.0f;
        else static_cast<T*>(a.out)[at + n] = from_f32<T>(0.0f);
      }
    }
  }

  const int blocks = (a.outputs + kInt4Rows - 1) / kInt4Rows, units = (a.inputs + kInt4Inputs - 1) / kInt4Inputs;
  const int64_t rows = static_cast<int64_t>(sm.entries) * blocks;
  const int64_t row0 = rows * blockIdx.x / gridDim.x, row1 = rows * (blockIdx.x + 1) / gridDim.x;
  if (row0 >= row1) {
    pdl_wait();                                      // (the end of this kernel is the end of the one before it, too)
    return;
  }
  Int4Item item;
  item.left = static_cast<int>(row1 - row0);
  item.entry = static_cast<int>(row0 / blocks);
  item.block = static_cast<int>(row0 - static_cast<int64_t>(item.entry) * blocks);
  item.settle(a, blocks, units, warp);

  Int4Cursor cursor;
  cursor.left = item.left;
  cursor.entry = item.entry;
  cursor.block = item.block;
  cursor.more = 0;
  cursor.head = 0;
  int4_point<kGroup, kZeros>(a, sm, blocks, units, warp, cursor);
#pragma unroll 1
  for (int i = 0; i < kInt4Stages; ++i) int4_fetch<kGroup, kZeros>(a, sm, blocks, units, warp, lane, cursor);
  pdl_wait();
  int before = kInt4MaxLog;
  uint32_t tail = 0;
  do {
    if (sm.entry_slots[item.entry] > 8) int4_item<T, 2, kGroup, kZeros>(a, sm, item, blocks, units, warp, lane, tail, before, cursor);
    else int4_item<T, 1, kGroup, kZeros>(a, sm, item, blocks, units, warp, lane, tail, before, cursor);
  } while (item.next(a, blocks, units, warp));
  if (*static_cast<volatile int*>(&sm.stuck) != 0) int4_drain(smem_u32(&sm.full[warp][0]), cursor.head);
}

// out[t] = sum_j weights[t, j] * y[t * k + j] over the choices that have an expert; y in 32 bits.
template <typename T>
__global__ void __launch_bounds__(256)
int4_combine_kernel(const float* y, const int32_t* __restrict__ ids, const float* __restrict__ weights,
                    T* __restrict__ out, int64_t tokens, int k, int experts, int outputs) {
  pdl_wait();
  const int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  const int64_t t = i / outputs;
  if (t >= tokens) return;
  const int n = static_cast<int>(i - t * outputs);
  float acc = 0.0f;
  for (int j = 0; j < k; ++j) {
    const int64_t s = t * k + j;
    const int e = ids[s];
    if (e >= 0 && e < experts) acc = fmaf(weights[s], load_written(y + s * outputs + n), acc);
  }
  out[i] = from_f32<T>(acc);
}

template <typename T, int kGroup, bool kZeros>
static int int4_launch(Int4Args a, int64_t slots, bool after, cudaStream_t stream) {  // after: programmatic dependent launch
  static std::atomic<int> sms[64] = {};              // (two threads may fill it at once)
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return STK_ERR_LAUNCH;
  const auto kernel = int4_matvec_kernel<T, kGroup, kZeros>;
  constexpr int kBytes = sizeof(Int4Smem<kGroup, kZeros>);
  int n = sms[dev];
  if (n == 0) {
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0 ||
        cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kBytes) != cudaSuccess) {
      cudaGetLastError();
      return STK_ERR_LAUNCH;
    }
    sms[dev] = n;
  }
  const int units = (a.inputs + kInt4Inputs - 1) / kInt4Inputs;
  a.min_log = 0;                                      // no more warps along the inputs than there are records
  while ((kInt4Warps >> a.min_log) > units) ++a.min_log;
  for (int64_t first = 0; first < slots; first += kInt4MaxSlots) {
    a.first_slot = static_cast<int>(first);
    a.slots = static_cast<int>(slots - first < kInt4MaxSlots ? slots - first : kInt4MaxSlots);
    if (after && first == 0)
      launch_dependent(kernel, n, kInt4Threads, kBytes, stream, a);
    else
      kernel<<<static_cast<unsigned>(n), kInt4Threads, kBytes, stream>>>(a);
    if (cudaGetLastError() != cudaSuccess) return STK_ERR_LAUNCH;
  }
  return STK_OK;
}
template <typename T>
static int int4_by_group(const Int4Args& a, int group, int zeros, int64_t slots, bool after, cudaStream_t stream) {
  if (!zeros) {
    if (group == 32) return int4_launch<T, 32, false>(a, slots, after, stream);
    if (group == 64) return int4_launch<T, 64, false>(a, slots, after, stream);
    return int4_launch<T, 128, false>(a, slots, after, stream);
  }
  if (group == 32) return int4_launch<T, 32, true>(a, slots, after, stream);
  if (group == 64) return int4_launch<T, 64, true>(a, slots, after, stream);
  return int4_launch<T, 128, true>(a, slots, after, stream);
}

static int int4_check(const void* records, const void* x, const int32_t* ids, const void* out, int64_t slots, int x_div,
                      int experts, int64_t outputs, int64_t inputs, int group, int dtype) {
  if (slots < 0 || x_div < 1 || experts < 1 || outputs < 1 || inputs < 1) return STK_ERR_BAD_DIMS;
  if ((group != 32 && group != 64 && group != 128) || inputs % group) return STK_ERR_BAD_DIMS;
  if (dtype != STK_F16 && dtype != STK_BF16) return STK_ERR_BAD_DTYPE;
  if (slots > INT32_MAX || outputs > (1 << 20) || inputs / group > kInt4MaxGroups || experts > kInt4MaxExperts)
    return STK_ERR_TOO_LARGE;
  if (slots == 0) return STK_OK;
  if (!records || !x || !ids || !out) return STK_ERR_NULL_POINTER;
  if ((reinterpret_cast<uintptr_t>(records) | reinterpret_cast<uintptr_t>(x)) % 16) return STK_ERR_BAD_LAYOUT;
  return STK_OK;
}
static int int4_matvec(const void* records, const void* x, const int32_t* ids, void* out, int64_t slots, int x_div,
                       int experts, int64_t outputs, int64_t inputs, int group, int zeros, int gelu, int out_f32,
                       int dtype, bool after, cudaStream_t stream) {
  const int rc = int4_check(records, x, ids, out, slots, x_div, experts, outputs, inputs, group, dtype);
  if (rc != STK_OK || slots == 0) return rc;
  const Int4Args a{static_cast<const unsigned char*>(records), x, ids, out, 0, 0, x_div, experts,
                   static_cast<int>(outputs), static_cast<int>(inputs), 0, gelu, out_f32};
  return dtype == STK_BF16 ? int4_by_group<__nv_bfloat16>(a, group, zeros, slots, after, stream)
                           : int4_by_group<__half>(a, group, zeros, slots, after, stream);
}

// Where the hidden activations and the second products lie in the workspace of int4_mlp.  The activations are rounded to the
// inputs' type, as dmoe.expert_mlp's are: they are the B operand of the second product, and as pairs of 16-bit numbers,
// which would keep 32 bits of them nearly whole, they would be twice the columns (2048 x 8192, 16 experts: 61 us with about
// twice the columns where 43 without).  What it costs: the output's error against 64 bits is 1.70e-3 of its norm with and
// without this rounding for 16 tokens of 4096 x 14336 (bf16; the output's own rounding is nearly all of it), and 1.82e-3
// instead of 1.66e-3 for 64 tokens of 2048 x 8192 in groups of 64 with zero points, the largest seen.
static size_t int4_hidden_bytes(int64_t slots, int64_t ffn) { return (static_cast<size_t>(slots) * ffn * 2 + 255) / 256 * 256; }

}  // namespace stk

extern "C" size_t stk_b200_int4_record_bytes(int group, int zeros) {
  if (group != 32 && group != 64 && group != 128) return 0;
  return 2048 + static_cast<size_t>(stk::kInt4Inputs / group) * stk::kInt4Rows * (zeros ? 3 : 2);
}

extern "C" int stk_b200_int4_matvec(const void* records, const void* x, const int32_t* ids, void* out, int64_t slots,
                                    int x_div, int experts, int64_t outputs, int64_t inputs, int group, int zeros,
                                    int gelu, int out_f32, int dtype, void* stream) {
  return stk::int4_matvec(records, x, ids, out, slots, x_div, experts, outputs, inputs, group, zeros, gelu, out_f32, dtype,
                          false, static_cast<cudaStream_t>(stream));
}

extern "C" size_t stk_b200_int4_mlp_workspace_bytes(int64_t slots, int64_t ffn, int64_t outputs) {
  if (slots < 1 || ffn < 1 || outputs < 1) return 0;
  return stk::int4_hidden_bytes(slots, ffn) + static_cast<size_t>(slots) * outputs * sizeof(float);
}

extern "C" int stk_b200_int4_mlp(const void* records1, const void* records2, const void* x, const int32_t* ids,
                                 const float* weights, void* out, int64_t tokens, int top_k, int experts, int64_t hidden,
                                 int64_t ffn, int64_t outputs, int group1, int zeros1, int group2, int zeros2, int dtype,
                                 void* workspace, size_t workspace_bytes, void* stream) {
  if (tokens < 0 || top_k < 1 || outputs < 1 || ffn < 1) return STK_ERR_BAD_DIMS;
  if (tokens == 0) return STK_OK;
  if (!weights || !out) return STK_ERR_NULL_POINTER;
  if (tokens > INT32_MAX / top_k || outputs > (1 << 20) || ffn > (1 << 20)) return STK_ERR_TOO_LARGE;
  const int64_t slots = tokens * top_k, blocks = (tokens * outputs + 255) / 256;
  if (blocks > INT32_MAX) return STK_ERR_TOO_LARGE;
  if (workspace == nullptr || reinterpret_cast<uintptr_t>(workspace) % 16 ||
      workspace_bytes < stk_b200_int4_mlp_workspace_bytes(slots, ffn, outputs))
    return STK_ERR_WORKSPACE;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  // both products' arguments before the first one runs
  int rc = stk::int4_check(records1, x, ids, workspace, slots, top_k, experts, ffn, hidden, group1, dtype);
  if (rc == STK_OK) rc = stk::int4_check(records2, workspace, ids, workspace, slots, 1, experts, outputs, ffn, group2, dtype);
  if (rc != STK_OK) return rc;
  float* y = reinterpret_cast<float*>(static_cast<unsigned char*>(workspace) + stk::int4_hidden_bytes(slots, ffn));
  rc = stk::int4_matvec(records1, x, ids, workspace, slots, top_k, experts, ffn, hidden, group1, zeros1, 1, 0, dtype, false, s);
  if (rc != STK_OK) return rc;
  rc = stk::int4_matvec(records2, workspace, ids, y, slots, 1, experts, outputs, ffn, group2, zeros2, 0, 1, dtype, true, s);
  if (rc != STK_OK) return rc;
  const int grid = static_cast<int>(blocks), width = static_cast<int>(outputs);
  if (dtype == STK_BF16)
    stk::launch_dependent(stk::int4_combine_kernel<__nv_bfloat16>, grid, 256, 0, s, y, ids, weights,
                          static_cast<__nv_bfloat16*>(out), tokens, top_k, experts, width);
  else
    stk::launch_dependent(stk::int4_combine_kernel<__half>, grid, 256, 0, s, y, ids, weights, static_cast<__half*>(out),
                          tokens, top_k, experts, width);
  return cudaGetLastError() == cudaSuccess ? STK_OK : STK_ERR_LAUNCH;
}
