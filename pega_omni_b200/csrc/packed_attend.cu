// Causal attention over packed prompts on the tensor cores (kv8.h).
//
// Bound by the tensor cores, next to it by the exponentials: a block of 128 queries and 128 keys is two products of
// 128 x 128 x D and 16,384 exponentials, which an SM makes 16 a clock. A CTA works on two tiles of 128 queries that share their keys
// - two heads of one group where the group is even, otherwise 256 rows of one head - so a block of K and V is fetched once for
// both, and one tile's products run under the other tile's softmax.
//
// Warps 0-3 and 4-7: the softmax of a tile, a thread a row. Warp 8: copies. Warp 9: matrix instructions. Warps 10 and 11: values
// behind the diagonal. TMEM: per tile 128 columns of scores S, whose first 64 the weights P take over (bf16, the left operand of
// P V), and D columns of O. A tile's instructions are issued as S(0) | P V(0) S(1) | P V(1) S(2) ..., each group when its
// P is there; since they run in order, S(j + 1) having arrived says that P V(j) is done with O, and no other barrier guards it.
//
// Scores, maxima, sums and O are f32. Weights go to bf16 because V does (one type for both operands): 2^-8 at most of a weight,
// which averages out over a row's keys and is what the result itself is rounded by. A row's reference is a maximum that may lag by
// 2^8 behind the true one, so O is rarely rescaled.
//
// A weight of 0 does not silence a NaN or an infinity in V. Where a block has keys that some row must not see (the diagonal, the
// rows behind the sequence's end, which are another sequence's) two warps look through it before it is used: rows behind the end become 0;
// of the others what is not finite becomes 0 and is noted as the column's first row of such a value, and the rows from there on
// take it up at the end.
#include <algorithm>

#include "f32x2.cuh"
#include "gemm.h"
#include "kv8.h"
#include "sm100.cuh"

namespace omni {
namespace {

constexpr int kTile = 128;
constexpr int kThreads = 384;
constexpr int kCopyWarp = 8, kMmaWarp = 9, kGuardWarp = 10;
constexpr float kLag = 8.f;  // powers of two
#ifndef KC
#define KC 0x24
#endif
constexpr int kCubic = KC;
constexpr float kNegInf = -__builtin_huge_valf();
constexpr int kNever = 0x7fffffff;

template <int D>
struct Shape {
  static constexpr int kTileBytes = kTile * D * 2;
  static constexpr int kSlots = D == 128 ? 5 : 8;
  static constexpr int kSmem = (2 + kSlots) * kTileBytes + 1024;  // and what the ring's alignment costs
};

struct Args {
  const int32_t* indptr;
  int n, rows, q_heads, kv_heads;
  int tiles_apart;  // 1: a CTA's tiles are neighbouring heads, 0: neighbouring rows of one head
  int slots;        // places for blocks of rows in the grid
  float scale;      // of scores in powers of two
  bf16* out;
  int64_t ldo;
};

using namespace sm100;

// Thirty-two f32 columns of this thread's lane. The registers hold them only behind tmem_ld_done().
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, float* v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, "
      "%26, %27, %28, %29, %30, %31}, [%32];"
      : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]),
        "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]), "=f"(v[16]),
        "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]), "=f"(v[24]),
        "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31])
      : "r"(taddr)
      : "memory");
}
// The wait for loads issued before; values are given so that no use of them moves in front of it.
template <int N>
__device__ __forceinline__ void tmem_ld_done(float* v) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+f"(v[i])::"memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, "
      "%27, %28, %29, %30, %31, %32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
      "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]),
      "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]),
      "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_st_done() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// D[tmem] (+)= A[tmem] * B[smem]: the left operand's rows in the lanes, two bf16 a column.
__device__ __forceinline__ void mma_bf16_ta(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t"
      "}\n" ::"r"(tmem_d),
      "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// Descriptor of V as the right operand: [keys][64 of D] blocks of 128-byte rows under the 128-byte swizzle, the product's N along the
// rows' bytes. Eight keys are 1024 bytes apart (stride), the blocks of 64 elements kTile * 128 (leading).
__device__ __forceinline__ uint64_t values_desc(uint32_t smem_byte_addr) {
  uint64_t d = 0;
  d |= (uint64_t)((smem_byte_addr & 0x3FFFFu) >> 4);
  d |= (uint64_t)((kTile * 128) >> 4) << 16;
  d |= (uint64_t)(1024 >> 4) << 32;
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)2 << 61;
  return d;
}
constexpr uint32_t kRightTransposed = 1u << 16;  // of an instruction descriptor: B with N contiguous

constexpr int kUsed = 4;

struct Bars {
  uint64_t q_full[2], s_full[2], p_full[2][2], o_full[2], v_full[2], v_clean[2], full[8], used[kUsed], done;
};

template <int D>
__global__ void __launch_bounds__(kThreads, 1) packed_attend_kernel(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap,
                                                                    const __grid_constant__ CUtensorMap vmap, const __grid_constant__ Args a,
                                                                    uint32_t* err) {
  constexpr int SLOTS = Shape<D>::kSlots, BYTES = Shape<D>::kTileBytes;
  extern __shared__ unsigned char raw[];
  __shared__ Bars bars;
  __shared__ uint32_t tmem_slot;
  __shared__ int found;
  __shared__ int odd_row[3][D];  // first row of a NaN, an infinity, a negative infinity in a column of V, where rows must not see all
  __shared__ int any_odd;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t base = (smem_addr(raw) + 1023) & ~1023u;
  const uint32_t q_at = base, ring = base + 2 * BYTES;

  // the block of rows and the heads; the last blocks, which have the most keys, first
  const int units = a.q_heads >> a.tiles_apart;
  const int slot = a.slots - 1 - (int)blockIdx.x / units, unit = blockIdx.x % units;
  const int span = a.tiles_apart ? kTile : 2 * kTile;
  if (tid == 0) found = -1, any_odd = 0;
  __syncthreads();
  for (int i = tid; i < a.n; i += kThreads)
    if (a.indptr[i] / span + i <= slot) atomicMax(&found, i);
  for (int i = tid; i < 3 * D; i += kThreads) (&odd_row[0][0])[i] = kNever;
  __syncthreads();
  const int seq = found;
  if (seq < 0) return;
  const int first = a.indptr[seq], last = a.indptr[seq + 1];
  if (first < 0 || last > a.rows || first > last) {
    if (tid == 0) raise(err, kErrBadIndex);
    return;
  }
  const int len = last - first;
  if ((int64_t)(slot - (first / span + seq)) * span >= len) return;
  const int row0 = (slot - (first / span + seq)) * span;

  const int group = a.q_heads / a.kv_heads;
  int head[2], begin[2], blocks[2];  // of the tiles: head, first row, blocks of keys
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    head[i] = a.tiles_apart ? 2 * unit + i : unit;
    begin[i] = a.tiles_apart ? row0 : row0 + i * kTile;
    blocks[i] = begin[i] < len ? begin[i] / kTile + 1 : 0;
  }
  const int kv_head = head[0] / group, all = max(blocks[0], blocks[1]);
  const int seen_by_all = row0 / kTile;  // blocks of keys before this one are; one block or two are not

  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_addr(&bars.q_full[i]), 1), mbar_init(smem_addr(&bars.s_full[i]), 1);
      mbar_init(smem_addr(&bars.p_full[i][0]), 4), mbar_init(smem_addr(&bars.p_full[i][1]), 4);
      mbar_init(smem_addr(&bars.o_full[i]), 1);
      mbar_init(smem_addr(&bars.v_full[i]), 1), mbar_init(smem_addr(&bars.v_clean[i]), 2);
    }
    for (int i = 0; i < SLOTS; ++i) mbar_init(smem_addr(&bars.full[i]), 1);
    for (int i = 0; i < kUsed; ++i) mbar_init(smem_addr(&bars.used[i]), 1);
    mbar_init(smem_addr(&bars.done), 1);
    mbar_init_fence();
    prefetch_tensormap(&qmap), prefetch_tensormap(&kmap), prefetch_tensormap(&vmap);
  }
  if (warp == kMmaWarp) tmem_alloc(smem_addr(&tmem_slot), 512);
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = tmem_slot;
  const auto bar = [](uint64_t& b) { return smem_addr(&b); };
  // Item 2 j of the ring is block j of K, item 2 j + 1 of V. Blocks of V that are looked through have barriers of their own, since
  // the warps that do it do not follow the ring; they are the last of V.
  const auto guarded = [&](int item) { return (item & 1) && (item >> 1) >= seen_by_all; };
  const auto filling = [&](int item) { return guarded(item) ? bar(bars.v_full[(item >> 1) - seen_by_all]) : bar(bars.full[item % SLOTS]); };
  const auto filled = [&](int item) { return mbar_wait(filling(item), guarded(item) ? 0 : (item / SLOTS) & 1, err); };

  // registers: 2 * 128 * 224 + 128 * 56 = 384 * 168, what the launch has
  if (warp < kCopyWarp) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
    const int i = warp >> 2, quarter = warp & 3;
    const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16);
    const uint32_t s_at = lanes + i * kTile, o_at = lanes + 256 + i * kTile;
    const int begin_i = i ? begin[1] : begin[0], blocks_i = i ? blocks[1] : blocks[0], head_i = i ? head[1] : head[0];
    const int row = begin_i + quarter * 32 + lane;  // of the sequence
    float m = kNegInf, l = 0.f;
    bool ok = true;
    for (int j = 0; j < blocks_i; ++j) {
      ok = mbar_wait(bar(bars.s_full[i]), j & 1, err);
      if (!ok) break;
      tc_fence_after_sync();
      float s[kTile];
#pragma unroll
      for (int c = 0; c < kTile; c += 32) tmem_ld32(s_at + c, s + c);
      tmem_ld_done<kTile>(s);
      if ((j + 1) * kTile > begin_i) {  // the diagonal
        const int limit = row - j * kTile;
#pragma unroll
        for (int c = 0; c < kTile; ++c) s[c] = c <= limit ? s[c] : kNegInf;
      }
      // The weights' first half is made under the reference as it is, with the row's maximum beside it, and once more where that turns
      // out to be too far off. In front of all a maximum comes first.
      const auto largest = [&] {
        float top[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
        for (int c = 4; c + 7 < kTile; c += 8)
#pragma unroll
          for (int t = 0; t < 4; ++t) top[t] = max3_nan(top[t], s[c + t], s[c + 4 + t]);
#pragma unroll
        for (int t = 0; t < 4; ++t) top[t] = max3_nan(top[t], s[kTile - 4 + t], s[kTile - 4 + t]);
        return max3_nan(top[0], top[1], max3_nan(top[2], top[3], top[3])) * a.scale;
      };
      float2 sum[2];
      uint32_t p[32];
      const auto weights = [&](int half) {
        const float2 scale = both(a.scale), minus_ref = both(m == kNegInf ? 0.f : -m);
#pragma unroll
        for (int e = 0; e < 32; ++e) {
          const int c = half * 64 + 2 * e;
          const float2 x = fma2(make_float2(s[c], s[c + 1]), scale, minus_ref);
          const float2 w = kCubic >> (e & 7) & 1 ? exp2_cubic(x) : make_float2(exp2_of(x.x), exp2_of(x.y));
          sum[e & 1] = add2(sum[e & 1], w);
          const __nv_bfloat162 h = __floats2bfloat162_rn(w.x, w.y);
          p[e] = *reinterpret_cast<const uint32_t*>(&h);
        }
      };
      const auto give = [&](int half) {
        tmem_st32(s_at + half * 32, p);
        tmem_st_done();
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(bars.p_full[i][half]));
      };
      if (j == 0) m = largest();
      sum[0] = sum[1] = both(0.f);
      weights(0);
      const float now = largest();
      if (__any_sync(0xffffffffu, now > m + kLag)) {
        const float next = now > m + kLag ? now : m;
        const float f = m == next ? 1.f : m == kNegInf ? 0.f : exp2_of(m - next);
        m = next, l *= f;
#pragma unroll
        for (int c = 0; c < D; c += 32) {
          float o[32];
          tmem_ld32(o_at + c, o);
          tmem_ld_done<32>(o);
          uint32_t r[32];
#pragma unroll
          for (int e = 0; e < 32; ++e) r[e] = __float_as_uint(o[e] * f);
          tmem_st32(o_at + c, r);
        }
        sum[0] = sum[1] = both(0.f);
        weights(0);
      }
      give(0);
      weights(1);
      give(1);
      sum[0] = add2(sum[0], sum[1]);
      // a score that is no number, or infinite: neither is the sum
      l += sum[0].x + sum[0].y + (now == kNegInf ? 0.f : now - now);
    }
    if (ok && blocks_i) ok = mbar_wait(bar(bars.o_full[i]), 0, err);
    for (int j = seen_by_all; j < all && ok && blocks_i; ++j) ok = mbar_wait(bar(bars.v_clean[j - seen_by_all]), 0, err);
    if (ok && blocks_i) {
      tc_fence_after_sync();
      const float f = 1.f / l;
      const bool odd = *reinterpret_cast<volatile int*>(&any_odd);
      bf16* const dst = a.out + (int64_t)(first + row) * a.ldo + (int64_t)head_i * D;
#pragma unroll
      for (int c = 0; c < D; c += 32) {
        float o[32];
        tmem_ld32(o_at + c, o);
        tmem_ld_done<32>(o);
#pragma unroll
        for (int e = 0; e < 32; ++e) o[e] *= f;
        if (odd) {
          for (int e = 0; e < 32; ++e) {
            const bool nan = row >= odd_row[0][c + e], pos = row >= odd_row[1][c + e], neg = row >= odd_row[2][c + e];
            if (pos) o[e] += __builtin_huge_valf();
            if (neg) o[e] -= __builtin_huge_valf();
            if (nan) o[e] = __int_as_float(0x7fffffff);
          }
        }
        if (row < len) {
#pragma unroll
          for (int e = 0; e < 32; e += 8) st8(dst + c + e, o + e);
        }
      }
    }
  } else {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
  if (warp == kCopyWarp) {
    if (elect_one()) {
      int issued = 0;
      bool ok = true;
      for (int i = 0; i < 2; ++i) {
        if (!blocks[i]) continue;
        mbar_expect_tx(bar(bars.q_full[i]), BYTES);
        tma_load_3d(q_at + i * BYTES, &qmap, bar(bars.q_full[i]), 0, first + begin[i], head[i] * (D / 64), kEvictFirst);
      }
      for (int item = 0; item < 2 * all; ++item) {
        if (item >= SLOTS) {  // what the slot held was used up in this turn
          const int turn = (item - SLOTS - 1) / 2;
          ok = mbar_wait(bar(bars.used[turn % kUsed]), (turn / kUsed) & 1, err);
          if (!ok) break;
        }
        const int s = item % SLOTS;
        const uint32_t full = filling(item);
        mbar_expect_tx(full, BYTES);
        tma_load_3d(ring + s * BYTES, item & 1 ? &vmap : &kmap, full, 0, first + (item >> 1) * kTile, kv_head * (D / 64), kEvictLast);
        ++issued;
      }
      if (!ok) {
        for (int item = max(0, issued - SLOTS); item < issued; ++item) filled(item);
        for (int i = 0; i < 2; ++i)
          if (blocks[i]) mbar_wait(bar(bars.q_full[i]), 0, err);
      }
    }
  } else if (warp == kMmaWarp) {
    // one thread for both tiles, in turns: it keeps them apart, so that one's products run under the other's exponentials
    if (elect_one()) {
      constexpr uint32_t kScores = idesc_bf16_f32(kTile, kTile), kSums = idesc_bf16_f32(kTile, D) | kRightTransposed;
      const auto scores = [&](int i, int j) {  // S of tile i against keys j
        const uint32_t q = q_at + i * BYTES, k = ring + (2 * j % SLOTS) * BYTES;
#pragma unroll
        for (int x = 0; x < D / 16; ++x) {
          const uint32_t at = (x >> 2) * (kTile * 128) + (x & 3) * 32;
          mma_bf16(tmem + i * kTile, kmajor_sw128_desc(q + at), kmajor_sw128_desc(k + at), kScores, x > 0);
        }
        mma_commit(bar(bars.s_full[i]));
      };
      // Turn j: P V(j) and S(j + 1) of both tiles. What it needs of the ring was waited for in the turn before, between the tiles.
      const auto ready = [&](int j) {
        const bool v = j < seen_by_all ? filled(2 * j + 1) : mbar_wait(bar(bars.v_clean[j - seen_by_all]), 0, err);
        return v && (j + 1 >= all || filled(2 * j + 2));
      };
      bool ok = filled(0);
      for (int i = 0; i < 2 && ok; ++i) {
        if (!blocks[i]) continue;
        ok = mbar_wait(bar(bars.q_full[i]), 0, err);
        if (!ok) break;
        tc_fence_after_sync();
        scores(i, 0);
      }
      ok = ok && ready(0);
      uint32_t v = ring + BYTES;
      for (int j = 0; j < all && ok; ++j) {
        for (int i = 0; i < 2 && ok; ++i) {
          if (j < blocks[i]) {
            for (int half = 0; half < 2 && ok; ++half) {  // of the block's keys, whose weights come in turn
              ok = mbar_wait(bar(bars.p_full[i][half]), j & 1, err);
              if (!ok) break;
              tc_fence_after_sync();
#pragma unroll
              for (int x = 0; x < kTile / 32; ++x) {
                const int k = half * (kTile / 32) + x;
                mma_bf16_ta(tmem + 256 + i * kTile, tmem + i * kTile + k * 8, values_desc(v + k * 2048), kSums, j > 0 || k > 0);
              }
            }
            if (!ok) break;
            if (j + 1 < blocks[i]) scores(i, j + 1);
            else mma_commit(bar(bars.o_full[i]));
          }
          if (i == 0 && j + 1 < all) ok = ready(j + 1);
        }
        if (!ok) break;
        if (2 * j + SLOTS < 2 * all) mma_commit(bar(bars.used[j % kUsed]));  // items wait for it
        v = v + 2 * BYTES >= ring + SLOTS * BYTES ? v + 2 * BYTES - SLOTS * BYTES : v + 2 * BYTES;
      }
      if (!ok) {  // what is under way uses shared memory and TMEM
        mma_commit(bar(bars.done));
        mbar_wait(bar(bars.done), 0, err);
      }
    }
  } else {
    const int t = tid - kGuardWarp * 32;
    for (int j = seen_by_all; j < all; ++j) {
      const int item = 2 * j + 1;
      if (!filled(item)) break;
      unsigned char* const v = raw + (ring - smem_addr(raw)) + (item % SLOTS) * BYTES;
      const int keys = len - j * kTile;  // rows of the sequence in the block, or more
      for (int i = t; i < BYTES / 16; i += 64) {
        uint4* const at = reinterpret_cast<uint4*>(v) + i;
        const int row = (i >> 3) & (kTile - 1);
        if (row >= keys) {
          *at = make_uint4(0, 0, 0, 0);
          continue;
        }
        const uint4 u = *at;
        const uint32_t mark = 0x7f807f80u, one = 0x00800080u, top = 0x80008000u;  // an exponent of all ones carries into the top bit
        if ((((u.x & mark) + one) | ((u.y & mark) + one) | ((u.z & mark) + one) | ((u.w & mark) + one)) & top) {
          const int col = (i / (kTile * 8)) * 64 + (((i & 7) ^ (row & 7)) << 3);
          uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const uint32_t h = (w[e >> 1] >> (16 * (e & 1))) & 0xffffu;
            if ((h & 0x7f80u) == 0x7f80u) {
              atomicMin(&odd_row[h & 0x7fu ? 0 : h >> 15 ? 2 : 1][col + e], j * kTile + row);
              w[e >> 1] &= e & 1 ? 0xffffu : 0xffff0000u;
              any_odd = 1;
            }
          }
          *at = make_uint4(w[0], w[1], w[2], w[3]);
        }
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(bars.v_clean[j - seen_by_all]));
    }
  }
  }
  tc_fence_before_sync();
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after_sync();
    tmem_dealloc(tmem, 512);
  }
}

template <int D>
cudaError_t go(const PackedAttend& p, const CUtensorMap* maps, const Args& a, uint32_t* err, cudaStream_t s) {
  const cudaError_t e = allow_large<packed_attend_kernel<D>>(Shape<D>::kSmem);
  if (e != cudaSuccess) return e;
  const unsigned units = p.q_heads >> a.tiles_apart;
  packed_attend_kernel<D><<<a.slots * units, kThreads, Shape<D>::kSmem, s>>>(maps[0], maps[1], maps[2], a, err);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_packed_attend(const PackedAttend& p, uint32_t* err, cudaStream_t s) {
  const int group = p.q_heads / p.kv_heads, D = p.head_dim;
  Args a;
  a.indptr = p.indptr, a.n = p.n, a.rows = p.rows, a.q_heads = p.q_heads, a.kv_heads = p.kv_heads;
  a.tiles_apart = group % 2 == 0;
  a.slots = p.rows / (a.tiles_apart ? kTile : 2 * kTile) + p.n;
  a.scale = p.scale * 1.44269504088896340736f;
  a.out = p.out, a.ldo = p.ldo;
  CUtensorMap maps[3];
  const bf16* at[3] = {p.q, p.k, p.v};
  const int64_t ld[3] = {p.ldq, p.ldk, p.ldv};
  const uint32_t box[3] = {64, kTile, (uint32_t)(D / 64)};
  for (int i = 0; i < 3; ++i) {
    const uint64_t dims[3] = {64, (uint64_t)p.rows, (uint64_t)(i ? p.kv_heads : p.q_heads) * (D / 64)};
    const uint64_t strides[2] = {(uint64_t)ld[i] * 2, 128};
    if (tc_encode_bf16(&maps[i], at[i], 3, dims, strides, box) != 0) return cudaErrorInvalidValue;
  }
  if (D == 128) return go<128>(p, maps, a, err, s);
  if (D == 64) return go<64>(p, maps, a, err, s);
  return cudaErrorInvalidValue;
}

}  // namespace omni
