// Causal attention over packed prompts on the tensor cores (kv8.h).
//
// Bound by the tensor cores and the exponentials alike: a block of 128 queries and 128 keys is two products of 128 x 128 x D and
// 16,384 exponentials, which an SM makes 16 a clock. TMEM holds a tile's 128 columns of scores S, whose first 64 the weights P take
// over (bf16, the left operand of P V), and D columns of O. A tile's matrix instructions run in their order - S(0) | P V(0) S(1) |
// P V(1) S(2) .., each group when its P is there - so S(j + 1) having arrived says that P V(j) is done with O, and no other barrier guards it.
// Softmax has a thread a row of a tile; one warp copies, one issues matrix instructions, two look through values (below).
//
// CTAs stay and take items (a tile's or two tiles' rows of a sequence) in turns, the longest first and back and forth: an item's Q and K
// are fetched and its first scores made under the end of the one before. A tile is 128 rows of one head, or as many fewer of each of 2, 4,
// 8 or 16 heads of a group as halve its number: less of a sequence's last tile is empty then (43 sequences of 6 to 12 tokens, 16 heads of
// 128 over one: 8.3 us instead of 16.2, 64 of 1 to 120, 32 over 8: 28 instead of 39; 16 of 512, 16 over 8: 39 instead of 38).
//
// Two kernels, chosen below; both have two tiles on an SM, one's products under the other's exponentials.
//  - paired_kernel: one CTA, whose tiles are other heads of the same group and rows, so that a block of K and V is fetched once for both.
//  - single_kernel: two CTAs of a tile each, which read K and V twice as often, but are out of step at an item's end, and smaller.
// Of a turn of paired_kernel (a block of keys for both tiles, 3,400 clocks) the tensor cores have work for 2,050, the exponentials' pipe as
// much; the rest is the way from the last weights to the next scores, and an item's end. The clock is what power leaves at this rate: 8,192
// tokens of 32 heads take 470 to 515 us from a graph, 520 to 540 call after call. A cubic for every eighth or fourth exponential, two threads a row, an issuing
// warp a tile (which lets both tiles fall into step), weights in unequal parts, a first reference from part of a row and 32-byte stores of results made it no faster.
//
// Scores, maxima, sums and O are f32. Weights go to bf16 because V does (one type for both operands): 2^-8 at most of a weight,
// which averages out over a row's keys and is what the result itself is rounded by. A row's reference is a maximum that may lag by
// 2^8 behind the true one, so O is rarely rescaled, and the weights need not wait for the maximum.
//
// A weight of 0 does not silence a NaN or an infinity in V. Where a block has keys that some row must not see (the diagonal, the
// rows behind the sequence's end, which are another sequence's) two warps look through it before it is used: rows behind the end become 0;
// of the others what is not finite becomes 0 and is noted as the column's first row of such a value, and the rows from there on
// take it up at the end.
#include <algorithm>

#include "f32x2.cuh"
#include "gemm.h"
#include "kv8.h"
#include "pdl.cuh"
#include "sm100.cuh"

namespace omni {
namespace {

constexpr int kTile = 128;
constexpr float kLag = 8.f;  // powers of two
constexpr float kFar = 268435456.f;  // 2^28 powers of two: references beyond are off by more than sixteen when they are rounded
constexpr float kNegInf = -__builtin_huge_valf();

struct Args {
  const int32_t* indptr;
  int n, rows, q_heads, kv_heads;
  float scale;  // of scores in powers of two
  bf16* out;
  int64_t ldo;
  int span;   // log2 of a tile's rows of one head, of which it holds 128 >> span
  int share;  // log2 of an item's heads
};

using namespace sm100;

template <int D>
constexpr int kTileBytes = kTile * D * 2;

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
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
      "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
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


// ---- what the kernels share ---------------------------------------------------------------------------------------------

// S of a tile: Q and K as they lie in shared memory.
template <int D>
__device__ __forceinline__ void issue_scores(uint32_t s, uint32_t q, uint32_t k) {
  constexpr uint32_t kShape = idesc_bf16_f32(kTile, kTile);
#pragma unroll
  for (int x = 0; x < D / 16; ++x) {
    const uint32_t at = (x >> 2) * (kTile * 128) + (x & 3) * 32;
    mma_bf16(s, kmajor_sw128_desc(q + at), kmajor_sw128_desc(k + at), kShape, x > 0);
  }
}
// O (+)= P V for half of a block's keys.
template <int D>
__device__ __forceinline__ void issue_sums(uint32_t o, uint32_t p, uint32_t v, int half, bool first) {
  constexpr uint32_t kShape = idesc_bf16_f32(kTile, D) | kRightTransposed;
#pragma unroll
  for (int x = 0; x < kTile / 32; ++x) {
    const int k = half * (kTile / 32) + x;
    mma_bf16_ta(o, p + k * 8, values_desc(v + k * 2048), kShape, !first || k > 0);
  }
}

// A row's reference, a score as the product gives it, and the sum of its weights.
struct Row {
  float m = kNegInf, l = 0.f;
};
// Weights of a block, whose scores have arrived: give(0) and give(1) when half of them are in TMEM. `first`: there is no O yet;
// `seen`: the last key that the row sees.
template <int D, typename Give>
__device__ __forceinline__ void make_weights(Row& row, uint32_t s_at, uint32_t o_at, float scale_to_2, bool first, bool diagonal, int seen, Give&& give) {
  float s[kTile];
#pragma unroll
  for (int c = 0; c < kTile; c += 32) tmem_ld32(s_at + c, s + c);
  tmem_ld_done<kTile>(s);
  if (diagonal) {
#pragma unroll
    for (int c = 1; c < kTile; ++c) s[c] = c <= seen ? s[c] : kNegInf;
  }
  const auto largest = [&] {
    float top[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
    for (int c = 4; c + 7 < kTile; c += 8)
#pragma unroll
      for (int t = 0; t < 4; ++t) top[t] = max3_nan(top[t], s[c + t], s[c + 4 + t]);
#pragma unroll
    for (int t = 0; t < 4; ++t) top[t] = max3_nan(top[t], s[kTile - 4 + t], s[kTile - 4 + t]);
    return max3_nan(top[0], top[1], max3_nan(top[2], top[3], top[3]));
  };
  float2 sum[2];
  // A weight is 2^((s - off) * scale + minus_ref): near 0 the reference goes into the sum, rounded, which is a factor in common; far from
  // it, where that factor would not fit, it is taken off the scores.
  float off, minus_ref;
  const auto refer = [&] {
    const float ref = row.m == kNegInf ? 0.f : row.m * scale_to_2;
    off = fabsf(ref) > kFar ? row.m : 0.f, minus_ref = fabsf(ref) > kFar ? 0.f : -ref;
  };
  const auto weights = [&](int q) {  // of a quarter of the keys
    const float2 scale = both(scale_to_2), minus = both(minus_ref);
    uint32_t p[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const int c = q * 32 + 2 * e;
      const float2 x = fma2(make_float2(s[c], s[c + 1]), scale, minus), w = make_float2(exp2_of(x.x), exp2_of(x.y));
      sum[e & 1] = add2(sum[e & 1], w);
      const __nv_bfloat162 h = __floats2bfloat162_rn(w.x, w.y);
      p[e] = *reinterpret_cast<const uint32_t*>(&h);
    }
    tmem_st16(s_at + q * 16, p);
  };
  const auto done = [&](int half) {
    tmem_st_done();
    tc_fence_before_sync();
    __syncwarp();
    give(half);
  };
  const auto raise_to = [&](float next) {
    const float was = row.m, was_off = off, was_minus = minus_ref;
    row.m = next;
    refer();
    const float f = was == next ? 1.f : was == kNegInf ? 0.f : exp2_of(fmaf(was_off - off, scale_to_2, minus_ref - was_minus));
    row.l *= f;
#pragma unroll 1
    for (int c = 0; c < D; c += 16) {
      float o[16];
      tmem_ld16(o_at + c, o);
      uint32_t r[16];
#pragma unroll
      for (int e = 0; e < 16; ++e) r[e] = __float_as_uint(o[e] * f);
      tmem_st16(o_at + c, r);
    }
  };
  // The first half is made under the reference as it is, with the row's maximum beside it, and once more where that turns out to be
  // too far off. In front of all a maximum comes first, and where a row's reference is far from 0.
  float now;
  if (first) row.m = now = largest();
  refer();
  bool far = __any_sync(0xffffffffu, off != 0.f), last = first;
#pragma unroll 1
  for (;;) {
    if (far) {
      if (!first) now = largest(), raise_to(fmaxf(row.m, now));
#pragma unroll
      for (int c = 0; c < kTile; ++c) s[c] -= off;
      last = true;
    }
    sum[0] = sum[1] = both(0.f);
    weights(0), weights(1);
    if (last) break;
    now = largest();
    const bool over = (now - row.m) * scale_to_2 > kLag;
    if (!__any_sync(0xffffffffu, over)) break;
    raise_to(over ? now : row.m);
    far = __any_sync(0xffffffffu, off != 0.f);
  }
  done(0);
  weights(2), weights(3);
  done(1);
  sum[0] = add2(sum[0], sum[1]);
  // a score that is no number, or infinite: neither is the sum
  row.l += sum[0].x + sum[0].y + (now == kNegInf ? 0.f : now - now);
}

// The warp's rows of O over the sums of their weights. place(r): where row r goes, null: nowhere; sees(kind, column): the row takes up
// a NaN (0), an infinity (1), a negative infinity (2), asked where `odd`. Through 2 KB of shared memory, 16 bytes of a row in an
// order of its own: the warp then writes 64 bytes of eight rows at a time, not 16 of 32.
template <int D, typename Sees, typename Place>
__device__ __forceinline__ void write_rows(uint32_t o_at, float l, bool odd, Sees&& sees, unsigned char* stage, Place&& place, int lane) {
  const float f = 1.f / l;
  bf16* dst[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) dst[e] = place(e * 8 + (lane >> 2));
#pragma unroll 1
  for (int c = 0; c < D; c += 32) {
    float o[32];
    tmem_ld32(o_at + c, o);
    tmem_ld_done<32>(o);
#pragma unroll
    for (int e = 0; e < 32; ++e) o[e] *= f;
    if (odd) {
#pragma unroll 1
      for (int e = 0; e < 32; ++e) {
        float add = 0.f;
        if (sees(1, c + e)) add += __builtin_huge_valf();
        if (sees(2, c + e)) add -= __builtin_huge_valf();
        if (sees(0, c + e)) add = __int_as_float(0x7fffffff);
#pragma unroll
        for (int k = 0; k < 32; ++k) o[k] += k == e ? add : 0.f;
      }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) *reinterpret_cast<uint4*>(stage + lane * 64 + ((e ^ (lane >> 1 & 3)) << 4)) = pack8v(o + 8 * e);
    __syncwarp();
    uint4 u[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int r = e * 8 + (lane >> 2);
      u[e] = *reinterpret_cast<const uint4*>(stage + r * 64 + (((lane & 3) ^ (r >> 1 & 3)) << 4));
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (dst[e]) *reinterpret_cast<uint4*>(dst[e] + c + (lane & 3) * 8) = u[e];
    __syncwarp();
  }
}

// Looks through a block of V, thread t of 64: rows from `keys` on become 0, what is not finite in front of them too, behind
// note(kind, column, row of the block).
template <int D, typename Note>
__device__ __forceinline__ void look_through(unsigned char* v, int keys, int t, Note&& note) {
  const int own = min(keys, kTile) * 8;  // pieces of 16 bytes of 64 columns
  __nv_bfloat162 most = __floats2bfloat162_rn(0.f, 0.f);
  for (int half = 0; half < D / 64; ++half) {
    uint4* const at = reinterpret_cast<uint4*>(v) + half * (kTile * 8);
#pragma unroll 4
    for (int i = t; i < own; i += 64) {
      const uint4 u = at[i];
      const __nv_bfloat162* const w = reinterpret_cast<const __nv_bfloat162*>(&u);
#pragma unroll
      for (int e = 0; e < 4; ++e) most = __hmax2_nan(most, __habs2(w[e]));
    }
    for (int i = own + t; i < kTile * 8; i += 64) at[i] = make_uint4(0, 0, 0, 0);
  }
  // infinities and NaN are among the largest magnitudes: once more, piece by piece
  const float low = __low2float(most), high = __high2float(most);
  if (!(low < __builtin_huge_valf() && high < __builtin_huge_valf())) {
#pragma unroll 1
    for (int i = t; i < D / 64 * own; i += 64) {
      const int half = i / own, at = i - half * own, r = at >> 3, col = half * 64 + (((at & 7) ^ (r & 7)) << 3);
      bf16* const w = reinterpret_cast<bf16*>(v + half * (kTile * 128) + at * 16);
#pragma unroll 1
      for (int e = 0; e < 8; ++e) {
        const float x = __bfloat162float(w[e]);
        if (fabsf(x) < __builtin_huge_valf()) continue;
        note(x != x ? 0 : x > 0.f ? 1 : 2, col + e, r);
        w[e] = __float2bfloat16(0.f);
      }
    }
  }
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  __syncwarp();
}

// ---- items -----------------------------------------------------------------------------------------------------------------

struct Item {
  int first, len;  // of the sequence: first row, rows
  int row0, head;  // of the item: its first row, its first head; head < 0: there is none any more
};

// The items in their order, for one warp: by blocks of keys, the most first, then by sequence, row and heads.
struct Order {
  const Args& a;
  int lane;
  int units = a.q_heads >> a.share;  // items of the same rows
  int level = -1;               // blocks of the items that come now but one
  int at_level = 0, longer = 0; // tiles of them; sequences that have any
  int until = 0;                // no sequence ends between this level and the one last counted
  int base = 0;                 // items in front of them
  int from_i = 0, from_k = 0;   // sequences that need not be looked at again, and their tiles
  int from = 0, to = 0;         // rows of this lane's sequence of the first thirty-two, which are all that most calls have

  __device__ __forceinline__ int rows(int i0) const {  // of sequence i0 + lane
    const int i = i0 + lane;
    int x = from, y = to;
    if (i0 > 0 && i < a.n) x = __ldcg(a.indptr + i), y = __ldcg(a.indptr + i + 1);
    return i >= a.n || x < 0 || y > a.rows || x > y ? 0 : y - x;
  }
  __device__ __forceinline__ static int blocks(int rows) { return (rows + kTile - 1) / kTile; }
  __device__ __forceinline__ int tiles(int rows) const {  // of this level, of a sequence with so many rows
    const int left = min(max(rows - level * kTile, 0), kTile);
    return (left + (1 << a.span) - 1) >> a.span;
  }
  __device__ __forceinline__ void count() {
    int sum = 0, next = 0;  // next: blocks of the longest sequence that has no such item
    longer = 0;
    for (int i0 = 0; i0 < a.n; i0 += 32) {
      const int its = rows(i0);
      sum += tiles(its);
      longer += __popc(__ballot_sync(0xffffffffu, blocks(its) > level));
      if (blocks(its) <= level) next = max(next, blocks(its));
    }
    at_level = (int)__reduce_add_sync(0xffffffffu, (unsigned)sum);
    until = (int)__reduce_max_sync(0xffffffffu, (unsigned)next);
  }
  __device__ __forceinline__ void begin(uint32_t* err) {
    constexpr int kMany = 1 << 25;  // more than there can be
    if (lane < a.n) from = __ldcg(a.indptr + lane), to = __ldcg(a.indptr + lane + 1);
    int most = 0, sum = 0;
    for (int i0 = 0; i0 < a.n; i0 += 32) {
      int x = from, y = to;
      if (i0 > 0 && i0 + lane < a.n) x = __ldcg(a.indptr + i0 + lane), y = __ldcg(a.indptr + i0 + lane + 1);
      if (i0 + lane >= a.n) break;
      const bool wrong = x < 0 || y > a.rows || x > y;
      if (wrong && blockIdx.x == 0) raise(err, kErrBadIndex);
      const int its = wrong ? 0 : blocks(y - x);
      most = max(most, its), sum = min(sum + its, kMany);
    }
    __syncwarp();
    level = (int)__reduce_max_sync(0xffffffffu, (unsigned)most) - 1;
    // sequences that overlap, between which an end lies in front of a beginning: an error by now, and no end of work
    if ((int)__reduce_add_sync(0xffffffffu, (unsigned)sum) > a.rows / kTile + a.n) level = -1;
    if (level >= 0) count();
  }
  // Item t, not in front of the one asked for before.
  __device__ __forceinline__ Item item(int t) {
    while (level >= 0 && t - base >= at_level * units) {
      base += at_level * units;
      --level;
      from_i = from_k = 0;
      if (level < until && level >= 0) count();
      else at_level = longer << (7 - a.span);  // all of the sequences go on beyond this level
    }
    const int k = (t - base) / units, unit = t - base - k * units;
    for (; level >= 0 && from_i < a.n; from_i += 32) {  // the sequence that has the k-th tile
      const int its = tiles(rows(from_i));
      int incl = its;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += up;
      }
      const uint32_t has = __ballot_sync(0xffffffffu, from_k + incl > k);
      if (has) {
        const int l = __ffs(has) - 1, tile = k - from_k - __shfl_sync(0xffffffffu, incl - its, l);
        int x = __shfl_sync(0xffffffffu, from, l), y = __shfl_sync(0xffffffffu, to, l);
        if (from_i > 0) x = __ldcg(a.indptr + from_i + l), y = __ldcg(a.indptr + from_i + l + 1);
        return Item{x, y - x, level * kTile + (tile << a.span), unit << a.share};
      }
      from_k += __shfl_sync(0xffffffffu, incl, 31);
    }
    return Item{0, 0, 0, -1};
  }
};

// ---- one tile at a time ---------------------------------------------------------------------------------------------------

namespace single {

constexpr int kThreads = 256, kPerSm = 2;
constexpr int kItemWarp = 4, kMmaWarp = 5, kGuardWarp = 6;
constexpr uint32_t kColumns = 256;  // of TMEM: S, then O
template <int D>
constexpr int kSmem = 3 * kTileBytes<D> + 1024;  // Q, K and V, and what their alignment costs

// One of each of what an item or a block needs in turn: a barrier's phase is the item's or the block's number.
struct Bars {
  uint64_t item_full[2], item_empty[2];
  uint64_t q_full, o_full, last_full, last_clean;  // by items; the last block of V has barriers of its own
  uint64_t k_full, s_full, p_full[2], v_used;      // by blocks
  uint64_t v_full;                                 // by blocks that are not an item's last
  uint64_t done;
};

template <int D>
__global__ void __launch_bounds__(kThreads, kPerSm)
    single_kernel(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                         const __grid_constant__ Args a, uint32_t* err) {
  constexpr int BYTES = kTileBytes<D>;
  extern __shared__ unsigned char raw[];
  __shared__ Bars bars;
  __shared__ Item items[2];
  __shared__ uint32_t tmem_slot;
  // what is not finite in the last block of V, by items: the item's number + 1, and for each column the item's number * 256 + 127 - the
  // first such row of the block, of NaN, infinities and negative infinities
  __shared__ int any_odd[2], odd_row[2][3][D];
  __shared__ __align__(16) unsigned char stages[4][32 * 64];  // 32 columns of a warp's rows on their way out
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t base = (smem_addr(raw) + 1023) & ~1023u;
  const uint32_t q_at = base, k_at = base + BYTES, v_at = base + 2 * BYTES;
  const auto bar = [](uint64_t& b) { return smem_addr(&b); };
  const auto wait = [&](uint64_t& b, int phase) { return mbar_wait(smem_addr(&b), phase & 1, err); };

  if (warp == kMmaWarp) {
    grid_wait();  // columns only then: the kernel in front may want them for CTAs that have not begun
    tmem_alloc(smem_addr(&tmem_slot), kColumns);
  }
  if (tid == kItemWarp * 32) {
    prefetch_tensormap(&qmap), prefetch_tensormap(&kmap), prefetch_tensormap(&vmap);
    for (int i = 0; i < 2; ++i) mbar_init(bar(bars.item_full[i]), 1), mbar_init(bar(bars.item_empty[i]), 7), mbar_init(bar(bars.p_full[i]), 4);
    mbar_init(bar(bars.q_full), 1), mbar_init(bar(bars.o_full), 1), mbar_init(bar(bars.last_full), 1), mbar_init(bar(bars.last_clean), 2);
    mbar_init(bar(bars.k_full), 1), mbar_init(bar(bars.s_full), 1), mbar_init(bar(bars.v_used), 1), mbar_init(bar(bars.v_full), 1);
    mbar_init(bar(bars.done), 1);
    mbar_init_fence();
  }
  const auto fetch = [&](const CUtensorMap* map, uint32_t to, uint64_t& full, int at_row, int at_head, uint64_t hint) {
    mbar_expect_tx(bar(full), BYTES);
    tma_load_3d(to, map, bar(full), 0, at_row, at_head * (D / 64), hint);
  };
  const auto fetch_q = [&](const Item& it) {  // rows of its heads, one head behind the other
    mbar_expect_tx(bar(bars.q_full), BYTES);
#pragma unroll
    for (int c = 0; c < D / 64; ++c) tma_load_4d(q_at + c * (kTile * 128), &qmap, bar(bars.q_full), 0, it.first + it.row0, it.head, c, kEvictFirst);
  };
  const int group = a.q_heads / a.kv_heads;
  // the first item, and the first of its copies, while the CTA sets itself up
  Order order{a, lane};
  Item it{0, 0, 0, -1};  // of the item warp
  if (warp == kItemWarp) {
    grid_wait();
    order.begin(err);
    it = order.item(blockIdx.x);
    if (lane == 0) {
      items[0] = it;
      mbar_arrive(bar(bars.item_full[0]));
      if (it.head >= 0) {
        fence_async_global();
        fetch_q(it);
        fetch(&kmap, k_at, bars.k_full, it.first, it.head / group, kEvictLast);
        fetch(&vmap, v_at, it.row0 < kTile ? bars.last_full : bars.v_full, it.first, it.head / group, kEvictLast);
      }
    }
    __syncwarp();
  }
  for (int i = tid; i < 2 * 3 * D; i += kThreads) (&odd_row[0][0][0])[i] = -1;
  if (tid < 2) any_odd[tid] = 0;
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = tmem_slot;
  grid_trigger();

  const auto item_there = [&](int n) { return wait(bars.item_full[n & 1], n >> 1) && items[n & 1].head >= 0; };
  const auto leave_item = [&](int n) { mbar_arrive(bar(bars.item_empty[n & 1])); };

  // registers: 128 * 184 + 128 * 72 = 256 * 128, what the launch has
  if (warp < kItemWarp) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 184;");
    const uint32_t lanes = tmem + ((uint32_t)(warp * 32) << 16), s_at = lanes, o_at = lanes + kTile;
    const int local = (warp * 32 + lane) & ((1 << a.span) - 1);  // row of its head's in the tile
    int g = 0;  // blocks so far
    for (int n = 0;; ++n) {
      bool ok = __all_sync(0xffffffffu, item_there(n));
      if (!ok) break;
      const int blocks = items[n & 1].row0 / kTile + 1, seen = items[n & 1].row0 % kTile + local;  // the last key in the last block that the row sees
      Row sums;
      for (int j = 0; j < blocks; ++j, ++g) {
        ok = __all_sync(0xffffffffu, wait(bars.s_full, g));
        if (!ok) break;
        tc_fence_after_sync();
        const bool last = j == blocks - 1;
        make_weights<D>(sums, s_at, o_at, a.scale, j == 0, last, seen, [&](int half) {
          // behind the last block's look-through, which P V waits for as well: write_rows() below reads what it found
          if (half == 1 && last) ok = __all_sync(0xffffffffu, wait(bars.last_clean, n));
          if (lane == 0) mbar_arrive(bar(bars.p_full[half]));
        });
      }
      ok = ok && wait(bars.o_full, n);
      if (!__all_sync(0xffffffffu, ok)) break;
      tc_fence_after_sync();
      const Item it = items[n & 1];
      const auto sees = [&](int kind, int c) {
        const int x = odd_row[n & 1][kind][c];
        return x >> 8 == n && seen >= 127 - (x & 255);
      };
      const auto place = [&](int r) {
        const int in_tile = warp * 32 + r, row = it.row0 + (in_tile & ((1 << a.span) - 1)), head = it.head + (in_tile >> a.span);
        return row < it.len ? a.out + (int64_t)(it.first + row) * a.ldo + (int64_t)head * D : nullptr;
      };
      write_rows<D>(o_at, sums.l, *reinterpret_cast<volatile int*>(&any_odd[n & 1]) == n + 1, sees, stages[warp], place, lane);
      if (lane == 0) leave_item(n);
      tc_fence_before_sync();  // O has been read: in front of the next item's first weights
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    if (warp == kItemWarp) {
      int g = 0, gv = 0;
      bool ok = true;
      for (int n = 0; ok; ++n) {
        if (n > 0) it = order.item(n * gridDim.x + (n & 1 ? gridDim.x - 1 - blockIdx.x : blockIdx.x));
        if (lane == 0) {
          if (n > 0) {
            ok = n < 2 || wait(bars.item_empty[n & 1], (n >> 1) - 1);
            if (ok) items[n & 1] = it, mbar_arrive(bar(bars.item_full[n & 1]));
          }
          const int blocks = it.head < 0 ? 0 : it.row0 / kTile + 1;
          for (int j = 0; j < blocks && ok; ++j, ++g) {
            if (g > 0) {
              // the scores against the block in front are there: K's slot is free, and with an item's last ones Q's; V's behind P V
              ok = wait(bars.s_full, g - 1);
              if (!ok) break;
              if (j == 0) fetch_q(it);
              fetch(&kmap, k_at, bars.k_full, it.first + j * kTile, it.head / group, kEvictLast);
              ok = wait(bars.v_used, g - 1);
              if (ok) fetch(&vmap, v_at, j + 1 == blocks ? bars.last_full : bars.v_full, it.first + j * kTile, it.head / group, kEvictLast);
              else wait(bars.k_full, g), j == 0 && wait(bars.q_full, n);  // the copies under way land in shared memory
            }
            if (ok && j + 1 < blocks) ++gv;
          }
          if (!ok && g > 0) {  // so does the last V
            if (gv > 0) wait(bars.v_full, gv - 1);
            if (n > 0) wait(bars.last_full, n - 1);
          }
        }
        ok = __shfl_sync(0xffffffffu, ok, 0);
        if (it.head < 0) break;
      }
    } else if (warp == kMmaWarp) {
      if (elect_one()) {
        const auto scores = [&] {
          issue_scores<D>(tmem, q_at, k_at);
          mma_commit(bar(bars.s_full));
        };
        int g = 0, gv = 0;
        bool ok = true;
        for (int n = 0; ok; ++n) {
          if (!item_there(n)) break;
          const int blocks = items[n & 1].row0 / kTile + 1;
          leave_item(n);
          ok = wait(bars.q_full, n) && wait(bars.k_full, g);
          if (!ok) break;
          tc_fence_after_sync();
          scores();
          for (int j = 0; j < blocks && ok; ++j, ++g) {
            ok = j + 1 == blocks ? wait(bars.last_clean, n) : wait(bars.v_full, gv++);
            for (int half = 0; half < 2 && ok; ++half) {  // of the block's keys, whose weights come in turn
              ok = wait(bars.p_full[half], g);
              if (!ok) break;
              tc_fence_after_sync();
              issue_sums<D>(tmem + kTile, tmem, v_at, half, j == 0);
              if (half == 0 && j + 1 < blocks) ok = wait(bars.k_full, g + 1);
            }
            if (!ok) break;
            mma_commit(bar(bars.v_used));
            if (j + 1 < blocks) scores();
            else mma_commit(bar(bars.o_full));
          }
        }
        // what is under way uses shared memory and TMEM
        mma_commit(bar(bars.done));
        wait(bars.done, 0);
      }
    } else {
      const int t = tid - kGuardWarp * 32;
      for (int n = 0;; ++n) {
        if (!__all_sync(0xffffffffu, item_there(n))) break;
        const int keys = items[n & 1].len - items[n & 1].row0 / kTile * kTile;
        __syncwarp();
        if (lane == 0) leave_item(n);
        // Nobody looks at what was found two items ago any more: this item's last V is fetched behind the end of the one before it.
        if (!__all_sync(0xffffffffu, wait(bars.last_full, n))) break;
        look_through<D>(raw + (v_at - smem_addr(raw)), keys, t, [&](int kind, int c, int r) {
          atomicMax(&odd_row[n & 1][kind][c], n * 256 + 127 - r);
          any_odd[n & 1] = n + 1;
        });
        if (lane == 0) mbar_arrive(bar(bars.last_clean));
      }
    }
  }
  tc_fence_before_sync();
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after_sync();
    tmem_dealloc(tmem, kColumns);
  }
}

}  // namespace single

// ---- two tiles that share their keys ------------------------------------------------------------------------------------------

namespace paired {

constexpr int kThreads = 384;
constexpr int kItemWarp = 8, kMmaWarp = 9, kGuardWarp = 10;
constexpr uint32_t kColumns = 512;  // of TMEM: S of both tiles, then O
constexpr int kO = 2 * kTile;
template <int D>
constexpr int kSmem = 6 * kTileBytes<D> + 1024;  // Q of both tiles, two blocks of K, two of V, and what their alignment costs

// A barrier's phase is the number of what it stands for: an item (with two of them, half of it), a block, a use of a slot, or a block
// that is not an item's last on a slot. With one for every item, the slowest of those that wait could be two phases behind.
struct Bars {
  uint64_t item_full[2], item_empty[2], last_full[2], last_clean[2];  // by every other item
  uint64_t q_full, q_used, o_full[2];                                 // by items; o_full of each tile
  uint64_t s_full[2], p_full[2][2];                                   // by blocks, of each tile
  uint64_t k_full[2], k_used[2], v_used[2];                           // by uses of a slot
  uint64_t v_full[2];                                                 // by uses by blocks that are not an item's last
  uint64_t done;
};

template <int D>
__global__ void __launch_bounds__(kThreads, 1)
    paired_kernel(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                  const __grid_constant__ Args a, uint32_t* err) {
  constexpr int BYTES = kTileBytes<D>;
  extern __shared__ unsigned char raw[];
  __shared__ Bars bars;
  __shared__ Item items[2];
  __shared__ uint32_t tmem_slot;
  __shared__ int any_odd[2], odd_row[2][3][D];                // as in single_kernel
  __shared__ __align__(16) unsigned char stages[8][32 * 64];  // 32 columns of a warp's rows on their way out
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t base = (smem_addr(raw) + 1023) & ~1023u;
  const uint32_t q_at = base, k_at = base + 2 * BYTES, v_at = base + 4 * BYTES;
  const auto bar = [](uint64_t& b) { return smem_addr(&b); };
  const auto wait = [&](uint64_t& b, int phase) { return mbar_wait(smem_addr(&b), phase & 1, err); };

  if (warp == kMmaWarp) {
    grid_wait();  // columns only then: the kernel in front may want them for CTAs that have not begun
    tmem_alloc(smem_addr(&tmem_slot), kColumns);
  }
  if (tid == kItemWarp * 32) {
    prefetch_tensormap(&qmap), prefetch_tensormap(&kmap), prefetch_tensormap(&vmap);
    for (int i = 0; i < 2; ++i) {
      mbar_init(bar(bars.item_full[i]), 1), mbar_init(bar(bars.item_empty[i]), 11);
      mbar_init(bar(bars.last_full[i]), 1), mbar_init(bar(bars.last_clean[i]), 2);
      mbar_init(bar(bars.o_full[i]), 1), mbar_init(bar(bars.s_full[i]), 1);
      mbar_init(bar(bars.p_full[i][0]), 4), mbar_init(bar(bars.p_full[i][1]), 4);
      mbar_init(bar(bars.k_full[i]), 1), mbar_init(bar(bars.k_used[i]), 1), mbar_init(bar(bars.v_full[i]), 1), mbar_init(bar(bars.v_used[i]), 1);
    }
    mbar_init(bar(bars.q_full), 1), mbar_init(bar(bars.q_used), 1), mbar_init(bar(bars.done), 1);
    mbar_init_fence();
  }
  const int group = a.q_heads / a.kv_heads;
  const auto fetch = [&](const CUtensorMap* map, uint32_t to, uint64_t& full, const Item& it, int j) {  // block j of K or V
    mbar_expect_tx(bar(full), BYTES);
    tma_load_3d(to, map, bar(full), 0, it.first + j * kTile, it.head / group * (D / 64), kEvictLast);
  };
  const auto fetch_q = [&](const Item& it) {  // rows of its heads, one head behind the other
    mbar_expect_tx(bar(bars.q_full), 2 * BYTES);
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int c = 0; c < D / 64; ++c)
        tma_load_4d(q_at + i * BYTES + c * (kTile * 128), &qmap, bar(bars.q_full), 0, it.first + it.row0, it.head + (i << (a.share - 1)), c, kEvictFirst);
  };
  const auto blocks_of = [](const Item& it) { return it.row0 / kTile + 1; };
  // the first item, and the first of its copies, while the CTA sets itself up
  Order order{a, lane};
  Item it{0, 0, 0, -1};  // of the item warp
  if (warp == kItemWarp) {
    grid_wait();
    order.begin(err);
    it = order.item(blockIdx.x);
    if (lane == 0) {
      items[0] = it;
      mbar_arrive(bar(bars.item_full[0]));
      if (it.head >= 0) {
        fence_async_global();
        fetch(&kmap, k_at, bars.k_full[0], it, 0);
        fetch_q(it);
        fetch(&vmap, v_at, it.row0 < kTile ? bars.last_full[0] : bars.v_full[0], it, 0);
      }
    }
    __syncwarp();
  }
  for (int i = tid; i < 2 * 3 * D; i += kThreads) (&odd_row[0][0][0])[i] = -1;
  if (tid < 2) any_odd[tid] = 0;
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = tmem_slot;
  grid_trigger();

  const auto item_there = [&](int n) { return wait(bars.item_full[n & 1], n >> 1) && items[n & 1].head >= 0; };
  const auto leave_item = [&](int n) { mbar_arrive(bar(bars.item_empty[n & 1])); };

  // registers: 256 * 216 + 128 * 72 = 384 * 168, what the launch has
  if (warp < kItemWarp) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    const int i = warp >> 2, quarter = warp & 3;
    const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16), s_at = lanes + i * kTile, o_at = lanes + kO + i * kTile;
    const int local = (quarter * 32 + lane) & ((1 << a.span) - 1);  // row of its head's in the tile
    int g = 0;  // blocks so far
    for (int n = 0;; ++n) {
      bool ok = __all_sync(0xffffffffu, item_there(n));
      if (!ok) break;
      const int blocks = blocks_of(items[n & 1]), seen = items[n & 1].row0 % kTile + local;  // the last key in the last block that the row sees
      Row sums;
      for (int j = 0; j < blocks; ++j, ++g) {
        ok = __all_sync(0xffffffffu, wait(bars.s_full[i], g));
        if (!ok) break;
        tc_fence_after_sync();
        const bool last = j == blocks - 1;
        make_weights<D>(sums, s_at, o_at, a.scale, j == 0, last, seen, [&](int half) {
          // behind the last block's look-through, which P V waits for as well: write_rows() below reads what it found
          if (half == 1 && last) ok = __all_sync(0xffffffffu, wait(bars.last_clean[n & 1], n >> 1));
          if (lane == 0) mbar_arrive(bar(bars.p_full[i][half]));
        });
      }
      ok = ok && wait(bars.o_full[i], n);
      if (!__all_sync(0xffffffffu, ok)) break;
      tc_fence_after_sync();
      const Item it = items[n & 1];
      const auto sees = [&](int kind, int c) {
        const int x = odd_row[n & 1][kind][c];
        return x >> 8 == n && seen >= 127 - (x & 255);
      };
      const auto place = [&](int r) {
        const int in_tile = quarter * 32 + r, row = it.row0 + (in_tile & ((1 << a.span) - 1)), head = it.head + (i << (a.share - 1)) + (in_tile >> a.span);
        return row < it.len ? a.out + (int64_t)(it.first + row) * a.ldo + (int64_t)head * D : nullptr;
      };
      write_rows<D>(o_at, sums.l, *reinterpret_cast<volatile int*>(&any_odd[n & 1]) == n + 1, sees, stages[warp], place, lane);
      if (lane == 0) leave_item(n);
      tc_fence_before_sync();  // O has been read: in front of the next item's first weights
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    if (warp == kItemWarp) {
      int g = 0, v0 = 0, v1 = 0;                     // blocks so far; of those that are not an item's last, on each slot
      int k_n = it.head >= 0, q_n = k_n, last_n = -1;  // copies of K and Q asked for; the item whose last V is
      bool ok = true;
      for (int n = 0; ok; ++n) {
        if (n > 0) it = order.item(n * gridDim.x + (n & 1 ? gridDim.x - 1 - blockIdx.x : blockIdx.x));
        if (lane == 0) {
          if (n > 0) {
            ok = n < 2 || wait(bars.item_empty[n & 1], (n >> 1) - 1);
            if (ok) items[n & 1] = it, mbar_arrive(bar(bars.item_full[n & 1]));
          }
          const int blocks = it.head < 0 ? 0 : blocks_of(it);
          for (int j = 0; j < blocks && ok; ++j, ++g) {
            const int slot = g & 1, use = g >> 1;
            const bool last = j + 1 == blocks;
            if (g > 0) {
              ok = use == 0 || wait(bars.k_used[slot], use - 1);
              if (!ok) break;
              fetch(&kmap, k_at + slot * BYTES, bars.k_full[slot], it, j), ++k_n;
              if (j == 0) {
                ok = wait(bars.q_used, n - 1);
                if (ok) fetch_q(it), ++q_n;
              }
              ok = ok && (use == 0 || wait(bars.v_used[slot], use - 1));
              if (ok) fetch(&vmap, v_at + slot * BYTES, last ? bars.last_full[n & 1] : bars.v_full[slot], it, j);
            }
            if (ok && last) last_n = n;
            else if (ok) ++(slot ? v1 : v0);
          }
          if (!ok) {  // the copies under way land in shared memory
            for (int i = 0; i < 2; ++i) {
              const int uses = (k_n + 1 - i) / 2, plain = i ? v1 : v0, item = last_n - i;
              if (uses > 0) wait(bars.k_full[i], uses - 1);
              if (plain > 0) wait(bars.v_full[i], plain - 1);
              if (item >= 0) wait(bars.last_full[item & 1], item >> 1);
            }
            if (q_n > 0) wait(bars.q_full, q_n - 1);
          }
        }
        ok = __shfl_sync(0xffffffffu, ok, 0);
        if (it.head < 0) break;
      }
    } else if (warp == kMmaWarp) {
      if (elect_one()) {
        const auto scores = [&](int i, int g, bool frees_q) {  // of tile i against block g
          issue_scores<D>(tmem + i * kTile, q_at + i * BYTES, k_at + (g & 1) * BYTES);
          mma_commit(bar(bars.s_full[i]));
          if (i == 0) return;
          mma_commit(bar(bars.k_used[g & 1]));
          if (frees_q) mma_commit(bar(bars.q_used));
        };
        int g = 0, v0 = 0, v1 = 0, blocks = 0;
        bool more = item_there(0), ok = true;
        if (more) {
          blocks = blocks_of(items[0]);
          leave_item(0);
          ok = wait(bars.q_full, 0) && wait(bars.k_full[0], 0);
          if (ok) {
            tc_fence_after_sync();
            scores(0, 0, false), scores(1, 0, blocks == 1);
          }
        }
        for (int n = 0; more && ok; ++n) {
          int next = 0;  // blocks of the next item
          for (int j = 0; j < blocks && ok; ++j, ++g) {
            const bool last = j + 1 == blocks;
            const int slot = g & 1;
            ok = last ? wait(bars.last_clean[n & 1], n >> 1) : wait(bars.v_full[slot], slot ? v1++ : v0++);
            for (int i = 0; i < 2 && ok; ++i) {
              for (int half = 0; half < 2 && ok; ++half) {  // of the block's keys, whose weights come in turn
                ok = wait(bars.p_full[i][half], g);
                if (!ok) break;
                tc_fence_after_sync();
                issue_sums<D>(tmem + kO + i * kTile, tmem + i * kTile, v_at + slot * BYTES, half, j == 0);
              }
              if (!ok) break;
              if (last) mma_commit(bar(bars.o_full[i]));
              if (i == 1) mma_commit(bar(bars.v_used[slot]));
              if (i == 0) {  // what comes behind: the item's next block, or the next item's first
                more = !last || item_there(n + 1);
                if (last && more) {
                  next = blocks_of(items[(n + 1) & 1]);
                  leave_item(n + 1);
                  ok = wait(bars.q_full, n + 1);
                }
                if (more && ok) ok = wait(bars.k_full[(g + 1) & 1], (g + 1) >> 1);
                tc_fence_after_sync();
              }
              if (more && ok) scores(i, g + 1, last ? next == 1 : j + 2 == blocks);
            }
          }
          blocks = next;
        }
        // what is under way uses shared memory and TMEM
        mma_commit(bar(bars.done));
        wait(bars.done, 0);
      }
    } else {
      const int t = tid - kGuardWarp * 32;
      int g = -1;  // the item's last block
      for (int n = 0;; ++n) {
        if (!__all_sync(0xffffffffu, item_there(n))) break;
        const int keys = items[n & 1].len - items[n & 1].row0 / kTile * kTile;
        g += blocks_of(items[n & 1]);
        __syncwarp();
        if (lane == 0) leave_item(n);
        // Nobody looks at what was found two items ago any more: both tiles have left that item, or this one would not be here.
        if (!__all_sync(0xffffffffu, wait(bars.last_full[n & 1], n >> 1))) break;
        look_through<D>(raw + (v_at - smem_addr(raw)) + (g & 1) * BYTES, keys, t, [&](int kind, int c, int r) {
          atomicMax(&odd_row[n & 1][kind][c], n * 256 + 127 - r);
          any_odd[n & 1] = n + 1;
        });
        if (lane == 0) mbar_arrive(bar(bars.last_clean[n & 1]));
      }
    }
  }
  tc_fence_before_sync();
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after_sync();
    tmem_dealloc(tmem, kColumns);
  }
}

}  // namespace paired

}  // namespace

cudaError_t launch_packed_attend(const PackedAttend& p, int sm_count, uint32_t* err, cudaStream_t s) {
  const int D = p.head_dim;
  if (D != 64 && D != 128) return cudaErrorInvalidValue;
  Args a;
  a.indptr = p.indptr, a.n = p.n, a.rows = p.rows, a.q_heads = p.q_heads, a.kv_heads = p.kv_heads;
  a.scale = p.scale * 1.44269504088896340736f;
  a.out = p.out, a.ldo = p.ldo;
  // Heads of a group share an item's keys as far as their number halves: up to sixteen a tile, eight rows of each, which a swizzled
  // tile's pattern repeats after. Pairs of tiles where the group is even, there is work for every SM and a half more, and sequences have
  // two items' rows in the mean. us, single | paired, 16 heads of 128 over 8: 1 of 2,048 tokens (0.9 items an SM) 36 | 38, 2 of 2,048 (1.8) 45 |
  // 42, 1 of 8,192 250 | 229; 30 of 130 tokens (1 item's rows) 24 | 30, 28 of 32 to 512 (2.1) 36 | 35, 16 of 512 (4) 40 | 37.
  const int halves = __builtin_ctz(p.q_heads / p.kv_heads);
  const auto items_of = [&](int share, int tiles) {  // at most
    a.share = share, a.span = 6 + tiles - share;
    return (((int64_t)p.rows >> a.span) + p.n) * (p.q_heads >> share);
  };
  int64_t items = items_of(std::min(5, halves), 2);
  const bool in_pairs = halves > 0 && items * 2 >= (int64_t)sm_count * 3 && p.rows / p.n >> a.span >= 2;
  if (!in_pairs) items = items_of(std::min(4, halves), 1);
  CUtensorMap maps[3];
  const bf16* at[3] = {p.q, p.k, p.v};
  const int64_t ld[3] = {p.ldq, p.ldk, p.ldv};
  for (int i = 0; i < 3; ++i) {
    const uint64_t heads = i ? p.kv_heads : p.q_heads;
    int rc;
    if (i > 0) {
      const uint64_t dims[3] = {64, (uint64_t)p.rows, heads * (D / 64)}, strides[2] = {(uint64_t)ld[i] * 2, 128};
      const uint32_t box[3] = {64, kTile, (uint32_t)(D / 64)};
      rc = tc_encode_bf16(&maps[i], at[i], 3, dims, strides, box);
    } else {
      const uint64_t dims[4] = {64, (uint64_t)p.rows, heads, (uint64_t)(D / 64)}, strides[3] = {(uint64_t)ld[i] * 2, (uint64_t)D * 2, 128};
      const uint32_t box[4] = {64, 1u << a.span, (uint32_t)kTile >> a.span, 1};
      rc = tc_encode_bf16(&maps[i], at[i], 4, dims, strides, box);
    }
    if (rc != 0) return cudaErrorInvalidValue;
  }
  const auto go = [&](auto d) {
    constexpr int kD = decltype(d)::value;
    cudaError_t e;
    if (in_pairs) {
      if ((e = allow_large<paired::paired_kernel<kD>>(paired::kSmem<kD>)) != cudaSuccess) return e;
      return launch_pdl(paired::paired_kernel<kD>, dim3((unsigned)std::min<int64_t>(items, sm_count)), dim3(paired::kThreads), paired::kSmem<kD>, s,
                        maps[0], maps[1], maps[2], a, err);
    } else {
      if ((e = allow_large<single::single_kernel<kD>>(single::kSmem<kD>)) != cudaSuccess) return e;
      const unsigned ctas = (unsigned)std::min<int64_t>(items, (int64_t)sm_count * single::kPerSm);
      return launch_pdl(single::single_kernel<kD>, dim3(ctas), dim3(single::kThreads), single::kSmem<kD>, s, maps[0], maps[1], maps[2], a, err);
    }
  };
  return D == 128 ? go(std::integral_constant<int, 128>()) : go(std::integral_constant<int, 64>());
}

}  // namespace omni
