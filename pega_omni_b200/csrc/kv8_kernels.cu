// Page tables from lengths, norm + rotary embedding of q and k, and the append to 8-bit pages.
#include <cooperative_groups.h>
#include <cuda_fp8.h>

#include <algorithm>
#include <cmath>

#include "f32x2.cuh"
#include "kv8.h"
#include "pdl.cuh"

namespace omni {
namespace {

namespace cg = cooperative_groups;

// ---- page tables ------------------------------------------------------------------------------------------------------
// Four prefix sums over the sequences (pages, rows, pages wanted, pages given back), then every page, row and free entry finds
// its sequence in them: nothing depends on the order in which anything runs. Every CTA makes the sums for itself (they are a few
// KB): one launch, no workspace. Where lengths or height are kept in place, as a captured step does, the CTAs are one cluster, whose
// barrier stands between the last read of them and their overwriting. What takes the time is the way from the lengths to the last
// page, not the bytes: 4.1 us for 64 sequences that step, 7.2 us for 1,000 of up to 8,000 tokens (2 MB).

constexpr int kTablesThreads = 1024;  // at most
constexpr int kChunk = 256;            // pages

struct Sums {
  int v[4];
  __device__ __forceinline__ void operator+=(const Sums& o) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] += o.v[i];
  }
};

// Index i of the prefix array p[0..n] with p[i] <= x < p[i + 1], which is there.
__device__ __forceinline__ int owner_of(const int* p, int n, int x) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (p[mid + 1] > x) hi = mid;
    else lo = mid + 1;
  }
  return lo;
}

__device__ __forceinline__ int pages_of(int tokens) { return (tokens >> 4) + ((tokens & 15) != 0); }

__global__ void __launch_bounds__(kTablesThreads) kv_tables_kernel(const TablesCall c) {
  extern __shared__ int tables_smem[];
  __shared__ Sums warp_sums[kTablesThreads / 32];
  const int block = blockDim.x, warps = block >> 5;
  const cg::cluster_group cluster = cg::this_cluster();
  const int n = c.n, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int* const want = tables_smem;        // [n + 1] pages of the sequences in front
  int* const rows = want + n + 1;       // [n + 1] rows
  int* const need = rows + n + 1;       // [n + 1] pages to be taken
  int* const back = need + n + 1;       // [n + 1] pages given back
  int* const held = back + n + 1;       // [n] tokens held
  grid_wait();
  grid_trigger();
  const int count = __ldcg(c.free_count);

  const int per = (n + block - 1) / block, begin = min(n, tid * per), end = min(n, begin + per);
  bool bad = false;
  Sums mine = {};
  for (int pass = 0; pass < 2; ++pass) {
    Sums at = {};
    if (pass) {  // the sums of the threads in front
      Sums incl = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        Sums up;
#pragma unroll
        for (int i = 0; i < 4; ++i) up.v[i] = __shfl_up_sync(0xffffffffu, incl.v[i], o);
        if (lane >= o) incl += up;
      }
      if (lane == 31) warp_sums[warp] = incl;
      __syncthreads();
      at = incl;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int in_front = lane < warp ? warp_sums[lane].v[i] : 0;  // every warp adds them up for itself
        at.v[i] += __reduce_add_sync(0xffffffffu, in_front) - mine.v[i];
      }
    }
    for (int s = begin; s < end; ++s) {
      int len, add;
      if (pass == 0) {
        len = __ldcg(c.lens + s), add = __ldcg(c.add + s);
        const bool wrong = len < 0 || add < -1 || (int64_t)len + max(add, 0) > (int64_t)c.width * kPageTokens;
        bad |= wrong;
        if (wrong) len = 0, add = 0;
        held[s] = len;
        rows[s] = add;  // until the second pass
      } else {
        len = held[s], add = rows[s];
      }
      const bool gone = add < 0;
      const int had = pages_of(len), total = gone ? 0 : pages_of(len + add);
      if (pass) want[s] = at.v[0], rows[s] = at.v[1], need[s] = at.v[2], back[s] = at.v[3];
      Sums one;
      one.v[0] = total, one.v[1] = max(add, 0), one.v[2] = gone ? 0 : total - had, one.v[3] = gone ? had : 0;
      if (pass) at += one;
      else mine += one;
    }
    if (pass && tid == block - 1) want[n] = at.v[0], rows[n] = at.v[1], need[n] = at.v[2], back[n] = at.v[3];
  }
  bad = __syncthreads_or(bad);
  cg::cluster_group::arrival_token all_read = cluster.barrier_arrive();  // this CTA has read the lengths and the count

  const int pages_n = want[n], rows_n = rows[n], need_n = need[n], back_n = back[n];
  int32_t status = bad ? kTablesBadLength : 0;
  if (count < 0 || count > c.free_cap || (int64_t)count + back_n - need_n > c.free_cap) status |= kTablesFree;
  if ((int64_t)count + back_n < need_n) status |= kTablesNoPages;
  if (rows_n > c.row_cap) status |= kTablesRows;
  if (pages_n > c.page_cap) status |= kTablesPages;
  const bool ok = status == 0;
  const int first = blockIdx.x * block + tid, threads = gridDim.x * block;

  const auto returned = [&](int k) {  // the k-th page given back
    const int s = owner_of(back, n, k);
    return __ldcg(c.table + (int64_t)s * c.width + (k - back[s]));
  };
  const auto taken = [&](int j) {  // the j-th page from the top of the stack
    const int i = count + back_n - 1 - j;
    return i >= count ? returned(i - count) : __ldcg(c.free_pages + i);
  };
  // a warp takes kChunk pages and rows of a sequence at a time, so a long one among many is shared
  const int chunks = ok ? (c.width + kChunk - 1) / kChunk : 0;
  for (int task = blockIdx.x * warps + warp; task < n * chunks; task += gridDim.x * warps) {
    const int chunk = task / n, s = task - chunk * n, len = held[s], had = pages_of(len), total = want[s + 1] - want[s];
    const int32_t* const mine = c.table + (int64_t)s * c.width;
    const int p0 = chunk * kChunk, p1 = min(total, p0 + kChunk), own = min(had, p1);
#pragma unroll 4
    for (int p = p0 + lane; p < own; p += 32) c.pages[want[s] + p] = __ldcg(mine + p);
    for (int p = max(p0, had) + lane; p < p1; p += 32) {
      const int page = taken(need[s] + p - had);
      c.pages[want[s] + p] = page, c.table[(int64_t)s * c.width + p] = page;
    }
    __syncwarp();  // the rows' pages are those that this warp has just entered
    const int32_t* const pages_of_s = c.pages + want[s];
    const int pos1 = min(len + (rows[s + 1] - rows[s]), p1 * kPageTokens), to_row = rows[s] - len;
#pragma unroll 4
    for (int pos = max(len, p0 * kPageTokens) + lane; pos < pos1; pos += 32) {
      c.slot[pos + to_row] = (int)((uint32_t)pages_of_s[pos >> 4] * kPageTokens + (pos & 15));
      c.pos[pos + to_row] = pos, c.seq[pos + to_row] = s;
    }
  }
  for (int r = (ok ? rows_n : 0) + first; r < c.row_cap; r += threads) c.pos[r] = c.slot[r] = c.seq[r] = -1;
  // what comes back and is not taken again goes on top of the stack, behind the entries that are taken from it
  if (ok)
    for (int k = first; k < back_n - need_n; k += threads) c.free_pages[count + k] = returned(k);
  for (int s = first; s <= n; s += threads) c.indptr[s] = ok ? want[s] : 0, c.row_ptr[s] = ok ? rows[s] : 0;
  cluster.barrier_wait(std::move(all_read));
  for (int s = first; s < n; s += threads) {
    const int len = __ldcg(c.lens + s);  // this thread alone writes it
    c.lens_out[s] = !ok ? len : __ldcg(c.add + s) < 0 ? 0 : len + (rows[s + 1] - rows[s]);
  }
  if (first == 0) {
    *c.free_count_out = ok ? count + back_n - need_n : count;
    *c.status = status;
  }
}

// ---- norm + rotary embedding --------------------------------------------------------------------------------------------
// Bound by HBM: every q and k element is read and written once, 16 bytes an access. A lane holds eight pairs (i, i + D / 2) of a
// head, D / 16 neighbouring lanes a head, and a warp takes up to kRopeBatch such loads of one row at a time, all under way before
// the first is used. The angle of a pair is the same for all heads of a row, so a warp makes each once, under its loads, and a
// lane keeps its eight: in turns and in f64, since f32 would be off by 2^-24 of a far position's whole angle, and only what is left
// of a turn goes to f32 and sincospi. All else is f32 with one rounding. 8,192 rows of 40 heads of 128: 29.3 us, 5.7 TB/s, where a
// plain copy of them takes 27.6 us; angles and norms are half of what the SMs can issue meanwhile. 64 rows of 24 heads: 2.3 us.

struct Turns {
  double per_pos[64];
};

constexpr int kRopeWarps = 2, kRopeBatch = 2;

__device__ __forceinline__ void pairs_of(const uint4& u, float2 (&v)[4]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
}
__device__ __forceinline__ uint4 packed_of(const float2 (&v)[4]) {
  uint4 u;
  uint32_t* const w = &u.x;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(v[i].x, v[i].y);
    w[i] = *reinterpret_cast<const uint32_t*>(&h);
  }
  return u;
}

// Block y of a row's y_blocks: heads of q where y < q_blocks, otherwise of k.
template <int D>
__global__ void __launch_bounds__(kRopeWarps * 32, 14) qk_norm_rope_kernel(const bf16* x, int64_t ldx, const bf16* q_norm,
                                                                       const bf16* k_norm, const int32_t* pos,
                                                                       int rows, int hq, int heads, int q_blocks, int y_blocks, float eps,
                                                                       const __grid_constant__ Turns turns, bf16* out, int64_t ldo) {
  constexpr int LANES = D / 16, HEADS = 32 / LANES;  // lanes of a head, heads of a warp's access
  __shared__ __align__(16) float2 rot[kRopeWarps][D / 2];
  grid_wait();
  grid_trigger();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t row = (int64_t)(blockIdx.x / y_blocks) * kRopeWarps + warp;
  const int y = blockIdx.x % y_blocks;
  if (row >= rows) return;
  const bool is_q = y < q_blocks;
  const int end = is_q ? hq : heads, at = lane % LANES * 8;
  const int head0 = (is_q ? y : y - q_blocks) * (HEADS * kRopeBatch) + (is_q ? 0 : hq) + lane / LANES;
  const int my_pos = __ldcg(pos + row);
  const bf16* const src = x + row * ldx + head0 * D + at;
  uint4 lo_raw[kRopeBatch], hi_raw[kRopeBatch];
#pragma unroll
  for (int b = 0; b < kRopeBatch; ++b) {
    lo_raw[b] = hi_raw[b] = make_uint4(0, 0, 0, 0);
    if (head0 + b * HEADS < end) {
      lo_raw[b] = __ldcg(reinterpret_cast<const uint4*>(src + b * HEADS * D)), hi_raw[b] = __ldcg(reinterpret_cast<const uint4*>(src + b * HEADS * D + D / 2));
    }
  }
  const bf16* const gain = is_q ? q_norm : k_norm;
  uint4 lo_gain = {}, hi_gain = {};
  if (gain) lo_gain = __ldcg(reinterpret_cast<const uint4*>(gain + at)), hi_gain = __ldcg(reinterpret_cast<const uint4*>(gain + D / 2 + at));
  if (my_pos < 0) return;
#pragma unroll
  for (int p = lane; p < D / 2; p += 32) {
    double per_pos;  // through a generic address: as a constant, each lane's would be read by itself (32 us instead of 29 for the case above)
    asm("ld.f64 %0, [%1];" : "=d"(per_pos) : "l"(&turns.per_pos[p]));
    const double t = (double)my_pos * per_pos;
    float2 f;
    sincospif(2.f * (float)(t - rint(t)), &f.y, &f.x);
    rot[warp][(((p >> 1) & 3) * LANES + (p >> 3)) * 2 + (p & 1)] = f;  // the lanes' pairs side by side, so that no banks collide
  }
  __syncwarp();
  // (lo, hi) -> (lo * lc - hi * hs, hi * hc + lo * ls), the gains in the angles
  float2 lc[4], ls[4], hc[4], hs[4];
  pairs_of(lo_gain, lc), pairs_of(hi_gain, hc);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float4 f = *reinterpret_cast<const float4*>(&rot[warp][(e * LANES + lane % LANES) * 2]);
    const float2 cs = make_float2(f.x, f.z), sn = make_float2(f.y, f.w), minus = make_float2(-f.y, -f.w);
    if (gain) ls[e] = mul2(lc[e], sn), hs[e] = mul2(hc[e], minus), lc[e] = mul2(lc[e], cs), hc[e] = mul2(hc[e], cs);
    else ls[e] = sn, hs[e] = minus, lc[e] = cs, hc[e] = cs;
  }
  bf16* const dst = out + row * ldo + head0 * D + at;
#pragma unroll
  for (int b = 0; b < kRopeBatch; ++b) {
    float2 lo[4], hi[4];
    pairs_of(lo_raw[b], lo), pairs_of(hi_raw[b], hi);
    float2 rn = make_float2(1.f, 1.f);
    if (gain) {
      float2 ss = mul2(lo[0], lo[0]);
#pragma unroll
      for (int e = 1; e < 4; ++e) ss = fma2(lo[e], lo[e], ss);
#pragma unroll
      for (int e = 0; e < 4; ++e) ss = fma2(hi[e], hi[e], ss);
      float sum = ss.x + ss.y;
#pragma unroll
      for (int o = LANES / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      rn.x = rn.y = rsqrtf(sum * (1.f / D) + eps);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 l = mul2(lo[e], rn), h = mul2(hi[e], rn);
      lo[e] = fma2(l, lc[e], mul2(h, hs[e])), hi[e] = fma2(h, hc[e], mul2(l, ls[e]));
    }
    if (head0 + b * HEADS < end) {
      *reinterpret_cast<uint4*>(dst + b * HEADS * D) = packed_of(lo);
      *reinterpret_cast<uint4*>(dst + b * HEADS * D + D / 2) = packed_of(hi);
    }
  }
}

// ---- append ---------------------------------------------------------------------------------------------------------------
// A run is what a call puts into one page: neighbouring rows in ascending slots. A warp takes the runs that begin in 16 rows (up to
// 31 rows then: sixteen and what the last run has behind them), of K or V of one kv head. A run by itself, as prompts make them, is
// held in registers as sixteen rows from its first on; several are taken row by row, from memory again where they are more than
// sixteen rows. No warp waits for another. Lane r keeps what there is to know of row r: its slot, the row that begins its run, that
// run's largest magnitude and scale.
// Bound by HBM where there are many rows (2 bytes in, 1 out an element), but a warp's page is a chain of slots, rows, maximum and store:
// 7,600 rows of 8 heads of 128 take 13.7 us, 3.4 TB/s; the first sixteen rows are under way before the slots are known (14.1 otherwise), and
// more warps at fewer registers make it no faster. 61 rows of as many sequences: 4.3 us.

// The smallest 2^e >= 2^-100 with amax <= 448 * 2^e; amax finite, not negative. 448 = 1.75 * 2^8.
__device__ __forceinline__ float page_scale(float amax) {
  const uint32_t bits = __float_as_uint(amax);
  const int e = (int)(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u);
  return __uint_as_float((uint32_t)(max(e, -100) + 127) << 23);
}

__device__ __forceinline__ uint32_t e4m3_of4(float a, float b, float c, float d) {
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
  return lo | hi << 16;
}

__device__ __forceinline__ uint2 e4m3_of8(const float* v, float mul) {
  return make_uint2(e4m3_of4(v[0] * mul, v[1] * mul, v[2] * mul, v[3] * mul), e4m3_of4(v[4] * mul, v[5] * mul, v[6] * mul, v[7] * mul));
}
__device__ __forceinline__ uint2 e4m3_of8(const uint4& u, float mul) {
  float2 v[4];
  pairs_of(u, v);
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = mul2(v[i], make_float2(mul, mul));
  return make_uint2(e4m3_of4(v[0].x, v[0].y, v[1].x, v[1].y), e4m3_of4(v[2].x, v[2].y, v[3].x, v[3].y));
}

// The largest magnitude of eight bf16 in each half, infinities and (unless there is nothing else) no NaN among them.
__device__ __forceinline__ __nv_bfloat162 abs_max(const uint4& u) {
  __nv_bfloat162 m = __habs2(*reinterpret_cast<const __nv_bfloat162*>(&u.x));
  m = __hmax2(m, __habs2(*reinterpret_cast<const __nv_bfloat162*>(&u.y)));
  m = __hmax2(m, __habs2(*reinterpret_cast<const __nv_bfloat162*>(&u.z)));
  return __hmax2(m, __habs2(*reinterpret_cast<const __nv_bfloat162*>(&u.w)));
}

constexpr int kAppendWarps = 2;

template <int D>
__global__ void __launch_bounds__(kAppendWarps * 32, 12) kv8_append_kernel(const bf16* k, int64_t ldk, const bf16* v,
                                                                       int64_t ldv, const int32_t* slot, int rows, uint8_t* kv,
                                                                       float* scales, int kv_pages, int hk, int head_blocks, uint32_t* err) {
  constexpr int LANES = D / 8, TOGETHER = 32 / LANES, STEPS = 16 / TOGETHER;  // lanes of a row, rows of an access, accesses of 16 rows
  constexpr float kInf = __builtin_huge_valf();
  __shared__ float row_max[kAppendWarps][32];
  grid_wait();
  grid_trigger();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  // blocks of the same rows follow one another: neighbouring heads are neighbours in DRAM
  const int base = blockIdx.x / head_blocks * 16, what = blockIdx.x % head_blocks * kAppendWarps + warp, head = what >> 1, w = what & 1;
  if (head >= hk) return;
  const int sub = lane / LANES, at = lane % LANES * 8;
  const bf16* const src = (w ? v : k) + head * D + at;
  const int64_t ld = w ? ldv : ldk;
  uint4 x[STEPS];  // rows base + from + i * TOGETHER + sub
  const auto fetch = [&](int i, int r) { x[i] = __ldcg(reinterpret_cast<const uint4*>(src + (int64_t)(base + r) * ld)); };
#pragma unroll
  for (int i = 0; i < STEPS; ++i) {
    x[i] = make_uint4(0, 0, 0, 0);
    if (base + i * TOGETHER + sub < rows) fetch(i, i * TOGETHER + sub);  // under way before the slots are known
  }
  const int64_t limit = (int64_t)kv_pages * 16;
  const auto slot_of = [&](int r) {  // -2: none
    const int s = r >= 0 && r < rows ? __ldcg(slot + r) : -2;
    if (s >= limit) raise(err, kErrBadIndex);
    return s < 0 || s >= limit ? -2 : s;
  };
  int s = slot_of(base + lane);
  const int edge = lane == 0 ? slot_of(base - 1) : -2;
  int before = __shfl_up_sync(0xffffffffu, s, 1);
  if (lane == 0) before = edge;
  if (s >= 0 && before >= 0 && s >> 4 == before >> 4 && s != before + 1) {  // not its page's next token: two runs would write the page
    raise(err, kErrBadIndex);
    s = -2;
  }
  const uint32_t leaders = __ballot_sync(0xffffffffu, s >= 0 && ((s & 15) == 0 || before + 1 != s));
  const int l = 31 - __clz(leaders & (2u << lane) - 1u);  // that begins no later; -1 where the run begins in front of the window
  const int run = s >= 0 && l < 16 ? l : -1;
  const bool mine = run == lane;  // this lane's row begins a run of this warp
  float* const at_scale = scales + ((int64_t)(max(s, 0) >> 4) * hk + head) * 2 + w;
  const bool held = mine && (s & 15);  // the page holds tokens of this sequence
  const float old = held ? __ldcg(at_scale) : 0.f;
  const uint32_t ours = __ballot_sync(0xffffffffu, run >= 0);
  if (ours == 0) return;
  const uint32_t runs = leaders & 0xffffu;
  // one run as a prompt gives it: sixteen rows from its first on, in slots that follow one another
  const int first = __ffs(runs) - 1, from_first = __shfl_sync(0xffffffffu, s - lane, first);
  const bool one = (runs & (runs - 1)) == 0 && __all_sync(0xffffffffu, run < 0 || s - lane == from_first);
  const int lead = one ? first : 0;
  const int passes = !one && ours >> 16 ? 2 : 1;
  const auto is_ours = [&](int from, int i) { return (ours >> (from + i * TOGETHER + sub) & 1) != 0; };
  const auto load = [&](int from) {
#pragma unroll
    for (int i = 0; i < STEPS; ++i)
      if (is_ours(from, i)) fetch(i, from + i * TOGETHER + sub);
  };
  const auto finite_max = [&](int i) {
    float f[8], most = 0.f;
    unpack8v(x[i], f);
#pragma unroll
    for (int e = 0; e < 8; ++e) most = fabsf(f[e]) < kInf ? fmaxf(most, fabsf(f[e])) : most;
    return most;
  };
  if (lead > 0) load(lead);
  // the largest magnitudes: of the one run, otherwise row by row and run by run
  float m = 0.f;
  if (one) {
    __nv_bfloat162 m2 = __floats2bfloat162_rn(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < STEPS; ++i)
      if (is_ours(lead, i)) m2 = __hmax2(m2, abs_max(x[i]));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m2 = __hmax2(m2, __shfl_xor_sync(0xffffffffu, m2, o));
    m = fmaxf(__low2float(m2), __high2float(m2));
    if (m == kInf) {  // infinities do not count: once more without
      m = 0.f;
#pragma unroll
      for (int i = 0; i < STEPS; ++i)
        if (is_ours(lead, i)) m = fmaxf(m, finite_max(i));
      m = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(m)));
    }
  } else {
    for (int again = 0; again < 2; ++again) {
#pragma unroll 1
      for (int pass = 0; pass < passes; ++pass) {
        if (passes == 2 && pass + again > 0) load(16 * pass);
#pragma unroll
        for (int i = 0; i < STEPS; ++i) {
          float its;
          if (again) {
            its = finite_max(i);
#pragma unroll
            for (int o = LANES / 2; o > 0; o >>= 1) its = fmaxf(its, __shfl_xor_sync(0xffffffffu, its, o));
          } else {
            __nv_bfloat162 m2 = abs_max(x[i]);
#pragma unroll
            for (int o = LANES / 2; o > 0; o >>= 1) m2 = __hmax2(m2, __shfl_xor_sync(0xffffffffu, m2, o));
            its = fmaxf(__low2float(m2), __high2float(m2));
          }
          if (at == 0) row_max[warp][16 * pass + i * TOGETHER + sub] = its;
        }
      }
      __syncwarp();
      m = run >= 0 ? row_max[warp][lane] : 0.f;
      if (!__any_sync(0xffffffffu, m == kInf)) break;
      __syncwarp();
    }
  }
  const uint32_t my_max = __float_as_uint(fmaxf(m, 0.f));  // magnitudes order as their bits do; a row of NaN: 0
  uint32_t top = my_max;
  for (uint32_t left = one ? 0 : runs; left; left &= left - 1) {
    const int r = __ffs(left) - 1;
    const uint32_t its = __reduce_max_sync(0xffffffffu, run == r ? my_max : 0);
    if (lane == r) top = its;
  }
  float scale = page_scale(__uint_as_float(top)), ratio = 1.f;  // old scale / new, where it grew over a page that holds tokens
  if (held) scale = fmaxf(scale, old), ratio = old / scale;
  if (mine) *at_scale = scale;
  const int64_t to = (((int64_t)(max(s, 0) >> 4) * hk + head) * 32 + w * 16 + (s & 15)) * D;  // of lane r's row
  if (one) {  // one row behind the other
    const float by = __shfl_sync(0xffffffffu, 1.f / scale, lead);
    uint8_t* const dst = kv + (__shfl_sync(0xffffffffu, to, lead) + sub * D + at);
#pragma unroll
    for (int i = 0; i < STEPS; ++i)
      if (is_ours(lead, i)) *reinterpret_cast<uint2*>(dst + i * TOGETHER * D) = e4m3_of8(x[i], by);
  } else {
    const float mul = __shfl_sync(0xffffffffu, 1.f / scale, max(run, 0));
#pragma unroll 1
    for (int pass = 0; pass < passes; ++pass) {
      if (passes == 2) load(16 * pass);
#pragma unroll
      for (int i = 0; i < STEPS; ++i) {
        const int r = 16 * pass + i * TOGETHER + sub;
        const float by = __shfl_sync(0xffffffffu, mul, r);
        uint8_t* const dst = kv + (__shfl_sync(0xffffffffu, to, r) + at);
        if (is_ours(16 * pass, i)) *reinterpret_cast<uint2*>(dst) = e4m3_of8(x[i], by);
      }
    }
  }
  for (uint32_t left = __ballot_sync(0xffffffffu, mine && ratio != 1.f); left; left &= left - 1) {
    const int r = __ffs(left) - 1, its_slot = __shfl_sync(0xffffffffu, s, r);
    const float by = __shfl_sync(0xffffffffu, ratio, r);
    for (int t = sub; t < (its_slot & 15); t += TOGETHER) {
      uint2* const word = reinterpret_cast<uint2*>(kv + (((int64_t)(its_slot >> 4) * hk + head) * 32 + w * 16 + t) * D + at);
      const uint2 u = __ldcg(word);
      const float4 a = static_cast<float4>(*reinterpret_cast<const __nv_fp8x4_e4m3*>(&u.x));
      const float4 b = static_cast<float4>(*reinterpret_cast<const __nv_fp8x4_e4m3*>(&u.y));
      const float codes[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
      *word = e4m3_of8(codes, by);
    }
  }
}

}  // namespace

cudaError_t launch_kv_tables(const TablesCall& c, cudaStream_t s) {
  const size_t smem = (size_t)(5 * c.n + 4) * sizeof(int);
  const cudaError_t e = allow_large<kv_tables_kernel>((5 * kTablesMaxSeqs + 4) * 4);
  if (e != cudaSuccess) return e;
  // a warp for every sequence and for every 128 pages and rows that there may be; in one cluster (of sixteen CTAs at most) where
  // lengths or height are kept in place, otherwise without one
  const bool in_place = c.lens == c.lens_out || c.free_count == c.free_count_out;
  const int64_t warps = std::max<int64_t>(c.n, ((int64_t)c.page_cap + c.row_cap) / 128);
  const unsigned most = in_place ? 16 : 128;
  unsigned ctas = 1;
  while (ctas < most && warps > (int64_t)ctas * 16) ctas *= 2;
  const unsigned block = in_place && warps > 16 * 16 ? kTablesThreads : kTablesThreads / 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas), cfg.blockDim = dim3(block), cfg.dynamicSmemBytes = smem, cfg.stream = s;
  cudaLaunchAttribute attr[2] = {};
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = in_place ? ctas : 1, attr[0].val.clusterDim.y = 1, attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr, cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, kv_tables_kernel, c);
}

cudaError_t launch_qk_norm_rope(const bf16* x, int64_t ldx, const bf16* q_norm, const bf16* k_norm, const int32_t* pos, int rows,
                                int q_heads, int kv_heads, int head_dim, float eps, float theta, bf16* out, int64_t ldo,
                                cudaStream_t s) {
  Turns turns;
  double low[8];  // theta^(-2 i / head_dim) as a product of two powers
  for (int i = 0; i < 8; ++i) low[i] = std::pow((double)theta, -2.0 * i / head_dim);
  for (int i = 0; i < head_dim / 2; i += 8) {
    const double high = std::pow((double)theta, -2.0 * i / head_dim) / 6.283185307179586476925286766559;
    for (int j = 0; j < 8; ++j) turns.per_pos[i + j] = high * low[j];
  }
  const int per_warp = 32 / (head_dim / 16) * kRopeBatch;  // heads
  const int q_blocks = (q_heads + per_warp - 1) / per_warp, k_blocks = (kv_heads + per_warp - 1) / per_warp;
  const unsigned grid = (unsigned)((rows + kRopeWarps - 1) / kRopeWarps) * (q_blocks + k_blocks);
  const auto go = [&](auto kernel) {
    return launch_pdl(kernel, dim3(grid), dim3(kRopeWarps * 32), 0, s, x, ldx, q_norm, k_norm, pos, rows, q_heads, q_heads + kv_heads, q_blocks,
                      q_blocks + k_blocks, eps, turns, out, ldo);
  };
  if (head_dim == 128) return go(qk_norm_rope_kernel<128>);
  if (head_dim == 64) return go(qk_norm_rope_kernel<64>);
  return cudaErrorInvalidValue;
}

cudaError_t launch_kv8_append(const bf16* k, int64_t ldk, const bf16* v, int64_t ldv, const int32_t* slot, int rows, uint8_t* kv,
                              float* scales, int kv_pages, int kv_heads, int head_dim, uint32_t* err, cudaStream_t s) {
  const int head_blocks = (2 * kv_heads + kAppendWarps - 1) / kAppendWarps;
  const unsigned grid = (unsigned)((rows + 15) / 16) * head_blocks;
  const auto go = [&](auto kernel) {
    return launch_pdl(kernel, dim3(grid), dim3(kAppendWarps * 32), 0, s, k, ldk, v, ldv, slot, rows, kv, scales, kv_pages, kv_heads, head_blocks, err);
  };
  if (head_dim == 128) return go(kv8_append_kernel<128>);
  if (head_dim == 64) return go(kv8_append_kernel<64>);
  return cudaErrorInvalidValue;
}

}  // namespace omni
