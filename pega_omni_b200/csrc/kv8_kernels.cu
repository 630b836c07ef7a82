// Page tables from lengths, norm + rotary embedding of q and k, and the append to 8-bit pages.
#include <cooperative_groups.h>
#include <cuda_fp8.h>

#include <algorithm>
#include <cmath>

#include "kv8.h"

namespace omni {
namespace {

namespace cg = cooperative_groups;

// ---- page tables ------------------------------------------------------------------------------------------------------
// Four prefix sums over the sequences (pages, rows, pages wanted, pages given back), then every page, row and free entry finds
// its sequence in them by bisection: nothing depends on the order in which anything runs. A cluster of CTAs, each of which makes
// the sums for itself (they are a few KB): one launch, no workspace, and the cluster's barrier stands between the last read of
// the lengths and their overwriting, so a captured step can keep its lengths in place.

constexpr int kTablesThreads = 512;

struct Sums {
  int v[4];
  __device__ __forceinline__ void operator+=(const Sums& o) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] += o.v[i];
  }
};

// Index i of the prefix array p[0..n] with p[i] <= x < p[i + 1], for 0 <= x < p[n].
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
  const cg::cluster_group cluster = cg::this_cluster();
  const int n = c.n, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int* const want = tables_smem;        // [n + 1] pages of the sequences in front
  int* const rows = want + n + 1;       // [n + 1] rows
  int* const need = rows + n + 1;       // [n + 1] pages to be taken
  int* const back = need + n + 1;       // [n + 1] pages given back
  int* const held = back + n + 1;       // [n] tokens held
  const int count = *c.free_count;

  const int per = (n + kTablesThreads - 1) / kTablesThreads, begin = min(n, tid * per), end = min(n, begin + per);
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
      for (int i = 0; i < 4; ++i) at.v[i] -= mine.v[i];
      for (int w = 0; w < warp; ++w) at += warp_sums[w];
    }
    for (int s = begin; s < end; ++s) {
      int len, add;
      if (pass == 0) {
        len = c.lens[s], add = c.add[s];
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
    if (pass && tid == kTablesThreads - 1) want[n] = at.v[0], rows[n] = at.v[1], need[n] = at.v[2], back[n] = at.v[3];
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
  const int first = cluster.block_rank() * kTablesThreads + tid, threads = cluster.num_blocks() * kTablesThreads;

  const auto returned = [&](int k) {  // the k-th page given back
    const int s = owner_of(back, n, k);
    return c.table[(int64_t)s * c.width + (k - back[s])];
  };
  const auto page_of = [&](int s, int p) {  // page p of sequence s, which is not gone: its own, or one from the top of the stack
    const int had = pages_of(held[s]);
    if (p < had) return c.table[(int64_t)s * c.width + p];
    const int i = count + back_n - 1 - (need[s] + p - had);
    return i >= count ? returned(i - count) : c.free_pages[i];
  };

  for (int r = first; r < c.row_cap; r += threads) {
    int pos = -1, slot = -1, seq = -1;
    if (ok && r < rows_n) {
      seq = owner_of(rows, n, r);
      pos = held[seq] + (r - rows[seq]);
      slot = (int)((uint32_t)page_of(seq, pos >> 4) * kPageTokens + (pos & 15));
    }
    c.pos[r] = pos, c.slot[r] = slot, c.seq[r] = seq;
  }
  if (ok) {
    for (int e = first; e < pages_n; e += threads) {
      const int s = owner_of(want, n, e), p = e - want[s];
      const int page = page_of(s, p);
      c.pages[e] = page;
      if (p >= pages_of(held[s])) c.table[(int64_t)s * c.width + p] = page;
    }
    // what comes back and is not taken again goes on top of the stack, behind the entries that page_of reads
    for (int k = first; k < back_n - need_n; k += threads) c.free_pages[count + k] = returned(k);
  }
  for (int s = first; s <= n; s += threads) c.indptr[s] = ok ? want[s] : 0, c.row_ptr[s] = ok ? rows[s] : 0;
  cluster.barrier_wait(std::move(all_read));
  for (int s = first; s < n; s += threads) {
    const int len = c.lens[s];  // this thread alone writes it
    c.lens_out[s] = !ok ? len : c.add[s] < 0 ? 0 : len + (rows[s + 1] - rows[s]);
  }
  if (first == 0) {
    *c.free_count_out = ok ? count + back_n - need_n : count;
    *c.status = status;
  }
}

// ---- norm + rotary embedding --------------------------------------------------------------------------------------------
// Bound by HBM: every q and k element is read and written once, 16 bytes an access. A thread holds eight pairs (i, i + D / 2) of
// a head, D / 16 neighbouring lanes a head. The angle of a pair is the same for all heads of a row, so a block makes it once a
// row: in turns and in f64, since f32 would be off by 2^-24 of a far position's whole angle, and only what is left of a turn
// goes to f32 and sincospi. All else is f32 with one rounding.

struct Turns {
  double per_pos[64];
};

constexpr int kRopeThreads = 256;

template <int D, int ROWS>
__global__ void __launch_bounds__(kRopeThreads) qk_norm_rope_kernel(const bf16* x, int64_t ldx, const bf16* __restrict__ q_norm,
                                                                    const bf16* __restrict__ k_norm, const int32_t* __restrict__ pos,
                                                                    int rows, int hq, int heads, float eps, const __grid_constant__ Turns turns,
                                                                    bf16* out, int64_t ldo) {
  constexpr int LANES = D / 16;  // of a head
  __shared__ float2 rot[ROWS][D / 2];
  const int row0 = blockIdx.x * ROWS;
  for (int i = threadIdx.x; i < ROWS * (D / 2); i += kRopeThreads) {
    const int r = i / (D / 2), p = i % (D / 2);
    if (row0 + r < rows) {
      const double t = (double)pos[row0 + r] * turns.per_pos[p];
      float2 f;
      sincospif(2.f * (float)(t - rint(t)), &f.y, &f.x);
      rot[r][p] = f;
    }
  }
  __syncthreads();
  const int per_row = heads * LANES, tasks = ROWS * per_row;
  const int at = (threadIdx.x % LANES) * 8;  // a step of the loop is a whole number of heads
  for (int i = threadIdx.x; i < (tasks + 31) / 32 * 32; i += kRopeThreads) {  // whole warps
    const int r = i / per_row, head = (i - r * per_row) / LANES;
    const bool live = i < tasks && row0 + r < rows && pos[row0 + r] >= 0;
    float lo[8] = {}, hi[8] = {};
    if (live) {
      const bf16* src = x + (int64_t)(row0 + r) * ldx + head * D + at;
      ld8(src, lo), ld8(src + D / 2, hi);
    }
    const bf16* gain = head < hq ? q_norm : k_norm;
    float rn = 1.f;
    float ss = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) ss += lo[e] * lo[e] + hi[e] * hi[e];
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    if (live) {
      if (gain) {
        rn = rsqrtf(ss / D + eps);
        float wl[8], wh[8];
        ld8(gain + at, wl), ld8(gain + D / 2 + at, wh);
#pragma unroll
        for (int e = 0; e < 8; ++e) lo[e] = lo[e] * rn * wl[e], hi[e] = hi[e] * rn * wh[e];
      }
      float a[8], b[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float2 f = rot[r][at + e];
        a[e] = lo[e] * f.x - hi[e] * f.y;
        b[e] = hi[e] * f.x + lo[e] * f.y;
      }
      bf16* dst = out + (int64_t)(row0 + r) * ldo + head * D + at;
      st8(dst, a), st8(dst + D / 2, b);
    }
  }
}

// ---- append ---------------------------------------------------------------------------------------------------------------
// A run is what a call puts into one page: neighbouring rows in ascending slots. A block takes the runs that begin in 16 rows
// (up to 31 rows then: sixteen and what the last run has behind them), of one kv head, K and V; a thread holds eight elements of
// two rows. Rows of a prompt give one run a block, those of a decode step sixteen of one row: both fill it. The runs' largest
// magnitudes meet in shared memory, then each run has its scale, and what the page held before is rounded again if that grew.

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

template <int D>
__global__ void __launch_bounds__(2 * D) kv8_append_kernel(const bf16* __restrict__ k, int64_t ldk, const bf16* __restrict__ v,
                                                           int64_t ldv, const int32_t* __restrict__ slot, int rows, uint8_t* kv,
                                                           float* scales, int kv_pages, int hk, uint32_t* err) {
  constexpr int LANES = D / 8;
  constexpr int kNone = -2;
  __shared__ int sl[33];             // slots of the row in front of the window and of 32 rows from its first
  __shared__ uint32_t amax[16][2];   // of the run that begins at a row of the window
  __shared__ float mul[16][2], ratio[16][2];  // 1 / scale; old scale / new, where it grew over a page that holds tokens
  const int base = blockIdx.x * 16, head = blockIdx.y, tid = threadIdx.x;
  if (tid < 33) {
    const int r = base - 1 + tid;
    int s = r >= 0 && r < rows ? slot[r] : kNone;
    if (s >= 0 && (s >> 4) >= kv_pages) {
      s = kNone;
      if (head == 0) raise(err, kErrBadIndex);
    }
    sl[tid] = s < 0 ? kNone : s;
    if (tid < 32) amax[tid >> 1][tid & 1] = 0, ratio[tid >> 1][tid & 1] = 1.f;
  }
  __syncthreads();
  const auto leads = [&](int i) { return sl[i + 1] >= 0 && ((sl[i + 1] & 15) == 0 || sl[i] + 1 != sl[i + 1]); };  // row base + i begins a run
  const int i0 = tid / LANES, at = tid % LANES * 8;
  float x[2][2][8];  // [row][K | V]
  int run[2];
#pragma unroll
  for (int pass = 0; pass < 2; ++pass) {
    const int i = i0 + 16 * pass;
    int l = -1;
    if (i < 31 && sl[i + 1] >= 0) {
      l = i;
      while (l >= 0 && !leads(l)) --l;  // at most 15 rows back, since a run lies in one page
      if (l >= 16) l = -1;
    }
    run[pass] = l;
    if (l >= 0) {
      ld8(k + (int64_t)(base + i) * ldk + head * D + at, x[pass][0]);
      ld8(v + (int64_t)(base + i) * ldv + head * D + at, x[pass][1]);
    }
  }
#pragma unroll
  for (int pass = 0; pass < 2; ++pass) {
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      float m = 0.f;
      if (run[pass] >= 0) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float a = fabsf(x[pass][w][e]);
          m = fmaxf(m, a < __int_as_float(0x7f800000) ? a : 0.f);
        }
      }
#pragma unroll
      for (int o = LANES / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
      if (run[pass] >= 0 && at == 0) atomicMax(&amax[run[pass]][w], __float_as_uint(m));  // magnitudes order as their bits do
    }
  }
  __syncthreads();
  if (tid < 32 && leads(tid >> 1)) {
    const int l = tid >> 1, w = tid & 1, s = sl[l + 1];
    float* const at_scale = scales + ((int64_t)(s >> 4) * hk + head) * 2 + w;
    float sc = page_scale(__uint_as_float(amax[l][w]));
    if (s & 15) {  // the page holds tokens of this sequence
      const float old = *at_scale;
      sc = fmaxf(sc, old);
      ratio[l][w] = old / sc;
    }
    *at_scale = sc;
    mul[l][w] = 1.f / sc;
  }
  __syncthreads();
#pragma unroll
  for (int pass = 0; pass < 2; ++pass) {
    const int l = run[pass];
    if (l >= 0) {
      const int s = sl[i0 + 16 * pass + 1];
      uint8_t* const dst = kv + (((int64_t)(s >> 4) * hk + head) * 32 + (s & 15)) * D + at;
      *reinterpret_cast<uint2*>(dst) = e4m3_of8(x[pass][0], mul[l][0]);
      *reinterpret_cast<uint2*>(dst + 16 * D) = e4m3_of8(x[pass][1], mul[l][1]);
    }
  }
  for (int l = 0; l < 16; ++l) {
    if (!leads(l)) continue;
    const int s = sl[l + 1];
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      const float f = ratio[l][w];
      if (f != 1.f && i0 < (s & 15)) {
        uint2* const word = reinterpret_cast<uint2*>(kv + (((int64_t)(s >> 4) * hk + head) * 32 + w * 16 + i0) * D + at);
        const uint2 u = *word;
        const float4 a = static_cast<float4>(*reinterpret_cast<const __nv_fp8x4_e4m3*>(&u.x));
        const float4 b = static_cast<float4>(*reinterpret_cast<const __nv_fp8x4_e4m3*>(&u.y));
        const float old[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
        *word = e4m3_of8(old, f);
      }
    }
  }
}

}  // namespace

cudaError_t launch_kv_tables(const TablesCall& c, cudaStream_t s) {
  const size_t smem = (size_t)(5 * c.n + 4) * sizeof(int);
  const cudaError_t e = cudaFuncSetAttribute(kv_tables_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (5 * kTablesMaxSeqs + 4) * 4);
  if (e != cudaSuccess) return e;
  // a CTA for every two thousand entries that there may be, eight at most (the portable cluster size)
  const int64_t entries = (int64_t)c.page_cap + c.row_cap;
  const unsigned ctas = entries > 16384 ? 8 : entries > 4096 ? 4 : entries > 2048 ? 2 : 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas), cfg.blockDim = dim3(kTablesThreads), cfg.dynamicSmemBytes = smem, cfg.stream = s;
  cudaLaunchAttribute attr = {};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = ctas, attr.val.clusterDim.y = 1, attr.val.clusterDim.z = 1;
  cfg.attrs = &attr, cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kv_tables_kernel, c);
}

cudaError_t launch_qk_norm_rope(const bf16* x, int64_t ldx, const bf16* q_norm, const bf16* k_norm, const int32_t* pos, int rows,
                                int q_heads, int kv_heads, int head_dim, float eps, float theta, bf16* out, int64_t ldo,
                                cudaStream_t s) {
  Turns turns;
  for (int i = 0; i < head_dim / 2; ++i)
    turns.per_pos[i] = std::pow((double)theta, -2.0 * i / head_dim) / 6.283185307179586476925286766559;
  const auto go = [&](auto kernel, int per) {
    kernel<<<(rows + per - 1) / per, kRopeThreads, 0, s>>>(x, ldx, q_norm, k_norm, pos, rows, q_heads, q_heads + kv_heads, eps, turns, out, ldo);
    return cudaGetLastError();
  };
  const bool many = rows >= 1024;  // rows enough for every SM at four a block
  if (head_dim == 128) return many ? go(qk_norm_rope_kernel<128, 4>, 4) : go(qk_norm_rope_kernel<128, 1>, 1);
  if (head_dim == 64) return many ? go(qk_norm_rope_kernel<64, 4>, 4) : go(qk_norm_rope_kernel<64, 1>, 1);
  return cudaErrorInvalidValue;
}

cudaError_t launch_kv8_append(const bf16* k, int64_t ldk, const bf16* v, int64_t ldv, const int32_t* slot, int rows, uint8_t* kv,
                              float* scales, int kv_pages, int kv_heads, int head_dim, uint32_t* err, cudaStream_t s) {
  const dim3 grid((rows + 15) / 16, kv_heads);
  if (head_dim == 128) kv8_append_kernel<128><<<grid, 256, 0, s>>>(k, ldk, v, ldv, slot, rows, kv, scales, kv_pages, kv_heads, err);
  else if (head_dim == 64) kv8_append_kernel<64><<<grid, 128, 0, s>>>(k, ldk, v, ldv, slot, rows, kv, scales, kv_pages, kv_heads, err);
  else return cudaErrorInvalidValue;
  return cudaGetLastError();
}

}  // namespace omni
