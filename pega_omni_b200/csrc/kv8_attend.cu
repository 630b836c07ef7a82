// Decode attention over pages in 8 bits (kv8.h): one query row a sequence, grouped heads.
//
// Bound by HBM: 2 D bytes a token and kv head are read once, for 4 D operations a query head on them. A warp takes every W-th page
// of a row and kv head, W being the warps of its cluster; its pages travel through a ring of its own in shared memory (cp.async,
// kStages deep), so warps never wait for one another before the end. There the warps' sums meet in shared memory and the CTAs'
// in distributed shared memory: one launch, no workspace, sums in a fixed order.
//
// Both products run on m16n8k16 with the page as the left operand and the queries as the eight columns, so a group of up to eight
// heads wastes no rows of it: S^T[16 tokens, 8 queries] = K Q^T and O^T[D, 8 queries] += V^T P^T. E4M3 widens to f16 without loss. The
// order of the head's elements within a sum is free, so a lane's operands are whole words of a key's row (Q is held in the same
// order), and those of V^T are bytes of two tokens put side by side. Queries go to f16 under a power of two of their own, which
// loses nothing above 2^-39 of the largest. With s the score in powers of two and u the log2 of the page's V scale, the
// weights of a row are 2^(s - r + u - R + 7) in f16, which reaches less far than a float: r + R is near the largest s + u, but goes
// down, and the sums up, for a page all of whose weights of a query lie 2^16 or more below it (where one token has nearly all of the
// weight and no value, as an attention sink does, such pages are the result). A weight is off by 2^-11 of itself or 2^-16 of its page's
// largest, whichever is more, down to pages 2^60 below the largest. The weights' sum is taken of 2^(s - r) in f32, r near the largest
// s. Scores may be of any size: R is kept from r on, since u would be lost in a sum with a score beyond 2^24.
//
// 128 rows of 500 to 8,000 tokens, 16 heads of 128 over 8: 175 to 177 us from a graph, 6.35 TB/s, 97 % of what a copy reaches (193 to
// 197 call after call, when power takes a tenth of the clock). Where the rows are few it is the way through one page that takes the
// time, 0.3 us a warp (0.7 us with sixteen heads), and the start and the join, 5 us.
#include <cooperative_groups.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "f32x2.cuh"
#include "kv8.h"
#include "pdl.cuh"
#include "sm100.cuh"

namespace omni {
namespace {

namespace cg = cooperative_groups;

// In powers of two: by how much a score may pass its reference before the sums are rescaled; what a weight at its reference is; between
// what the largest of a page's weights of a query may lie; by how much a reference may be lowered. A sum is at most
// 2^(kTop + kLowered) times a code (2^9) and the tokens (2^31) then, which a float holds.
constexpr float kSlack = 8.f, kLift = 7.f, kTop = kLift + kSlack, kFar = 9.f, kLowered = 60.f;
constexpr float kNegInf = -__builtin_huge_valf();
// References in front of all scores and weights: numbers, so that no difference is infinite minus infinite.
constexpr float kLowest = -3.402823466e38f, kLowestWeight = -1e30f;
constexpr float kNone = -1.f;  // what the sums of a row that is not attended to are to be multiplied by, in the first of its pieces' parts

constexpr int kWarps = 4;

template <int D>
constexpr int kPageBytes = 32 * D;  // K and V of one head
// CTAs that an SM's registers hold, and pages of a warp's ring, which fill its shared memory then
template <int NT>
constexpr int kPerSm = NT == 1 ? 4 : 3;
template <int D, int NT>
constexpr int kStages = (NT == 1 ? 3 : 4) * (128 / D);

template <int D, int NT>
constexpr int smem_bytes() {
  constexpr int ring = kWarps * kStages<D, NT> * kPageBytes<D>;
  constexpr int merge = (kWarps + 1) * NT * 8 * D * 4;
  return ring > merge ? ring : merge;
}

__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ uint4 lds16(uint32_t addr) {
  uint4 u;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(u.x), "=r"(u.y), "=r"(u.z), "=r"(u.w) : "r"(addr));
  return u;
}
__device__ __forceinline__ uint2 lds8(uint32_t addr) {
  uint2 u;
  asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(u.x), "=r"(u.y) : "r"(addr));
  return u;
}

// Four e4m3 (a word) as f16: bytes 0, 1 in lo, bytes 2, 3 in hi.
__device__ __forceinline__ void widen(uint32_t four, uint32_t& lo, uint32_t& hi) {
  asm("{\n.reg .b16 l, h;\nmov.b32 {l, h}, %2;\ncvt.rn.f16x2.e4m3x2 %0, l;\ncvt.rn.f16x2.e4m3x2 %1, h;\n}" : "=r"(lo), "=r"(hi) : "r"(four));
}

// An 8 x 8 matrix of 16-bit values, a row's pair a lane, transposed.
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

__device__ __forceinline__ uint32_t half2_of(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// Where 16-byte piece `col` of row `row` of a page lies in its stage: neighbouring rows' pieces in different banks.
template <int D>
__device__ __forceinline__ uint32_t piece_at(int row, int col) {
  return (uint32_t)(row * D + ((D == 128 ? col ^ (row & 7) : col ^ ((row >> 1) & 3)) << 4));
}

struct Part {  // of a query: reference of the scores, of the weights (from r on), sum of 2^(s - r), and what the weights' sums are to be multiplied by
  float r, R, l, f;
};
constexpr Part kNothing = {kLowest, kLowestWeight, 0.f, 0.f};
// Weight of summands under reference x when the largest reference is `top`.
__device__ __forceinline__ float weight_of(float x, float top) { return exp2_of(x - top); }
// 0 where nothing was attended to: all of the row's pages lie outside the cache.
__device__ __forceinline__ Part part_of(float r, float R, float l) { return Part{r, R, l, l == 0.f ? 0.f : exp2_of(R) / l}; }
__device__ __forceinline__ uint2 result_of(float4 v, float f) {
  const __nv_bfloat162 lo = __floats2bfloat162_rn(v.x * f, v.y * f), hi = __floats2bfloat162_rn(v.z * f, v.w * f);
  return make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
}

// How the work of a call is cut. Without pieces: a cluster a row and kv head (or part of its group), its warps taking turns. With
// pieces: rows are cut into pieces of about as many pages each as `room` CTAs would have if all pages were dealt out evenly
// (or a part of that); a row of one piece is finished by its CTA, the sums of others go to `parts` and `sums` for the second
// kernel. The cut follows from the rows' lengths alone, which every CTA adds up for itself.
struct Cut {
  int subgroups, per;  // parts of a group of query heads, heads of a part
  int room;            // 0: no pieces
  int least;           // pages of a piece
  Part* parts;         // [piece][kv head and part][per]
  float* sums;         // [piece][kv head and part][per][D]
};
constexpr int kCutRows = 1024;  // rows at most of a call in pieces

__device__ __forceinline__ int pages_of_row(const Kv8Attend& a, int row) {
  const int pos = __ldcg(a.pos + row);
  return pos < 0 ? 0 : min((pos >> 4) + 1, a.n_pages);
}

struct Piece {
  int row, index, count, pages;  // of the row's pieces, pages of each
  int before;                    // pieces of the rows in front
};
// The piece with this number, or (by_row) the first of this row; row = -1: there is none. Whole block, W warps.
template <int W>
__device__ __forceinline__ Piece find_piece(const Kv8Attend& a, const Cut& cut, int number, bool by_row) {
  __shared__ float sh_pages[W];
  __shared__ int sh_pieces[W];
  __shared__ Piece found;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int per = (a.rows + W * 32 - 1) / (W * 32), begin = min(a.rows, tid * per), end = min(a.rows, begin + per);
  float sum = 0.f;
  for (int r = begin; r < end; ++r) sum += (float)pages_of_row(a, r);
  sum = warp_add(sum);
  if (lane == 0) sh_pages[warp] = sum;
  if (tid == 0) found.row = -1;
  __syncthreads();
  sum = 0.f;
#pragma unroll
  for (int w = 0; w < W; ++w) sum += sh_pages[w];
  // the rounding of the sum is far below the hundredth
  const unsigned size = max((unsigned)cut.least, (unsigned)(sum * (float)(a.kv_heads * cut.subgroups) * (1.01f / (float)cut.room)) + 1u);
  const auto pieces_of = [&](int pages) { return pages <= (int)size ? 1 : (int)(((unsigned)pages + size - 1u) / size); };
  int mine = 0;
  for (int r = begin; r < end; ++r) mine += pieces_of(pages_of_row(a, r));
  int incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += up;
  }
  if (lane == 31) sh_pieces[warp] = incl;
  __syncthreads();
  int before = incl - mine;
#pragma unroll
  for (int w = 0; w < W; ++w) before += w < warp ? sh_pieces[w] : 0;
  if (by_row ? number >= begin && number < end : number >= before && number < before + mine)
    for (int r = begin; r < end; ++r) {
      const int pages = pages_of_row(a, r), n = pieces_of(pages);
      if (by_row ? r == number : number < before + n) {
        found = Piece{r, by_row ? 0 : number - before, n, (int)(((unsigned)pages + n - 1u) / n), before};
        break;
      }
      before += n;
    }
  __syncthreads();
  return found;
}

template <int D, int NT>
__global__ void __launch_bounds__(kWarps * 32, kPerSm<NT>) kv8_attend_kernel(const __grid_constant__ Kv8Attend a, const __grid_constant__ Cut cut, uint32_t* err) {
  constexpr int S = kStages<D, NT>, CW = D / 64;  // pieces of a key's row a lane holds
  constexpr int STEPS = D / 16;               // matrix instructions of K Q^T; as many of V^T P^T
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ Part parts[kWarps][NT * 8], joined[NT * 8];
  __shared__ float factor[8][NT * 8];  // of the sums of warps, then of CTAs
  grid_wait();
  grid_trigger();  // behind the wait: the second kernel, if there is one, looks at the rows' lengths before it waits itself
  const cg::cluster_group cluster = cg::this_cluster();
  const int ctas = cluster.num_blocks(), rank = cluster.block_rank();
  const int tid = threadIdx.x, lane = tid & 31, warp = warp_index(), g = lane >> 2, t = lane & 3;
  const int subgroups = cut.subgroups, groups = a.kv_heads * subgroups;
  const int unit = blockIdx.x / ctas, part = unit % groups, kh = part / subgroups, sub = part % subgroups;
  Piece piece{unit / groups, 0, 1, 0, 0};
  if (cut.room) {
    piece = find_piece<kWarps>(a, cut, unit / groups, false);
    if (piece.row < 0) return;
  }
  const int row = piece.row;
  const int group = a.q_heads / a.kv_heads, q0 = sub * cut.per, nq = min(cut.per, group - q0);
  const int head0 = kh * group + q0;
  bf16* const out = a.out + row * a.ldo + (int64_t)head0 * D;

  // queries: column n of a tile is query head head0 + n, lane t holds elements (D / 4) t .. of it; on their way before anything is known
  uint4 raw[NT][D / 32];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int j = 0; j < D / 32; ++j)
      raw[nt][j] = __ldcg(reinterpret_cast<const uint4*>(a.q + row * a.ldq + (int64_t)(head0 + min(nt * 8 + g, nq - 1)) * D + t * (D / 4)) + j);

  // the row's tokens and pages
  const int s_of = a.seq ? __ldcg(a.seq + row) : row, pos = __ldcg(a.pos + row);
  const bool named = s_of >= 0 && s_of < a.n_seqs;
  const int first = named ? __ldcg(a.indptr + s_of) : 0, last = named ? __ldcg(a.indptr + s_of + 1) : 0;
  int len = pos < 0 || pos == 0x7fffffff ? 0 : pos + 1;
  if (pos >= 0 && !(named && len > 0 && first >= 0 && last <= a.n_pages && (int64_t)last - first >= ((int64_t)len + 15) / 16)) {
    if (tid == 0) raise(err, kErrBadIndex);
    len = 0;
  }
  if (len == 0) {  // the same for every CTA of the cluster and every piece of the row
    if (rank == 0 && piece.index == 0)
      for (int i = tid; i < nq * (D / 8); i += kWarps * 32) *reinterpret_cast<uint4*>(out + i * 8) = make_uint4(0, 0, 0, 0);
    if (piece.count > 1 && tid < cut.per) cut.parts[(int64_t)(piece.before + piece.index) * groups * cut.per + part * cut.per + tid] = Part{0.f, 0.f, 0.f, kNone};
    return;
  }
  const int all = (len >> 4) + ((len & 15) != 0);
  const int page0 = piece.index * piece.pages, pages_n = piece.count > 1 ? max(0, min(piece.pages, all - page0)) : all;
  const int workers = ctas * kWarps, me = rank * kWarps + warp;
  const int mine = me < pages_n ? (pages_n - me + workers - 1) / workers : 0;
  const int32_t* const my_pages = a.pages + first + page0 + me;

  // pages and their scales, thirty-two at a time: lane i holds those of this warp's page 32 b + i
  const auto fetch_id = [&](int b) {
    const int i = b * 32 + lane;
    if (i >= mine) return 0;
    const int id = __ldcg(my_pages + (int64_t)i * workers);
    if (id >= 0 && id < a.kv_pages) return id;
    raise(err, kErrBadIndex);
    return -1;
  };
  const float2* const scales = reinterpret_cast<const float2*>(a.scales) + kh;
  int ids = fetch_id(0), ids_next = mine > 32 ? fetch_id(1) : 0;
  float2 sc = __ldcg(scales + (int64_t)max(ids, 0) * a.kv_heads), sc_next = sc;
  if (ids < 0) sc.x = -1.f;  // no tokens on it

  const uint32_t ring = sm100::smem_addr(smem) + warp * (S * kPageBytes<D>);
  const auto issue = [&](int i, int stage) {
    if (i < mine) {
      if ((i & 31) == 0 && i > 0) {
        ids = ids_next;
        sc_next = __ldcg(scales + (int64_t)max(ids, 0) * a.kv_heads);
        if (ids < 0) sc_next.x = -1.f;
        if (i + 32 < mine) ids_next = fetch_id(i / 32 + 1);
      }
      const int64_t id = max(__shfl_sync(0xffffffffu, ids, i & 31), 0);
      const uint8_t* const src = a.kv + (id * a.kv_heads + kh) * kPageBytes<D>;
      const uint32_t dst = ring + stage * kPageBytes<D>;
#pragma unroll
      for (int j = 0; j < D / 16; ++j) {
        const int piece = j * 32 + lane;
        copy16(dst + piece_at<D>(piece / (D / 16), piece % (D / 16)), src + piece * 16);
      }
    }
    copy_commit();
  };
#pragma unroll
  for (int i = 0; i < S - 1; ++i) issue(i, i);

  uint32_t qf[NT][STEPS][2];
  float unit_of[NT][2];  // scores of columns 2 t, 2 t + 1 in powers of two
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    float x[STEPS * 4];
#pragma unroll
    for (int j = 0; j < D / 32; ++j) unpack8v(nt * 8 + g < nq ? raw[nt][j] : make_uint4(0, 0, 0, 0), x + 8 * j);
    float top = 0.f;
#pragma unroll
    for (int j = 0; j < STEPS * 4; ++j) top = fmaxf(top, fabsf(x[j]) < __builtin_huge_valf() ? fabsf(x[j]) : 0.f);
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const int e = max((int)(__float_as_uint(top) >> 23) - 127, -112);  // largest in [2^14, 2^15) in f16
    const float up = __uint_as_float((uint32_t)(14 - e + 127) << 23), down = __uint_as_float((uint32_t)(e - 14 + 127) << 23);
#pragma unroll
    for (int j = 0; j < STEPS; ++j) qf[nt][j][0] = half2_of(x[4 * j] * up, x[4 * j + 1] * up), qf[nt][j][1] = half2_of(x[4 * j + 2] * up, x[4 * j + 3] * up);
    const float f = a.scale * 1.44269504088896340736f * down;
    unit_of[nt][0] = __shfl_sync(0xffffffffu, f, t * 8), unit_of[nt][1] = __shfl_sync(0xffffffffu, f, t * 8 + 4);
  }

  float r[NT][2], R[NT][2], l[NT][2], o[NT][STEPS][4];
  uint32_t lowered = 0;  // by how many powers of two at most R lies below the largest s + u, a byte a column
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    r[nt][0] = r[nt][1] = kLowest, R[nt][0] = R[nt][1] = kLowestWeight, l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
    for (int j = 0; j < STEPS; ++j) o[nt][j][0] = o[nt][j][1] = o[nt][j][2] = o[nt][j][3] = 0.f;
  }

  const uint32_t column = 0x11111111u << t;  // the lanes that share this one's columns
  int stage = 0;
  for (int i = 0; i < mine; ++i) {
    copy_wait<S - 2>();
    __syncwarp();  // every lane's pieces are there, and every lane is done with the stage that is filled next
    if ((i & 31) == 0 && i > 0) sc = sc_next;
    issue(i + S - 1, stage == 0 ? S - 1 : stage - 1);
    const uint32_t keys = ring + stage * kPageBytes<D>;
    stage = stage == S - 1 ? 0 : stage + 1;
    const float ks = __shfl_sync(0xffffffffu, sc.x, i & 31), vs = __shfl_sync(0xffffffffu, sc.y, i & 31);
    const int valid = ks < 0.f ? 0 : len - (page0 + me + i * workers) * 16;  // tokens from the page's first on
    if (valid <= 0) continue;
    const auto page = [&](auto part) {  // `part`: some of its tokens are none of the row's
      constexpr bool kPart = decltype(part)::value;
      float s[NT][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.f;
#pragma unroll
      for (int c = 0; c < CW; ++c) {
        const uint4 lo = lds16(keys + piece_at<D>(g, t * CW + c)), hi = lds16(keys + piece_at<D>(g + 8, t * CW + c));
        const uint32_t wl[4] = {lo.x, lo.y, lo.z, lo.w}, wh[4] = {hi.x, hi.y, hi.z, hi.w};
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          uint32_t a0, a1, a2, a3;
          widen(wl[w], a0, a2), widen(wh[w], a1, a3);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) sm100::mma_16816_f16(s[nt], a0, a1, a2, a3, qf[nt][c * 4 + w][0], qf[nt][c * 4 + w][1]);
        }
      }
      float lvs;
      asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(lvs) : "f"(vs));
      float to[NT][2];   // from scores above their reference to weights
      bool off = false;  // a score above its reference by more than kSlack, or a lane's largest weight of a column out of [2^-kFar, 2^kTop]
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[nt][e] *= ks * unit_of[nt][e & 1];
          if (kPart && g + (e & 2) * 4 >= valid) s[nt][e] = kNegInf;
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float most = fmaxf(s[nt][e], s[nt][e + 2]) - r[nt][e];
          to[nt][e] = lvs + kLift - R[nt][e];
          const float weight = most + to[nt][e];
          off |= most > kSlack || weight > kTop || (weight < -kFar && (!kPart || g < valid));
        }
      }
      if (__any_sync(0xffffffffu, off)) {
        bool go = false;  // is it more than a lane's part of a column that lies far below?
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float most = fmaxf(s[nt][e], s[nt][e + 2]) - r[nt][e], weight = most + to[nt][e];
            const uint32_t near = __ballot_sync(0xffffffffu, !(weight < -kFar));
            go |= most > kSlack || weight > kTop || (near & column) == 0;
          }
        if (__any_sync(0xffffffffu, go)) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              float m = fmaxf(s[nt][e], s[nt][e + 2]);
#pragma unroll
              for (int x = 4; x < 32; x <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, x));
              const float nr = fmaxf(r[nt][e], m), up = r[nt][e] - nr;
              l[nt][e] *= exp2_of(up);
              r[nt][e] = nr;
              const float was = fmaxf(R[nt][e] + up, kLowestWeight), top = m - nr + lvs, below = was - top;  // from the new r on
              const int at = 8 * (2 * nt + e);
              const float low = (float)(lowered >> at & 255);
              float nR = fmaxf(was, top);
              if (below > kFar + kLift && lvs > kNegInf) nR = was - fminf(floorf(below) - kSlack, kLowered - low);
              const float by = was - nR, f = exp2_of(by);
              R[nt][e] = nR, to[nt][e] = lvs + kLift - nR, lowered += (uint32_t)(int)fmaxf(by, -low) << at;
#pragma unroll
              for (int j = 0; j < STEPS; ++j) o[nt][j][e] *= f, o[nt][j][e + 2] *= f;
            }
        }
      }
      uint32_t p[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float above = s[nt][e] - r[nt][e & 1];
          l[nt][e & 1] += exp2_of(above);
          w[e] = exp2_of(above + to[nt][e & 1]);
        }
        p[nt][0] = transpose8(half2_of(w[0], w[1])), p[nt][1] = transpose8(half2_of(w[2], w[3]));
      }
      const uint32_t values = keys + 16 * D;
      constexpr int WORDS = D / 32;  // of a value's row that a lane holds: elements (D / 8) g ..
      uint32_t u[4][WORDS];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int tok = 2 * t + (k & 1) + (k >> 1) * 8;
        if constexpr (D == 128) {
          const uint4 v = lds16(values + piece_at<D>(tok, g));
          u[k][0] = v.x, u[k][1] = v.y, u[k][2] = v.z, u[k][3] = v.w;
        } else {
          const uint2 v = lds8(values + piece_at<D>(tok, g >> 1) + (g & 1) * 8);
          u[k][0] = v.x, u[k][1] = v.y;
        }
        if (kPart && tok >= valid) {  // what lies there may be NaN
#pragma unroll
          for (int w = 0; w < WORDS; ++w) u[k][w] = 0;
        }
      }
#pragma unroll
      for (int w = 0; w < WORDS; ++w)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          uint32_t a0, a1, a2, a3;
          widen(__byte_perm(u[0][w], u[1][w], half ? 0x7362 : 0x5140), a0, a1), widen(__byte_perm(u[2][w], u[3][w], half ? 0x7362 : 0x5140), a2, a3);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) sm100::mma_16816_f16(o[nt][w * 2 + half], a0, a1, a2, a3, p[nt][0], p[nt][1]);
        }
    };
    if (valid >= 16) page(std::false_type());
    else page(std::true_type());
  }

  // the warps' sums: o is [D / 8 bytes of lane g][column], a matrix instruction two neighbouring elements
  copy_wait<0>();
  __syncthreads();
  float* const sums = reinterpret_cast<float*>(smem);        // [warp][query][D]
  float* const total = sums + kWarps * NT * 8 * D;           // [query][D]
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int n = nt * 8 + 2 * t + e;
#pragma unroll
      for (int x = 4; x < 32; x <<= 1) l[nt][e] += __shfl_xor_sync(0xffffffffu, l[nt][e], x);
      if (n < nq) {
        if (g == 0) parts[warp][n] = Part{r[nt][e], R[nt][e] - kLift, l[nt][e], R[nt][e] + (float)(lowered >> 8 * (2 * nt + e) & 255) - kLift};
        float* const dst = sums + (warp * NT * 8 + n) * D + g * (D / 8);
#pragma unroll
        for (int j = 0; j < STEPS; j += 2)
          *reinterpret_cast<float4*>(dst + 2 * j) = make_float4(o[nt][j][e], o[nt][j][e + 2], o[nt][j + 1][e], o[nt][j + 1][e + 2]);
      }
    }
  __syncthreads();
  if (tid < nq) {
    float r_top = kLowest, R_top = kNegInf, l_sum = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) r_top = fmaxf(r_top, parts[w][tid].r);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) R_top = fmaxf(R_top, parts[w][tid].f + (parts[w][tid].r - r_top));  // as if no reference had been lowered
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float to_top = parts[w][tid].r - r_top;
      l_sum += parts[w][tid].l * exp2_of(to_top), factor[w][tid] = weight_of(parts[w][tid].R + to_top, R_top);
    }
    joined[tid] = part_of(r_top, R_top, l_sum);
  }
  __syncthreads();
  const int64_t at = ((int64_t)(piece.before + piece.index) * groups + part) * cut.per;
  if (piece.count > 1 && tid < nq) cut.parts[at + tid] = joined[tid];
#pragma unroll
  for (int k = 0; k < NT * 8 * (D / 4) / (kWarps * 32); ++k) {
    const int i = k * (kWarps * 32) + tid, n = i / (D / 4), d = i % (D / 4) * 4;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float f = factor[w][n];
      const float4 x = *reinterpret_cast<const float4*>(sums + (w * NT * 8 + n) * D + d);
      v.x += x.x * f, v.y += x.y * f, v.z += x.z * f, v.w += x.w * f;
    }
    if (n >= nq) continue;
    if (piece.count > 1) *reinterpret_cast<float4*>(cut.sums + (at + n) * D + d) = v;
    else if (ctas == 1) *reinterpret_cast<uint2*>(out + n * D + d) = result_of(v, joined[n].f);
    else *reinterpret_cast<float4*>(total + n * D + d) = v;
  }
  if (ctas == 1) return;
  cluster.sync();
  const int begin = rank * (kWarps * 32) + tid, end = nq * (D / 4), step = ctas * (kWarps * 32);
  float4 x[8];
  const auto fetch = [&](int i) {  // the CTAs' sums, all under way before the first is used
#pragma unroll
    for (int c = 0; c < 8; ++c)
      if (c < ctas && i < end) x[c] = *reinterpret_cast<const float4*>(cluster.map_shared_rank(total, c) + i * 4);
  };
  fetch(begin);
  {
    const int n = tid >> 3, c = tid & 7;
    Part p = kNothing;
    if (n < nq && c < ctas) p = *cluster.map_shared_rank(&joined[n], c);
    float r_top = p.r;
#pragma unroll
    for (int x = 1; x < 8; x <<= 1) r_top = fmaxf(r_top, __shfl_xor_sync(0xffffffffu, r_top, x));
    const float to_top = p.r - r_top, R = p.R + to_top;
    float R_top = R;
#pragma unroll
    for (int x = 1; x < 8; x <<= 1) R_top = fmaxf(R_top, __shfl_xor_sync(0xffffffffu, R_top, x));
    float l_sum = p.l * exp2_of(to_top);
#pragma unroll
    for (int x = 1; x < 8; x <<= 1) l_sum += __shfl_xor_sync(0xffffffffu, l_sum, x);
    if (n < nq) factor[c][n] = part_of(r_top, R_top, l_sum).f * weight_of(R, R_top);
  }
  __syncthreads();
  for (int i = begin; i < end; i += step) {
    if (i != begin) fetch(i);
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int c = 0; c < 8; ++c) {
      if (c >= ctas) break;
      const float f = factor[c][i / (D / 4)];
      v.x += x[c].x * f, v.y += x[c].y * f, v.z += x[c].z * f, v.w += x[c].w * f;
    }
    *reinterpret_cast<uint2*>(out + i * 4) = result_of(v, 1.f);
  }
  cluster.sync();  // no CTA leaves while another reads its sums
}

// The sums of a row's pieces, in an order of their own. A CTA a row and query head; D / 4 lanes a piece, as many pieces at a time as
// there are such groups of lanes, each with two under way and references of its own. It stands behind the last CTAs of the kernel in
// front, so it has to be small as well as short. One row of 60,000 tokens, 8 kv heads (74 pieces a row and head), both kernels: 28.2
// us; with four warps 29.7, with sixteen and four pieces under way 28.8, with which 24 rows in pieces of 2 heads of 64 take 30 us
// instead of 23.7.
constexpr int kJoinWarps = 8;
template <int D>
__global__ void __launch_bounds__(kJoinWarps * 32, 4) kv8_join_kernel(const __grid_constant__ Kv8Attend a, const __grid_constant__ Cut cut) {
  constexpr int LANES = D / 4, GROUPS = kJoinWarps * 32 / LANES, AHEAD = 2;
  __shared__ float4 v_of[GROUPS][LANES];
  __shared__ Part part_of_group[GROUPS];
  const int tid = threadIdx.x, group = a.q_heads / a.kv_heads;
  const int row = blockIdx.x / a.q_heads, head = blockIdx.x % a.q_heads, kh = head / group, n = head % group % cut.per;
  const int groups = a.kv_heads * cut.subgroups, part = kh * cut.subgroups + head % group / cut.per;
  const Piece piece = find_piece<kJoinWarps>(a, cut, row, true);
  grid_wait();  // on every path: with this kernel the one in front has ended
  grid_trigger();
  if (piece.count < 2) return;
  const int64_t step = (int64_t)groups * cut.per, at = (piece.before * (int64_t)groups + part) * cut.per + n;
  const float4* const parts = reinterpret_cast<const float4*>(cut.parts) + at;
  const int g = tid / LANES, d = tid % LANES;
  Part mine = kNothing;
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  const float first = __ldcg(parts).w;
  for (int c = g; c < piece.count; c += AHEAD * GROUPS) {
    float4 p[AHEAD], x[AHEAD];
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      const int at_piece = c + k * GROUPS;
      p[k] = make_float4(kNothing.r, kNothing.R, 0.f, 0.f), x[k] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (at_piece < piece.count) p[k] = __ldcg(parts + at_piece * step), x[k] = __ldcg(reinterpret_cast<const float4*>(cut.sums + (at + at_piece * step) * D) + d);
    }
    float r = mine.r;
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) r = fmaxf(r, p[k].x);
    mine.l *= exp2_of(mine.r - r), mine.R += mine.r - r, mine.r = r;
    float R = mine.R;
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) R = fmaxf(R, p[k].y + (p[k].x - r));
    const float old = weight_of(mine.R, R);
    mine.R = R;
    v.x *= old, v.y *= old, v.z *= old, v.w *= old;
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      const float to_top = p[k].x - r, f = weight_of(p[k].y + to_top, R);
      mine.l += p[k].z * exp2_of(to_top);
      v.x += x[k].x * f, v.y += x[k].y * f, v.z += x[k].z * f, v.w += x[k].w * f;
    }
  }
  if (first == kNone) return;  // its zeros are there
  v_of[g][d] = v;
  if (d == 0) part_of_group[g] = mine;
  __syncthreads();
  if (g > 0) return;
  Part all = {kLowest, kNegInf, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < GROUPS; ++i) all.r = fmaxf(all.r, part_of_group[i].r);
#pragma unroll
  for (int i = 0; i < GROUPS; ++i) all.R = fmaxf(all.R, part_of_group[i].R + (part_of_group[i].r - all.r));
  v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
  for (int i = 0; i < GROUPS; ++i) {
    const Part p = part_of_group[i];
    const float4 x = v_of[i][d];
    const float to_top = p.r - all.r, f = weight_of(p.R + to_top, all.R);
    all.l += p.l * exp2_of(to_top);
    v.x += x.x * f, v.y += x.y * f, v.z += x.z * f, v.w += x.w * f;
  }
  *reinterpret_cast<uint2*>(a.out + row * a.ldo + (int64_t)head * D + d * 4) = result_of(v, part_of(all.r, all.R, all.l).f);
}

template <int D, int NT>
cudaError_t go(const Kv8Attend& a, Cut cut, int ctas, int sm_count, cudaMemPool_t pool, uint32_t* err, cudaStream_t s) {
  constexpr int smem = smem_bytes<D, NT>();
  cudaError_t e = allow_large<kv8_attend_kernel<D, NT>>(smem);
  if (e != cudaSuccess) return e;
  const int groups = a.kv_heads * cut.subgroups;
  unsigned units = (unsigned)a.rows * groups;
  void* scratch = nullptr;
  if (cut.room) {
    const int64_t pieces = a.rows + cut.room / groups + 1;
    const size_t parts = (size_t)pieces * groups * cut.per;
    e = cudaMallocFromPoolAsync(&scratch, parts * (sizeof(Part) + D * sizeof(float)), pool, s);
    if (e != cudaSuccess) return e;
    cut.parts = static_cast<Part*>(scratch), cut.sums = reinterpret_cast<float*>(cut.parts + parts);
    units = (unsigned)(pieces * groups);
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(units * ctas), cfg.blockDim = dim3(kWarps * 32), cfg.dynamicSmemBytes = smem, cfg.stream = s;
  cudaLaunchAttribute attr[2] = {};
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ctas, attr[0].val.clusterDim.y = 1, attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr, cfg.numAttrs = cut.room ? 1 : 2;  // with pieces there is an allocation in front, not a kernel
  e = cudaLaunchKernelEx(&cfg, kv8_attend_kernel<D, NT>, a, cut, err);
  if (cut.room) {
    if (e == cudaSuccess) e = launch_pdl(kv8_join_kernel<D>, dim3((unsigned)a.rows * a.q_heads), dim3(kJoinWarps * 32), 0, s, a, cut);
    const cudaError_t done = cudaFreeAsync(scratch, s);
    if (e == cudaSuccess) e = done;
  }
  return e;
}

}  // namespace

cudaError_t launch_kv8_attend(const Kv8Attend& a, int sm_count, cudaMemPool_t pool, uint32_t* err, cudaStream_t s) {
  const int group = a.q_heads / a.kv_heads;
  Cut cut = {};
  cut.subgroups = (group + 15) / 16, cut.per = (group + cut.subgroups - 1) / cut.subgroups;
  const int64_t units = (int64_t)a.rows * a.kv_heads * cut.subgroups;
  const int64_t held = a.n_pages / std::max(a.n_seqs, 1);  // pages a sequence, as far as the host knows
  const int64_t at_once = (int64_t)sm_count * (cut.per > 8 ? kPerSm<2> : kPerSm<1>);
  // Either more CTAs a row as long as all run at once, to a page a warp; or, where they do not, as many as leave each some 40 pages
  // of 4 KB; or, where there are more pages than clusters of eight in little over a wave read evenly, pieces, which need room beside
  // the CTAs that every row has. Measured, us, cluster of 1 / 2 / 4 / 8 | pieces (heads of 128, groups of 2, the third: of 4):
  //   rows x kv heads, tokens
  //   1 x 8,   777              9.0 /  7.7 /  6.3 /  5.5 | 9.7
  //   1 x 8,   60,000           451 /  228 /  117 /   61 | 28
  //   12 x 8,  28,000 - 34,000  258 /  164 /  133 /  157 | 130 - 139
  //   20 x 8,  500 - 5,000       44 /   30 /   29 /   31 | 27
  //   64 x 8,  2,000 - 8,000    128 /  123 /  116 /  120 |
  //   128 x 8, 500 - 8,000      207 /  194 /  187 /  206 |  (the clock at rest: 175 with 4)
  //   256 x 8, 100 - 2,000       98 /  103 /  133 /  211 |
  int ctas = 1;
  if (a.rows <= kCutRows && units * 6 <= at_once && held >= 256) {
    cut.room = (int)(at_once - units), cut.least = 32;
  } else {
    while (ctas < 8 && ((units * 2 * ctas <= at_once && held >= 16 && held >= 8 * ctas) || held * a.head_dim >= 80 * 128 * ctas)) ctas *= 2;
  }
  const auto run = [&](auto d, auto nt) { return go<decltype(d)::value, decltype(nt)::value>(a, cut, ctas, sm_count, pool, err, s); };
  using std::integral_constant;
  if (a.head_dim == 128) return cut.per > 8 ? run(integral_constant<int, 128>(), integral_constant<int, 2>()) : run(integral_constant<int, 128>(), integral_constant<int, 1>());
  if (a.head_dim == 64) return cut.per > 8 ? run(integral_constant<int, 64>(), integral_constant<int, 2>()) : run(integral_constant<int, 64>(), integral_constant<int, 1>());
  return cudaErrorInvalidValue;
}

}  // namespace omni
