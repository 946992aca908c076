// Prefill attention over a batch's own bf16 pages (the 8-bit cache, read back),
// on the Blackwell tensor cores (tcgen05 + TMEM + TMA).
//
// Where the scratch pages of a request lie one after another, as page_plan puts
// them, a tile of keys is one TMA box per 64 dims, elsewhere a box per page. One
// CTA = two 128-row query tiles of one head, each with
// its own softmax warpgroup. Per query tile and tile of 64 keys:
//   S  = Q K^T    tcgen05.mma 128 x 64, fp32 in TMEM
//   P  = exp2(S * scale - m) by 4 warps, one thread per row, stored as bf16 in
//        TMEM (32 columns)
//   O += P V      tcgen05.mma with A = P from TMEM, V MN-major from shared memory
// Why this shape. Shared memory feeds the tensor core 128 bytes a cycle. With P
// written to and read from shared memory, as the kernel over the cache itself
// does (fmha_tc.cu), that port takes 1.75 times as long as the MMAs; with P in
// TMEM 1.25 times. Tiles of 128 keys would read Q half as often, but then P has
// to lie over S (TMEM is 512 columns, O takes 256), the next S has to wait for
// the PV product, and the chain S - softmax - PV leaves the tensor core idle
// half the time. Here S of the next tile is issued as soon as the softmax warps
// have the present one in registers, and PV runs under the next tile's softmax.
// Measured, 1024 queries over 8192 keys of 32 heads, read-back (7.5 us) included:
// 150 us on the same inputs again, 152 on changing ones (846 TFLOP/s, 51 % of the
// measured GEMM rate; 128 of 148 SMs have a CTA); the kernel over the cache itself
// on the same pages 173, 128-key tiles 155. A turn of 64 keys for both tiles takes
// 2300 cycles, 1280 of them tensor work: the softmax warps of the two tiles share a
// scheduler and its exponential unit and lengthen one another. Two threads per row
// (165 us), packed FMAs (150) and polynomials for some of the exponentials (153 to
// 159) did not help.
// P is rounded to bf16, which costs about as much again as the output's own
// rounding (1.35 times the error of fp32 weights against 64 bits): A and B of one
// product have the same type, and V's rows keep their exponents, for which f16 has
// no range. The row sum takes the weights before that rounding.
// Warps: 0 TMA producer, 1 TMEM allocator and MMA issuer, 2-5 / 6-9 softmax and
// epilogue of query tile 0 / 1. Every mbarrier wait is bounded; on timeout the
// CTA records an error, drains its copies and MMAs, frees TMEM and exits.
#include <cudaTypedefs.h>

#include <algorithm>
#include <mutex>
#include <stdexcept>
#include <string>

#include "../gemm/tcgen05.cuh"
#include "../kernels.h"

namespace mbx {
namespace {

constexpr int D = 128;
constexpr int BQ = 128;    // rows per query tile
constexpr int QT = 2;      // query tiles per CTA
constexpr int BKV = 64;    // keys per tile
constexpr int NS = 4;      // K and V stages
constexpr int PAGE = 16;
constexpr int kTilePages = BKV / PAGE;
constexpr int kThreads = 320;
constexpr int kQChunk = BQ * 64 * 2;      // 64 dims of a tile's rows: 16 KB
constexpr int kQBytes = 2 * kQChunk;
constexpr int kKVChunk = BKV * 64 * 2;
constexpr int kKVBytes = 2 * kKVChunk;
// The running output is rescaled only when a row's maximum grows by more than
// 2^8: weights stay at most 2^8, harmless in fp32 and bf16.
constexpr float kRescaleThreshold = 8.f;

struct PagesArgs {
  __nv_bfloat16* o;      // [T, nq, D]
  const int* cu_q;       // [R + 1]
  const int* kv_len;     // [R]
  const int* table;      // [R, cols]: scratch pages
  const int2* tiles;     // (request, q offset): 256-row query-tile pairs
  float* part_o;         // splits > 1: [T, nq, splits, D]
  float* part_lse;       //             [T, nq, splits]
  int splits, cols, nq, nkv, pages;  // pages: of K, behind which V's lie
  int placed;            // table entries outside [0, placed) name no page
  float scale_log2;
  uint32_t* err;
  uint64_t timeout_ns;
};

struct Smem {
  static constexpr int kQ = 0;
  static constexpr int kK = kQ + QT * kQBytes;
  static constexpr int kV = kK + NS * kKVBytes;
  static constexpr int kBar = kV + NS * kKVBytes;
  static constexpr int kTotal = kBar + 256 + 1024;
};

MBX_DEVICE void set_err(uint32_t* err, uint32_t code, volatile int* abort) {
  *abort = 1;
  if (err) atomicCAS(err, 0u, code);
}

// tc::mbar_wait for waits that last: each try suspends the thread for up to 10 us
// unless the phase completes. The issuing threads wait most of the time and
// share their scheduler with softmax warps, which a tight loop would slow down.
MBX_DEVICE bool mbar_wait_long(uint64_t* bar, uint32_t parity, volatile int* abort, uint64_t timeout_ns) {
  auto try_wait = [&] {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(tc::smem_u32(bar)), "r"(parity), "r"(10000u)
        : "memory");
    return ok != 0;
  };
  if (try_wait()) return true;
  const uint64_t t0 = globaltimer_ns();
  while (!try_wait())
    if (*abort || globaltimer_ns() - t0 > timeout_ns) return false;
  return true;
}

// D[tmem] (+)= A[tmem, bf16 pairs in 32-bit columns] * B[smem].
MBX_DEVICE void mma_bf16_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(tmem_d),
      "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}

__global__ void __launch_bounds__(kThreads, 1)
    fmha_pages_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmKV,
                      const __grid_constant__ CUtensorMap tmKV1, PagesArgs a) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + Smem::kBar);
  uint64_t* q_full = bars;
  uint64_t* k_full = bars + 1;           // [NS]
  uint64_t* k_empty = k_full + NS;       // [NS]
  uint64_t* v_full = k_empty + NS;       // [NS]
  uint64_t* v_empty = v_full + NS;       // [NS]
  uint64_t* s_full = v_empty + NS;       // [QT]
  uint64_t* s_empty = s_full + QT;       // [QT]
  uint64_t* p_full = s_empty + QT;       // [QT]
  uint64_t* pv_done = p_full + QT;       // [QT]
  uint64_t* mma_done = pv_done + QT;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(mma_done + 1);
  volatile int* abort = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_wait();
  const int2 tile = a.tiles[blockIdx.x];
  const int r = tile.x, qoff = tile.y;
  const int head = blockIdx.y;
  const int kvh = head / (a.nq / a.nkv);
  const int q_begin = a.cu_q[r], q_len = a.cu_q[r + 1] - q_begin;
  const int L = min(max(a.kv_len[r], 0), a.cols * PAGE);
  const int pos0 = L - q_len;  // position of the request's first query
  // the scratch pages of four pages in a row (the producer's), from page p on
  auto ids_of = [&](int p) {
    const int* row = a.table + (int64_t)r * a.cols;
    const int last = a.cols - 1;
    return last < 0 ? make_int4(-1, -1, -1, -1)
                    : make_int4(row[min(p, last)], row[min(p + 1, last)], row[min(p + 2, last)], row[min(p + 3, last)]);
  };
  int4 next_ids = make_int4(-1, -1, -1, -1);
  if (warp == 0) next_ids = ids_of(0);  // where the CTA's keys begin at 0: ahead of what follows
  int rows_t[QT], kvend_t[QT], n_t[QT];  // per query tile: rows, keys it sees, key tiles
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    rows_t[t] = max(0, min(BQ, q_len - qoff - t * BQ));
    kvend_t[t] = rows_t[t] > 0 ? max(0, min(L, pos0 + qoff + t * BQ + rows_t[t])) : 0;
    n_t[t] = (kvend_t[t] + BKV - 1) / BKV;
  }
  const int n_all = max(n_t[0], n_t[1]);
  const int last_page = (max(kvend_t[0], kvend_t[1]) - 1) / PAGE;  // of this CTA's keys
  const int split = blockIdx.z;
  const int per = (n_all + a.splits - 1) / a.splits;
  const int tb = min(n_all, split * per), te = min(n_all, tb + per);
  const int n_cta = te - tb;
  int nt[QT];
#pragma unroll
  for (int t = 0; t < QT; ++t) nt[t] = max(0, min(te, n_t[t]) - tb);

  if (threadIdx.x == 0) {
    tc::mbar_init(q_full, 1);
    for (int i = 0; i < NS; ++i) {
      tc::mbar_init(&k_full[i], 1);
      tc::mbar_init(&k_empty[i], 1);
      tc::mbar_init(&v_full[i], 1);
      tc::mbar_init(&v_empty[i], 1);
    }
    for (int t = 0; t < QT; ++t) {
      tc::mbar_init(&s_full[t], 1);
      tc::mbar_init(&s_empty[t], 4);
      tc::mbar_init(&p_full[t], 4);
      tc::mbar_init(&pv_done[t], 1);
    }
    tc::mbar_init(mma_done, 1);
    *abort = 0;
    tc::fence_barrier_init();
  }
  if (warp == 1) {
    tc::tmem_alloc(tmem_slot, 512);
    tc::tmem_relinquish();
  }
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  auto tS = [&](int t) { return tmem + (uint32_t)(t * BKV); };
  auto tP = [&](int t) { return tmem + (uint32_t)(QT * BKV + t * (BKV / 2)); };
  auto tO = [&](int t) { return tmem + 256u + (uint32_t)(t * D); };

  if (warp == 0) {
    // ------------------------------------------------------------------ producer
    if (tc::elect_one()) {
      int issued = 0;
      if (n_cta > 0) {
        tc::mbar_arrive_expect_tx(q_full, QT * kQBytes);
        for (int t = 0; t < QT; ++t)
          for (int c = 0; c < 2; ++c)
            tc::tma_load_3d(smem + Smem::kQ + t * kQBytes + c * kQChunk, &tmQ, q_full, c * 64, head,
                            q_begin + qoff + t * BQ);
      }
      // A tile whose pages all hold keys and lie in a row is one box per 64 dims;
      // in the last one the pages behind the last are that page again (masked keys
      // have to be finite, and what follows in the scratch is another request's).
      // A page that the table does not place reads as zeros (a coordinate behind
      // the scratch), and the error word says so.
      auto load = [&](uint8_t* dst, const int4& id, int first, uint64_t* bar, int p) {
        const bool row = p + kTilePages - 1 <= last_page && id.x >= 0 && id.w < a.placed && id.y == id.x + 1 &&
                         id.z == id.x + 2 && id.w == id.x + 3;
        for (int c = 0; c < 2; ++c) {
          if (row) {
            tc::tma_load_4d(dst + c * kKVChunk, &tmKV, bar, c * 64, 0, kvh, first + id.x);
          } else {
            for (int i = 0; i < kTilePages; ++i) {
              const int k = min(i, last_page - p);
              const int page = k == 0 ? id.x : k == 1 ? id.y : k == 2 ? id.z : id.w;
              const bool there = page >= 0 && page < a.placed;
              if (!there && a.err) atomicCAS(a.err, 0u, 24u);
              tc::tma_load_4d(dst + c * kKVChunk + i * (PAGE * 128), &tmKV1, bar, c * 64, 0, kvh,
                              there ? first + page : 2 * a.pages);
            }
          }
        }
      };
      if (tb > 0) next_ids = ids_of(tb * kTilePages);
      for (int j = 0; j < n_cta && !*abort; ++j, ++issued) {
        const int s = j % NS;
        const int p = (tb + j) * kTilePages;
        const int4 ids = next_ids;
        next_ids = ids_of(p + kTilePages);
        const uint32_t parity = ((j / NS) & 1) ^ 1;
        if (!mbar_wait_long(&k_empty[s], parity, abort, a.timeout_ns)) {
          set_err(a.err, 21, abort);
          break;
        }
        tc::mbar_arrive_expect_tx(&k_full[s], kKVBytes);
        load(smem + Smem::kK + s * kKVBytes, ids, 0, &k_full[s], p);
        if (!mbar_wait_long(&v_empty[s], parity, abort, a.timeout_ns)) {
          set_err(a.err, 21, abort);
          volatile int never = 0;
          tc::mbar_wait(&k_full[s], (j / NS) & 1, &never, 200000000ull);  // the K copy just issued
          break;
        }
        tc::mbar_arrive_expect_tx(&v_full[s], kKVBytes);
        load(smem + Smem::kV + s * kKVBytes, ids, a.pages, &v_full[s], p);
      }
      // copies in flight land before the CTA leaves
      volatile int never = 0;
      if (n_cta > 0) tc::mbar_wait(q_full, 0, &never, 200000000ull);
      for (int j = max(0, issued - NS); j < issued; ++j) {
        tc::mbar_wait(&k_full[j % NS], (j / NS) & 1, &never, 200000000ull);
        tc::mbar_wait(&v_full[j % NS], (j / NS) & 1, &never, 200000000ull);
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA issuer
    if (tc::elect_one()) {
      constexpr uint32_t idS = tc::idesc_bf16_f32_major(BQ, BKV, 0, 0);  // Q K-major, K K-major
      constexpr uint32_t idO = tc::idesc_bf16_f32_major(BQ, D, 0, 1);    // P in TMEM, V MN-major
      bool ok = true;
      auto wait = [&](uint64_t* bar, int parity) {
        if (ok && !mbar_wait_long(bar, parity, abort, a.timeout_ns)) {
          set_err(a.err, 22, abort);
          ok = false;
        }
        tc::tc_fence_after();
        return ok;
      };
      // descriptors of the operands' beginnings; an offset adds its 16-byte units
      const uint64_t dQ = tc::sw128_desc(tc::smem_u32(smem + Smem::kQ), 16, 1024);
      const uint64_t dK = tc::sw128_desc(tc::smem_u32(smem + Smem::kK), 16, 1024);
      const uint64_t dV = tc::sw128_desc(tc::smem_u32(smem + Smem::kV), kKVChunk, 1024);
      auto issue_s = [&](int t, int j) {
        const uint64_t q = dQ + t * (kQBytes >> 4), k = dK + (j % NS) * (kKVBytes >> 4);
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk)
          tc::mma_bf16(tS(t), q + (((kk >> 2) * kQChunk + (kk & 3) * 32) >> 4),
                       k + (((kk >> 2) * kKVChunk + (kk & 3) * 32) >> 4), idS, kk > 0 ? 1u : 0u);
        tc::mma_commit(&s_full[t]);
      };
      if (n_cta > 0 && wait(q_full, 0) && wait(&k_full[0], 0)) {
#pragma unroll
        for (int t = 0; t < QT; ++t)
          if (nt[t] > 0) issue_s(t, 0);
        tc::mma_commit(&k_empty[0]);
      }
      // Each tile's products in the order in which its softmax lets them go: P_{j-1}
      // is stored before S_j is read out. Tile 0's come first, so the two tiles
      // settle half a turn apart, one's products under the other's softmax.
      for (int j = 0; ok && j <= n_cta; ++j) {
        const bool has_v = j >= 1, has_k = j + 1 < n_cta;
        const int vs = (j + NS - 1) % NS, ks = (j + 1) % NS;
        if (has_v && !wait(&v_full[vs], ((j - 1) / NS) & 1)) break;
        const uint64_t v = dV + vs * (kKVBytes >> 4);
#pragma unroll
        for (int t = 0; t < QT; ++t) {
          if (has_v && j - 1 < nt[t] && wait(&p_full[t], (j - 1) & 1)) {
#pragma unroll
            for (int kk = 0; kk < BKV / 16; ++kk)
              // P: 16 keys = 8 columns; V: 16 key rows of 128 B, the dims' halves a chunk apart
              mma_bf16_ts(tO(t), tP(t) + kk * 8, v + (kk * 16 * 128 >> 4), idO, (j > 1 || kk > 0) ? 1u : 0u);
            tc::mma_commit(&pv_done[t]);
          }
          if (has_k && t == 0 && !wait(&k_full[ks], ((j + 1) / NS) & 1)) break;
          if (has_k && j + 1 < nt[t] && wait(&s_empty[t], j & 1)) issue_s(t, j + 1);
        }
        if (!ok) break;
        if (has_v) tc::mma_commit(&v_empty[vs]);
        if (has_k) tc::mma_commit(&k_empty[ks]);
      }
      tc::mma_commit(mma_done);
      volatile int never = 0;
      tc::mbar_wait(mma_done, 0, &never, 200000000ull);
    }
  } else {
    // ------------------------------------------------------------------ softmax / epilogue
    const int t = (warp - 2) >> 2;
    const int quad = warp & 3;
    const int row = quad * 32 + lane;
    const uint32_t lane_addr = (uint32_t)(quad * 32) << 16;
    const int q_pos = pos0 + qoff + t * BQ + row;
    const float sc = a.scale_log2;
    const int my_n = nt[t];
    float m = -INFINITY, l = 0.f;
    bool ok = true;
    for (int j = 0; j < my_n; ++j) {
      if (!tc::mbar_wait(&s_full[t], j & 1, abort, a.timeout_ns)) {
        if (lane == 0) set_err(a.err, 23, abort);
        ok = false;
        break;
      }
      tc::tc_fence_after();
      uint32_t v[BKV];
#pragma unroll
      for (int c = 0; c < BKV / 32; ++c)
        tc::tmem_ld_32x32b_x32(tS(t) + lane_addr + c * 32, *reinterpret_cast<uint32_t(*)[32]>(&v[c * 32]));
      tc::tmem_ld_wait();
      tc::tc_fence_before();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(&s_empty[t]);
      const int lim = min(q_pos + 1, kvend_t[t]) - (tb + j) * BKV;  // the row sees the tile's first lim keys
      if (lim < BKV) {
#pragma unroll
        for (int i = 0; i < BKV; ++i)
          if (i >= lim) v[i] = __float_as_uint(-INFINITY);
      }
      // Row maximum of the raw scores over 8 independent partial ones, scaled
      // once: sc > 0, so max(x * sc) = max(x) * sc.
      float m8[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) m8[k] = __uint_as_float(v[k]);
#pragma unroll
      for (int i = 8; i < BKV; ++i) m8[i & 7] = fmaxf(m8[i & 7], __uint_as_float(v[i]));
#pragma unroll
      for (int k = 4; k > 0; k >>= 1)
#pragma unroll
        for (int q = 0; q < k; ++q) m8[q] = fmaxf(m8[q], m8[q + k]);
      const float mx = m8[0] * sc;
      const bool grow = mx > m + kRescaleThreshold || (m == -INFINITY && mx != -INFINITY);
      const float m_new = grow ? mx : m;
      const float corr = (m == -INFINITY || !grow) ? 1.f : tc::ex2(m - m_new);
      const float neg = m_new == -INFINITY ? 0.f : -m_new;  // a row without keys so far: 2^(-inf) = 0
      float s8[8] = {};
      uint32_t pk[BKV / 2];
#pragma unroll
      for (int i = 0; i < BKV; i += 2) {
        const float p0 = tc::ex2(fmaf(__uint_as_float(v[i]), sc, neg));
        const float p1 = tc::ex2(fmaf(__uint_as_float(v[i + 1]), sc, neg));
        s8[(i >> 1) & 7] += p0 + p1;
        const __nv_bfloat162 h2 = __floats2bfloat162_rn(p0, p1);
        pk[i / 2] = *reinterpret_cast<const uint32_t*>(&h2);
      }
#pragma unroll
      for (int k = 4; k > 0; k >>= 1)
#pragma unroll
        for (int q = 0; q < k; ++q) s8[q] += s8[q + k];
      l = l * corr + s8[0];
      m = m_new;
      if (j > 0) {  // P_{j-1} V is complete before P is overwritten and O rescaled
        if (!tc::mbar_wait(&pv_done[t], (j - 1) & 1, abort, a.timeout_ns)) {
          if (lane == 0) set_err(a.err, 23, abort);
          ok = false;
          break;
        }
        tc::tc_fence_after();
      }
      tc::tmem_st_32x32b_x32(tP(t) + lane_addr, pk);
      if (j > 0 && __any_sync(0xffffffffu, corr < 1.f)) {
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {
          uint32_t tt[32];
          tc::tmem_ld_32x32b_x32(tO(t) + lane_addr + c * 32, tt);
          tc::tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 32; ++i) tt[i] = __float_as_uint(__uint_as_float(tt[i]) * corr);
          tc::tmem_st_32x32b_x32(tO(t) + lane_addr + c * 32, tt);
        }
      }
      tc::tmem_st_wait();
      tc::tc_fence_before();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(&p_full[t]);
    }
    const int rows_here = rows_t[t];
    const int64_t out_row = (int64_t)(q_begin + qoff + t * BQ + row) * a.nq + head;
    if (ok && my_n > 0 && !tc::mbar_wait(&pv_done[t], (my_n - 1) & 1, abort, a.timeout_ns)) {
      if (lane == 0) set_err(a.err, 23, abort);
      ok = false;
    }
    if (ok) {
      tc::tc_fence_after();
      const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);  // NaN stays
#pragma unroll
      for (int c = 0; c < D / 32; ++c) {
        uint32_t tt[32];
        if (my_n > 0) {
          tc::tmem_ld_32x32b_x32(tO(t) + lane_addr + c * 32, tt);
          tc::tmem_ld_wait();
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) tt[i] = 0u;
        }
        if (row < rows_here) {
          if (a.splits == 1) {
            __nv_bfloat16* dst = a.o + out_row * D + c * 32;
            float f[8];
#pragma unroll
            for (int g = 0; g < 4; ++g) {
#pragma unroll
              for (int i = 0; i < 8; ++i) f[i] = __uint_as_float(tt[g * 8 + i]) * inv;
              *reinterpret_cast<uint4*>(dst + g * 8) = pack_from<__nv_bfloat16>(f);
            }
          } else {
            float* dst = a.part_o + (out_row * a.splits + split) * D + c * 32;
#pragma unroll
            for (int g = 0; g < 8; ++g)
              *reinterpret_cast<float4*>(dst + g * 4) =
                  make_float4(__uint_as_float(tt[g * 4]) * inv, __uint_as_float(tt[g * 4 + 1]) * inv,
                              __uint_as_float(tt[g * 4 + 2]) * inv, __uint_as_float(tt[g * 4 + 3]) * inv);
          }
        }
      }
      if (a.splits > 1 && row < rows_here)
        a.part_lse[out_row * a.splits + split] = l == 0.f ? -INFINITY : m + log2f(l);
    }
  }

  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  if (warp == 1) tc::tmem_dealloc(tmem, 512);
}

// ---------------------------------------------------------------- host side
PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    cudaDriverEntryPointQueryResult q;
    void* p = nullptr;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
  });
  if (!fn) throw std::runtime_error("cuTensorMapEncodeTiled unavailable (no CUDA driver)");
  return fn;
}

CUtensorMap encode(const void* base, int rank, const cuuint64_t* dims, const cuuint64_t* strides_bytes,
                   const cuuint32_t* box) {
  if (((uint64_t)base & 15) != 0) throw std::runtime_error("fmha: tensor base must be 16-byte aligned");
  CUtensorMap m;
  const cuuint32_t estr[4] = {1, 1, 1, 1};
  const CUresult res = encode_fn()(&m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, rank, const_cast<void*>(base), dims,
                                   strides_bytes, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                   CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                                   CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (res != CUDA_SUCCESS) throw std::runtime_error("fmha: cuTensorMapEncodeTiled failed " + std::to_string((int)res));
  return m;
}

}  // namespace

void prefill_attention_pages_launch(const void* q, const void* kv, void* o, const int* cu_q, const int* kv_len,
                                    const int* table, int cols, const int* tiles, int n_tiles, int T, int nq, int nkv,
                                    int pages, int placed, float scale, int splits, float* part_o, float* part_lse,
                                    uint32_t* err, cudaStream_t s) {
  if (n_tiles == 0 || T == 0) return;
  if (nq % nkv != 0) throw std::runtime_error("fmha: nq must be a multiple of nkv");
  if (splits > 1 && (!part_o || !part_lse)) throw std::runtime_error("fmha: split-KV needs scratch buffers");
  // Q: [T, nq, D] -> dims {D, nq, T}, box {64, 1, 128}
  cuuint64_t qd[3] = {(cuuint64_t)D, (cuuint64_t)nq, (cuuint64_t)T};
  cuuint64_t qs[2] = {(cuuint64_t)D * 2, (cuuint64_t)nq * D * 2};
  const cuuint32_t qb[3] = {64, 1, BQ};
  const CUtensorMap tq = encode(q, 3, qd, qs, qb);
  // K's pages, then V's: [2 pages, nkv, PAGE, D] -> dims {D, PAGE, nkv, 2 pages}, boxes of a tile's pages and of one
  auto page_map = [&](cuuint32_t n) {
    cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)PAGE, (cuuint64_t)nkv, 2 * (cuuint64_t)pages};
    cuuint64_t str[3] = {(cuuint64_t)D * 2, (cuuint64_t)PAGE * D * 2, (cuuint64_t)nkv * PAGE * D * 2};
    const cuuint32_t box[4] = {64, PAGE, 1, n};
    return encode(kv, 4, dims, str, box);
  };
  const CUtensorMap tkv = page_map(kTilePages), tkv1 = page_map(1);
  PagesArgs a{static_cast<__nv_bfloat16*>(o), cu_q, kv_len, table, reinterpret_cast<const int2*>(tiles), part_o,
              part_lse, std::max(1, splits), cols, nq, nkv, pages, placed, scale * 1.4426950408889634f, err,
              2000000000ull};
  static SmemLimit limit;
  limit.ensure((const void*)fmha_pages_kernel, Smem::kTotal);
  launch_k(fmha_pages_kernel, dim3(n_tiles, nq, a.splits), dim3(kThreads), Smem::kTotal, s, tq, tkv, tkv1, a);
  MBX_CUDA_CHECK(cudaGetLastError());
  if (a.splits > 1) attn_combine_launch(part_o, part_lse, (int64_t)T * nq, a.splits, o, s);
}

}  // namespace mbx
