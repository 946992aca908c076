// The paged KV cache in 8 bits: writing it, reading it back, and attention of
// one new token per request over it (head_dim 128, pages of 16 tokens).
//
// A cached row x (one token, one kv head) is held as e4m3 numbers with one
// power-of-two scale:
//   e = the smallest integer with max|x_i| <= 448 * 2^e, at least -117
//   values_i = round_to_nearest_even_e4m3(x_i / 2^e),  exps = e + 127
// and stands for values_i * 2^e. e4m3 is a floating format, so a scale finer
// than a power of two would buy at most one exponent of range and no
// accuracy, while a power of two makes every scaling exact: a stored number
// below 2^128 is exact in bf16 and in fp32 products, and which e4m3 number a
// value rounds to does not depend on a division. Elements that are not finite
// are stored as NaN and do not take part in the maximum.
#include <cuda_fp8.h>

#include <algorithm>
#include <stdexcept>
#include <string>

#include "../common.cuh"
#include "../kernels.h"

namespace mbx {
namespace {

constexpr int D = 128;
constexpr int PAGE = 16;
constexpr int kMinExp = -117;  // 2^-9 * 2^-117 = 2^-126: every stored number is a normal fp32 / bf16 number or zero

// Rows on their way into the cache are held 2^8 smaller: a normalised and
// rotated k of finite inputs may lie beyond fp32 (below 16 * 2^128, though).
constexpr int kDown = 8;
constexpr float kSmaller = 1.f / (1 << kDown);

// A row's exponent from the largest magnitude of its finite elements, held
// 2^kDown smaller: 448 = 1.75 * 2^8.
MBX_DEVICE int row_exp(float top) {
  const uint32_t b = __float_as_uint(top);
  const int e = (int)(b >> 23) - 127 - 8 + kDown + ((b & 0x7fffffu) > 0x600000u ? 1 : 0);
  return max(e, kMinExp);
}

// 2^e for e in [-126, 127].
MBX_DEVICE float pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

MBX_DEVICE bool finite(float x) { return (__float_as_uint(x) & 0x7f800000u) != 0x7f800000u; }

// Two e4m3 numbers from lo and hi (lo in the low byte); what is not finite becomes NaN.
MBX_DEVICE uint32_t e4m3x2(float lo, float hi) {
  uint16_t r;
  const float nan = __uint_as_float(0x7fffffffu);
  lo = finite(lo) ? lo : nan;
  hi = finite(hi) ? hi : nan;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}

// e4m3 x 2 (the low or high half of w) to f16 x 2, exact.
MBX_DEVICE uint32_t f16x2_of(uint32_t w, int half) {
  uint32_t r;
  const uint16_t h = (uint16_t)(half ? w >> 16 : w);
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(h));
  return r;
}

// The fp32 number whose further rounding to fewer bits (22 or less) equals
// rounding x itself: x cut to 24 bits (fewer below fp32's normal range, whose
// last, 2^-149, is still far below what is kept of a row), the last one set if
// anything was cut.
MBX_DEVICE float round_to_odd(double x) {
  const float f = __double2float_rz(x);
  return (double)f != x ? __uint_as_float(__float_as_uint(f) | 1u) : f;
}

MBX_DEVICE float finite_abs(float x) { return finite(x) ? fabsf(x) : 0.f; }

// ---------------------------------------------------------------- append
struct AppendArgs {
  const __nv_bfloat16* qkv;  // [T, (nq + 2 nkv) * D]
  const int* pos;            // [T]
  const float* cos_sin;      // [max_pos, D]: cos(64) | sin(64)
  const int64_t* slots;      // [T]: block * PAGE + offset; negative or past the cache: not written
  __nv_bfloat16* q_out;      // [T, nq, D]
  uint8_t *kv, *vv;          // [blocks, nkv, PAGE, D] e4m3
  uint8_t *ke, *ve;          // [blocks, nkv, PAGE], row strides below
  int64_t ke_sb, ke_sh, ve_sb, ve_sh;
  const __nv_bfloat16 *q_norm, *k_norm;  // [D] or nullptr
  double eps;
  int64_t T, n_slots;
  int max_pos, nq, nkv;
};

// A row (one head of one token) takes eight lanes: lane i of them holds dims 8i
// .. 8i + 7 and their rotation partners 8i + 64 .. 8i + 71, two 16-byte loads,
// so a warp streams four rows at once and a row's maximum is three shuffles.
struct Row {
  uint4 lo, hi;
  MBX_DEVICE void load(const __nv_bfloat16* src, int i) {
    lo = ld_v4(src + 8 * i);
    hi = ld_v4(src + 64 + 8 * i);
  }
};
struct Angles {
  float c[8], s[8];
  MBX_DEVICE void load(const float* cs, int i) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const float4 x = *reinterpret_cast<const float4*>(cs + 8 * i + 4 * k);
      const float4 y = *reinterpret_cast<const float4*>(cs + 64 + 8 * i + 4 * k);
      c[4 * k] = x.x, c[4 * k + 1] = x.y, c[4 * k + 2] = x.z, c[4 * k + 3] = x.w;
      s[4 * k] = y.x, s[4 * k + 1] = y.y, s[4 * k + 2] = y.z, s[4 * k + 3] = y.w;
    }
  }
};
template <typename F>
MBX_DEVICE F eighth_sum(F v) {  // over a row's eight lanes
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// A row, held 2^kDown smaller, rounded into the cache at dst and *exp.
MBX_DEVICE void store_e4m3(const float (&x)[8], const float (&y)[8], uint8_t* dst, uint8_t* exp, int i, bool keep) {
  float top = 0.f;
#pragma unroll
  for (int k = 0; k < 8; ++k) top = fmaxf(top, fmaxf(finite_abs(x[k]), finite_abs(y[k])));
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  const int e = row_exp(top);
  const float inv = pow2(kDown - e);
  uint2 lo, hi;
  lo.x = e4m3x2(x[0] * inv, x[1] * inv) | e4m3x2(x[2] * inv, x[3] * inv) << 16;
  lo.y = e4m3x2(x[4] * inv, x[5] * inv) | e4m3x2(x[6] * inv, x[7] * inv) << 16;
  hi.x = e4m3x2(y[0] * inv, y[1] * inv) | e4m3x2(y[2] * inv, y[3] * inv) << 16;
  hi.y = e4m3x2(y[4] * inv, y[5] * inv) | e4m3x2(y[6] * inv, y[7] * inv) << 16;
  if (!keep) return;
  *reinterpret_cast<uint2*>(dst + 8 * i) = lo;
  *reinterpret_cast<uint2*>(dst + 64 + 8 * i) = hi;
  if (i == 0) *exp = (uint8_t)(e + 127);
}

constexpr int kAppendWarps = 8;
constexpr int kMaxTokens = 32;  // of a CTA that writes k and v

// Bound by the rows' stream: 316 MB in 64 us (76 % of the measured copy rate) for
// 8005 tokens of 64 q and 2 x 8 kv heads; 8.3 us for 1024 of 32 + 2 x 8, where a
// warp per head and 4-byte loads took 12. The search for later tokens of the same
// slot is quadratic: tokens^2 / 32 slots read above 16384 tokens, and with pages
// scattered over the cache most of them compared with a CTA's own (65536 tokens of
// 8 + 2 x 1 heads: 209 us with pages in a row, 519 scattered, of 54 for the bytes).
// CTAs 0 .. kv_ctas - 1 write k and v of `tokens` tokens each, the others rotate
// q: a warp takes `passes` times four heads of one token, whose angles it loads
// once. k is normalised and rotated in 64 bits, so that the stored byte is the
// one of the real number: two fp32 products and a sum would land on the other
// side of a rounding border now and then.
template <bool kNorm>
__global__ void __launch_bounds__(kAppendWarps * 32) append_kernel(AppendArgs a, int kv_ctas, int tokens, int passes) {
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sub = lane >> 3, i = lane & 7;
  const int heads = a.nq + 2 * a.nkv;
  auto angles_at = [&](int64_t t) { return a.cos_sin + (int64_t)min(max(a.pos[t], 0), a.max_pos - 1) * D; };
  if ((int)blockIdx.x >= kv_ctas) {
    const int per = (a.nq + 4 * passes - 1) / (4 * passes);  // tasks per token
    const int64_t task = (int64_t)(blockIdx.x - kv_ctas) * kAppendWarps + warp;
    const int64_t t = task / per;
    if (t >= a.T) return;
    const int h0 = (int)(task % per) * 4 * passes + sub;
    const __nv_bfloat16* src = a.qkv + t * heads * D;
    Row row;
    row.load(src + (int64_t)min(h0, a.nq - 1) * D, i);
    Angles g;
    g.load(angles_at(t), i);
#pragma unroll 1
    for (int p = 0; p < passes; ++p) {
      const int h = h0 + 4 * p;
      float x[8] = {}, y[8] = {};
      unpack_add<__nv_bfloat16>(row.lo, x);
      unpack_add<__nv_bfloat16>(row.hi, y);
      if (p + 1 < passes) row.load(src + (int64_t)min(h + 4, a.nq - 1) * D, i);
      if (kNorm) {
        float ss = 0.f, w[8] = {}, v[8] = {};
#pragma unroll
        for (int k = 0; k < 8; ++k) ss += x[k] * x[k] + y[k] * y[k];
        const float r = rsqrtf(eighth_sum(ss) * (1.f / D) + (float)a.eps);
        unpack_add<__nv_bfloat16>(ld_v4(a.q_norm + 8 * i), w);
        unpack_add<__nv_bfloat16>(ld_v4(a.q_norm + 64 + 8 * i), v);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          x[k] = x[k] * r * w[k];
          y[k] = y[k] * r * v[k];
        }
      }
      float u[8], v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        u[k] = x[k] * g.c[k] - y[k] * g.s[k];
        v[k] = y[k] * g.c[k] + x[k] * g.s[k];
      }
      if (h < a.nq) {
        __nv_bfloat16* dst = a.q_out + (t * a.nq + h) * D;
        *reinterpret_cast<uint4*>(dst + 8 * i) = pack_from<__nv_bfloat16>(u);
        *reinterpret_cast<uint4*>(dst + 64 + 8 * i) = pack_from<__nv_bfloat16>(v);
      }
    }
    return;
  }
  __shared__ int64_t slot_of[kMaxTokens];
  __shared__ int taken[kMaxTokens];  // the slot is a later token's as well, which is stored instead
  const int64_t t0 = (int64_t)blockIdx.x * tokens;
  const int n = (int)min((int64_t)tokens, a.T - t0);
  const int rows = n * 2 * a.nkv;  // token by token: its k heads, its v heads
  // four rows a warp and pass; what lies behind the last row repeats it unstored
  auto place = [&](int r, int& j, int& h) {
    const int x = min(r, rows - 1);
    j = x / (2 * a.nkv);
    h = x - j * 2 * a.nkv;
  };
  int j, h, r = warp * 4 + sub;
  place(r, j, h);
  Row row;
  row.load(a.qkv + ((t0 + j) * heads + a.nq + h) * D, i);
  if ((int)threadIdx.x < n) {
    const int64_t s = a.slots[t0 + threadIdx.x];
    slot_of[threadIdx.x] = s >= 0 && s < a.n_slots ? s : -1;
    taken[threadIdx.x] = 0;
  }
  __syncthreads();
  if (t0 + 1 < a.T) {
    int64_t lo = slot_of[0], hi = lo;
    for (int k = 1; k < n; ++k) {
      lo = min(lo, slot_of[k]);
      hi = max(hi, slot_of[k]);
    }
    for (int64_t u = t0 + 1 + threadIdx.x; u < a.T; u += blockDim.x) {
      const int64_t s = a.slots[u];
      if (s < lo || s > hi || s < 0) continue;
      for (int k = 0; k < n; ++k)
        if (slot_of[k] == s && u > t0 + k) taken[k] = 1;
    }
    __syncthreads();
  }
#pragma unroll 1
  for (int r0 = 0; r0 < rows; r0 += kAppendWarps * 4) {
    const int64_t t = t0 + j, slot = slot_of[j];
    const bool keep = r0 + r < rows && slot >= 0 && !taken[j];
    const bool is_k = h < a.nkv;
    const int kh = is_k ? h : h - a.nkv;
    float x[8] = {}, y[8] = {};
    unpack_add<__nv_bfloat16>(row.lo, x);
    unpack_add<__nv_bfloat16>(row.hi, y);
    if (r0 + kAppendWarps * 4 < rows) {
      place(r0 + kAppendWarps * 4 + r, j, h);
      row.load(a.qkv + ((t0 + j) * heads + a.nq + h) * D, i);
    }
    if (__any_sync(0xffffffffu, is_k)) {
      Angles g;
      g.load(angles_at(t), i);
      double rs = 1.0;
      float w[8] = {}, v[8] = {};
      if (kNorm) {
        double ss = 0.0;
#pragma unroll
        for (int k = 0; k < 8; ++k) ss += (double)x[k] * x[k] + (double)y[k] * y[k];
        rs = 1.0 / sqrt(eighth_sum(ss) * (1.0 / D) + a.eps);
        unpack_add<__nv_bfloat16>(ld_v4(a.k_norm + 8 * i), w);
        unpack_add<__nv_bfloat16>(ld_v4(a.k_norm + 64 + 8 * i), v);
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const double p = kNorm ? rs * w[k] * x[k] : (double)x[k], q = kNorm ? rs * v[k] * y[k] : (double)y[k];
        const float px = round_to_odd((p * g.c[k] - q * g.s[k]) * kSmaller);
        const float py = round_to_odd((q * g.c[k] + p * g.s[k]) * kSmaller);
        x[k] = is_k ? px : x[k] * kSmaller;
        y[k] = is_k ? py : y[k] * kSmaller;
      }
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) x[k] *= kSmaller, y[k] *= kSmaller;  // exact: bf16's smallest step is 2^-133, fp32's 2^-149
    }
    const int64_t blk = slot / PAGE;
    const int off = (int)(slot % PAGE);
    store_e4m3(x, y, (is_k ? a.kv : a.vv) + ((blk * a.nkv + kh) * PAGE + off) * D,
               is_k ? a.ke + blk * a.ke_sb + kh * a.ke_sh + off : a.ve + blk * a.ve_sb + kh * a.ve_sh + off, i, keep);
  }
}

// ---------------------------------------------------------------- read
struct ReadArgs {
  const uint8_t *kv, *vv, *ke, *ve;
  int64_t ke_sb, ke_sh, ve_sb, ve_sh;
  const int* block_table;  // [R, max_blocks], row stride bt_s
  const int* out_table;    // [R, max_blocks], row stride ot_s, or nullptr (page i of request r at r * max_blocks + i)
  const int* kv_len;       // [R]
  int64_t bt_s, ot_s;
  __nv_bfloat16 *k_out, *v_out;  // [out_pages, nkv, PAGE, D]
  int64_t out_pages;
  int max_blocks, nkv, num_blocks;
};

// 16 e4m3 numbers to bf16, times 2^e (exact), one 32-byte store.
MBX_DEVICE void emit16(const uint4& w, float scale, __nv_bfloat16* dst) {
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
  float f[16];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t h = f16x2_of(u[i >> 1], i & 1);
    const float2 p = __half22float2(*reinterpret_cast<const __half2*>(&h));
    f[2 * i] = p.x * scale;
    f[2 * i + 1] = p.y * scale;
  }
  const uint4 a = pack_from<__nv_bfloat16>(f), b = pack_from<__nv_bfloat16>(f + 8);
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(dst), "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w),
               "r"(b.x), "r"(b.y), "r"(b.z), "r"(b.w)
               : "memory");
}

// 258 bytes in, 512 out per token and kv head; 6.5 TB/s, 99 % of the measured
// copy rate, for 37 requests up to 8192 tokens of 8 kv heads (a thread per 16
// elements of one page's head: 81 %).
// One warp per (page, kv head): ten loads in flight a lane, lane l the 16
// elements of row l / 8 (of four at a time) from 16 (l % 8). Rows behind the
// length are written as zeros, so that whatever reads whole pages never meets
// what an earlier user of the page left there.
constexpr int kReadWarps = 8;
__global__ void __launch_bounds__(kReadWarps * 32) read_pages_kernel(ReadArgs a, int tasks) {
  pdl_wait();
  const int task = blockIdx.x * kReadWarps + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (task >= tasks) return;
  const int page = task / a.nkv, h = task - page * a.nkv;
  const int r = page / a.max_blocks, i = page - r * a.max_blocks;
  const int L = a.kv_len[r];
  const int blk = a.block_table[r * a.bt_s + i];
  const int64_t to = a.out_table ? a.out_table[r * a.ot_s + i] : page;
  if (i * PAGE >= L || to < 0 || to >= a.out_pages) return;
  const int live = blk >= 0 && blk < a.num_blocks ? L - i * PAGE : 0;  // rows that count
  const int64_t src = live > 0 ? ((int64_t)blk * a.nkv + h) * PAGE * D + lane * 16 : 0;
  const uint4 ke = live > 0 ? ld_v4(a.ke + blk * a.ke_sb + h * a.ke_sh) : make_uint4(0, 0, 0, 0);
  const uint4 ve = live > 0 ? ld_v4(a.ve + blk * a.ve_sb + h * a.ve_sh) : make_uint4(0, 0, 0, 0);
  uint4 k[4], v[4];
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const bool on = c * 4 + (lane >> 3) < live;
    k[c] = on ? ld_v4(a.kv + src + c * 512) : make_uint4(0, 0, 0, 0);
    v[c] = on ? ld_v4(a.vv + src + c * 512) : make_uint4(0, 0, 0, 0);
  }
  const int64_t dst = (to * a.nkv + h) * PAGE * D + lane * 16;
  const uint32_t kw[4] = {ke.x, ke.y, ke.z, ke.w}, vw[4] = {ve.x, ve.y, ve.z, ve.w};
  const int byte = (lane >> 3) * 8;
  auto scale = [&](uint32_t w, int c) {
    return c * 4 + (lane >> 3) < live ? __uint_as_float(((w >> byte) & 0xffu) << 23) : 0.f;
  };
#pragma unroll
  for (int c = 0; c < 4; ++c) emit16(k[c], scale(kw[c], c), a.k_out + dst + c * 512);
#pragma unroll
  for (int c = 0; c < 4; ++c) emit16(v[c], scale(vw[c], c), a.v_out + dst + c * 512);
}

// ---------------------------------------------------------------- decode
// Attention of one query row per request. The G = nq / nkv query heads that
// share a kv head are the columns of the tensor-core tiles: per page of 16
// keys, S^T = K Q^T (16 keys x 8 heads) and O^T += V^T P^T (128 dims x 8
// heads) as m16n8k16 f16 MMAs with fp32 sums.
//  * e4m3 is exact in f16, and the order of the contracted dimension is free:
//    lane (g, t) = (lane / 4, lane % 4) of a K fragment takes 16 contiguous
//    bytes of its rows g and g + 8, and Q is laid out to match. V fragments
//    pair two keys per register; a lane takes the same 16 dims of four keys
//    and pairs them with byte permutes.
//  * q is scaled per head by a power of two to [2^14, 2^15) before it becomes
//    f16: elements down to 2^-28 of the head's largest keep all their bits.
//  * softmax in base 2 with a running maximum m per head; the row sum takes the
//    weights 2^(s - m) in fp32. The value exponents join the weights of the
//    product: w = 2^(s - m) * 2^(ve + d) in f16, the integer d per head such that
//    the largest w lies between 2^10 and 2^15. d follows mv, the running maximum
//    of s + ve: what a key contributes to this head, not how large its value row
//    is. So keys that contribute down to 2^-24 of the largest keep 11 bits (bf16
//    would keep 8), and a row that the head ignores costs the others nothing,
//    whatever its exponent. The maxima only move when a page exceeds one by more
//    than 2^4. Weights below 2^-126 of the largest so far are zero, as fp32 has
//    none, and stay out of mv. (2^(s - m + ve + d) as an exponential of its own: 64 requests
//    of 4096 keys 101 -> 102 us, with 16 heads per kv head 131 -> 138.)
MBX_DEVICE float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

MBX_DEVICE void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

MBX_DEVICE uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

MBX_DEVICE uint32_t pack_f16(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

struct Kv8DecodeArgs {
  const __nv_bfloat16* q;  // [B, nq, D]
  const uint8_t *kv, *vv, *ke, *ve;
  int64_t ke_sb, ke_sh, ve_sb, ve_sh;
  __nv_bfloat16* o;        // [B, nq, D]
  float* part;             // partials of pairs that span CTAs [grid][2][heads][D], then their (m, l)
  int* counters;           // [grid] arrivals, zero between launches
  const int* kv_len;       // [B]
  const int* block_table;  // [B, max_blocks], row stride bt_s
  int64_t bt_s;
  int B, max_blocks, num_blocks, nq, nkv;
  float scale_log2;
};

constexpr float kTopWeight = 11.f;  // log2 of the largest weight w when the maxima move, rounded down
constexpr float kSlack = 4.f;       // log2 of what may exceed a maximum before it moves: w <= 2^15, inside f16

// Where a fetched page's 16-byte chunks lie in shared memory. The reader of a
// K chunk (row r, chunk c) is lane (g, t) = (r % 8, c % 4), of a V chunk lane
// (c, r % 8 / 2), one of its four chunks each; the exclusive ors spread the
// writes (8 chunks of a row at once) and the reads over all banks.
MBX_DEVICE uint32_t k_place(int row, int ch) {
  const int slot = (row >> 3) * 2 + (ch >> 2);
  return slot * 512 + ((((row & 7) * 4 + (ch & 3)) ^ ((ch >> 2) << 2)) << 4);
}
MBX_DEVICE uint32_t v_place(int row, int ch) {
  const int slot = (row >> 3) * 2 + (row & 1), t = (row & 7) >> 1;
  return slot * 512 + ((t * 8 + (ch ^ (2 * t))) << 4);
}

// One warp's running state over the pages of one (request, kv head); NT tiles
// of 8 query heads. Of tile n, lane (g, t) holds heads 8n + 2t and 8n + 2t + 1
// at dims 16g..16g+15 (o[n][i][0], [2]: dims 16g + 2i, 16g + 2i + 1 of the
// first head; [1], [3]: of the second).
template <int NT>
struct HeadState {
  uint32_t qf[NT][8][2];
  float qs[NT][2];  // softmax scale * log2(e) * the power of two taken out of q
  float o[NT][8][4];
  float m[NT][2], l[NT][2];  // l: this lane's keys only
  float mv[NT][2];
  int d23[NT][2];  // d, at the place of an fp32 number's exponent

  // This lane's elements of q [G, D] (heads behind G: zeros), in two steps, so
  // that the loads can be issued ahead of their use.
  struct Query {
    uint4 w[NT][4];
    MBX_DEVICE void load(const __nv_bfloat16* q, int G, int lane) {
      const int g = lane >> 2, t = lane & 3;
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int c = 0; c < 4; ++c)
          w[n][c] = n * 8 + g < G ? ld_v4(q + (n * 8 + g) * D + (t + 4 * (c >> 1)) * 16 + (c & 1) * 8)
                                  : make_uint4(0, 0, 0, 0);
    }
  };
  MBX_DEVICE void begin(const Query& q, float scale_log2, int lane) {
    const int t = lane & 3;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float x[2][16];
      float top = 0.f;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        float f[8] = {};
        unpack_add<__nv_bfloat16>(q.w[n][c], f);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          x[c >> 1][(c & 1) * 8 + i] = f[i];
          top = fmaxf(top, fabsf(f[i]));
        }
      }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const int e = max((int)(__float_as_uint(top) >> 23) - 127, -112);
      const float up = pow2(14 - e);
#pragma unroll
      for (int ks = 0; ks < 8; ++ks) {
        const float* f = &x[ks >> 2][(ks & 3) * 4];
        qf[n][ks][0] = pack_f16(f[0] * up, f[1] * up);
        qf[n][ks][1] = pack_f16(f[2] * up, f[3] * up);
      }
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        qs[n][c] = scale_log2 * pow2(__shfl_sync(0xffffffffu, e, (2 * t + c) * 4) - 14);
        m[n][c] = mv[n][c] = -INFINITY;
        l[n][c] = 0.f;
        d23[n][c] = 0;
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) o[n][i][0] = o[n][i][1] = o[n][i][2] = o[n][i][3] = 0.f;
    }
  }

  // Two pages at once (independent chains of tensor-core work), as fetched into
  // shared memory: K (k_place), V (v_place), then the exponents of the 16 keys
  // and of the 16 values. A lane takes K rows g and g + 8, chunks t and t + 4,
  // and chunk g of V's rows 2t, 2t + 1, 2t + 8, 2t + 9. Only a page's first
  // live[p] keys count.
  MBX_DEVICE void pages(const uint8_t* const (&src)[2], const int (&live)[2], int lane) {
    constexpr int P = 2;
    const int g = lane >> 2, t = lane & 3;
    float s[P][NT][4], s2[P][NT][4];  // halves of the sum: a shorter chain
    uint4 k[P][4];
#pragma unroll
    for (int p = 0; p < P; ++p)
#pragma unroll
      for (int c = 0; c < 4; ++c) k[p][c] = *reinterpret_cast<const uint4*>(src[p] + k_place(g + 8 * (c >> 1), t + 4 * (c & 1)));
#pragma unroll
    for (int p = 0; p < P; ++p)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[p][n][i] = s2[p][n][i] = 0.f;
#pragma unroll
    for (int ks = 0; ks < 8; ++ks)
#pragma unroll
      for (int p = 0; p < P; ++p) {
        const uint4 &w0 = k[p][ks >> 2], &w8 = k[p][2 + (ks >> 2)];
        const uint32_t r0 = (ks & 3) == 0 ? w0.x : (ks & 3) == 1 ? w0.y : (ks & 3) == 2 ? w0.z : w0.w;
        const uint32_t r8 = (ks & 3) == 0 ? w8.x : (ks & 3) == 1 ? w8.y : (ks & 3) == 2 ? w8.z : w8.w;
        const uint32_t af[4] = {f16x2_of(r0, 0), f16x2_of(r8, 0), f16x2_of(r0, 1), f16x2_of(r8, 1)};
#pragma unroll
        for (int n = 0; n < NT; ++n) mma_f16((ks & 1) ? s2[p][n] : s[p][n], af, qf[n][ks][0], qf[n][ks][1]);
      }
    int vx[P][2];
    bool grow = false;
#pragma unroll
    for (int p = 0; p < P; ++p)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const uint8_t* e = src[p] + 4096 + g + 8 * r;
        const bool on = g + 8 * r < live[p];
        vx[p][r] = ((int)e[16] - 127) << 23;
        const float ve = (float)(vx[p][r] >> 23);
        const float kf = __uint_as_float((uint32_t)e[0] << 23);
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const float x = on ? (s[p][n][2 * r + c] + s2[p][n][2 * r + c]) * (kf * qs[n][c]) : -INFINITY;
            s[p][n][2 * r + c] = x;
            grow |= x > m[n][c] + kSlack || x + ve > mv[n][c] + kSlack;
          }
      }
    if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float corr[2], vc[2];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float nm = m[n][c];
#pragma unroll
          for (int p = 0; p < P; ++p) nm = fmaxf(nm, fmaxf(s[p][n][c], s[p][n][2 + c]));
#pragma unroll
          for (int off = 4; off < 32; off <<= 1) nm = fmaxf(nm, __shfl_xor_sync(0xffffffffu, nm, off));
          float nv = mv[n][c];
#pragma unroll
          for (int p = 0; p < P; ++p)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              const float x = s[p][n][2 * r + c];
              nv = x - nm >= -126.f ? fmaxf(nv, x + (float)(vx[p][r] >> 23)) : nv;
            }
#pragma unroll
          for (int off = 4; off < 32; off <<= 1) nv = fmaxf(nv, __shfl_xor_sync(0xffffffffu, nv, off));
          corr[c] = vc[c] = 1.f;
          if (nm != -INFINITY) {
            const int old = d23[n][c] >> 23, nd = __float2int_rd(nm - nv + kTopWeight);
            const float down = m[n][c] - nm;
            corr[c] = ex2(down);
            vc[c] = m[n][c] == -INFINITY ? 0.f : ex2(down + (float)(nd - old));
            m[n][c] = nm;
            mv[n][c] = nv;
            d23[n][c] = nd << 23;
          }
          l[n][c] *= corr[c];
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          o[n][i][0] *= vc[0];
          o[n][i][1] *= vc[1];
          o[n][i][2] *= vc[0];
          o[n][i][3] *= vc[1];
        }
      }
    }
    uint32_t pf[P][NT][2];
#pragma unroll
    for (int p = 0; p < P; ++p)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          float w[2];
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const float x = ex2(s[p][n][2 * r + c] - (m[n][c] == -INFINITY ? 0.f : m[n][c]));
            l[n][c] += x;
            // x 2^(ve + d) by its exponent; below the smallest normal number: zero, or close to it
            const int y = max(__float_as_int(x) + vx[p][r] + d23[n][c], 0);
            w[c] = x > 0.f ? __int_as_float(y) : 0.f;
          }
          pf[p][n][r] = transpose8x8(pack_f16(w[0], w[1]));
        }
      }
#pragma unroll
    for (int p = 0; p < P; ++p) {
      uint4 v[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) v[c] = *reinterpret_cast<const uint4*>(src[p] + 2048 + v_place(2 * t + (c & 1) + 8 * (c >> 1), g));
      if (live[p] < PAGE) {  // rows behind the length may hold anything: 0 * NaN would not be 0
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (2 * t + (i & 1) + 8 * (i >> 1) >= live[p]) v[i] = make_uint4(0, 0, 0, 0);
      }
      const uint32_t vw[4][4] = {{v[0].x, v[0].y, v[0].z, v[0].w},
                                 {v[1].x, v[1].y, v[1].z, v[1].w},
                                 {v[2].x, v[2].y, v[2].z, v[2].w},
                                 {v[3].x, v[3].y, v[3].z, v[3].w}};
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t sel = (i & 1) ? 0x7362u : 0x5140u;
        const uint32_t a01 = __byte_perm(vw[0][i >> 1], vw[1][i >> 1], sel);
        const uint32_t a89 = __byte_perm(vw[2][i >> 1], vw[3][i >> 1], sel);
        const uint32_t af[4] = {f16x2_of(a01, 0), f16x2_of(a01, 1), f16x2_of(a89, 0), f16x2_of(a89, 1)};
#pragma unroll
        for (int n = 0; n < NT; ++n) mma_f16(o[n][i], af, pf[p][n][0], pf[p][n][1]);
      }
    }
  }

  MBX_DEVICE void end() {
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) l[n][c] += __shfl_xor_sync(0xffffffffu, l[n][c], off);
  }
};

// ---- the work's division
// One CTA per SM. The pages of all (request, kv head) pairs form one list, pairs
// one after another; every warp of the grid takes an equal run of it, whatever
// the lengths are (they live on the device, so a captured graph adapts too). A
// pair's pages inside one warp's run are a segment of that warp:
//   * a pair that lies in one warp's run is finished by the warp alone;
//   * otherwise each warp leaves a partial state (m, l, O) in shared memory, and
//     the CTA merges its warps' partials, in order, into the output or, for a
//     pair that reaches into other CTAs, into one partial in global memory; the
//     last of those CTAs to arrive merges these in CTA order.
// All orders are fixed, so results do not depend on timing. At most one pair
// enters a CTA's run and one leaves it, hence two global partials per CTA.
// Against a fixed split per request: 64 ragged requests 188 -> 109 us, 8 of
// 131072 keys on one kv head 185 -> 59 us, one token 15.6 -> 6.4 us (with the
// copies' shape and the look-ahead below).
constexpr int kWarps = 8;          // 12 and 16, with shallower rings, measured 0 to 40 % slower on few requests
constexpr int kAlone = 8;          // pages a warp takes alone rather than share them and merge (4 and 16: the same)
constexpr float kMergeCost = 1.f;  // see plan_work (one request of 32768 keys on one kv head: 0.5 and 2 +13 %)
constexpr int kPad = 2;            // pages that a pair costs a warp besides its own, see plan_work
constexpr int kStageBytes = 2 * PAGE * D + 64;  // K, V, 2 x 16 exponents
constexpr int kRow = D + 4;                     // floats per head of a partial in shared memory (bank spread)

template <int NT>
constexpr int kStages = NT == 1 ? 5 : 4;

// x / n for x / n below 2^20.
MBX_DEVICE int quotient(int x, int n) {
  int q = __float2int_rz(__fdividef((float)x, (float)n));
  const int r = x - q * n;
  return q + (r >= n) - (r < 0);
}

// How the work is cut. kList: runs of `run` entries of the list, in which every
// pair is followed by `pad` empty ones. Where no pair is longer than a few
// pages, sharing and merging it costs more than it saves: kWarp gives each warp
// a pair, kCta each CTA one (its warps `run` pages each).
enum Cut : int { kList, kWarp, kCta };
struct WorkPlan {
  int cut, run, pad;
};
// pages, some: of all requests together, and how many have any; top, low: the
// longest and the shortest of those.
MBX_DEVICE WorkPlan plan_work(int pages, int some, int top, int low, int pairs, int nkv, int grid, int warps) {
  if (top <= kAlone && pairs <= grid * warps) return {kWarp, top, 0};
  if (top <= kAlone * warps && pairs <= grid) return {kCta, (top + warps - 1) / warps, 0};
  const int n = grid * warps;
  int run = max(1, (pages * nkv + n - 1) / n);
  // Beginning and ending a pair takes a warp about as long as two pages. Where
  // runs can hold whole pairs, warps with many short ones would come late; where
  // they cannot, empty entries would only move pairs off the runs' borders. (64
  // requests up to 512 keys: 20.8 us without, 16.0 with; 64 of 4096: 93.7, 96.9.)
  const int pad = low < run ? kPad : 0;
  if (pad) run = max(1, ((pages + pad * some) * nkv + n - 1) / n);
  // with few pairs, one more CTA per pair costs its merge more than it saves
  float root;
  asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(root) : "f"((float)top));
  return {kList, max(run, (int)(root * (kMergeCost / warps) + 0.999f)), pad};
}

template <int NT>
struct DecodeSmem {
  static constexpr int kHeads = 8 * NT;
  static constexpr int kWarpBytes = kStages<NT> * kStageBytes;  // a warp's ring, then its last segment's partial
  static constexpr int kPartBytes = kHeads * kRow * 4;
  static constexpr int kPart = kWarps * kWarpBytes;             // [kWarps] partials of the warps' first segments
  static constexpr int kMl = kPart + kWarps * kPartBytes;       // float2 [2][kWarps][kHeads]
  static constexpr int kTotal = kMl + 2 * kWarps * kHeads * 8;
  static_assert(kWarpBytes >= kPartBytes, "a partial fits in the ring");
};

MBX_DEVICE uint32_t smem_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
MBX_DEVICE void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
MBX_DEVICE void cp_async4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
MBX_DEVICE void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
MBX_DEVICE void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// What a warp left for the merge: of its first segment, where that began before
// the warp's run (slot 0), and of its last, where that goes on behind it (slot
// 1). kEnds: the pair's pages end in this warp's run.
enum SegFlags : int { kHere = 1, kEnds = 2 };

MBX_DEVICE float merge_weight(float m, float M) { return M == -INFINITY ? 0.f : ex2(m - M); }
MBX_DEVICE float warp_max(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
// 1 / l, or 0 for a row without keys. One unit in the last place of fp32 is
// far below the bf16 rounding that follows.
MBX_DEVICE float inverse(float l) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(l));
  return l == 0.f ? 0.f : r;
}
// Loads of partials: shared memory, or global memory past L1 (other CTAs may
// have written them).
MBX_DEVICE float4 ld_partial4(const float* p) {
  float4 v;
  asm volatile("ld.volatile.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "l"(p));
  return v;
}
MBX_DEVICE float2 ld_partial2(const float* p) {
  float2 v;
  asm volatile("ld.volatile.v2.f32 {%0,%1}, [%2];" : "=f"(v.x), "=f"(v.y) : "l"(p));
  return v;
}
MBX_DEVICE void add_scaled(float4& o, float w, const float4& x) {
  o.x += w * x.x;
  o.y += w * x.y;
  o.z += w * x.z;
  o.w += w * x.w;
}
template <int NT>
__global__ void __launch_bounds__(kWarps * 32, 1) decode_kv8_kernel(Kv8DecodeArgs a) {
  using S = DecodeSmem<NT>;
  constexpr int kSt = kStages<NT>, kW = kWarps;
  pdl_wait();
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int flags[2][kW];   // SegFlags
  __shared__ int4 pairs[2][kW];  // of these segments: request, kv head, list index of the pair's first page, its pages
  __shared__ int s_last[2];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int G = a.nq / a.nkv;
  const int max_keys = a.max_blocks * PAGE;
  auto pages_of = [&](int b) { return b < a.B ? (min(max(a.kv_len[b], 0), max_keys) + PAGE - 1) / PAGE : 0; };
  if (lane < 2) flags[lane][warp] = 0;
  // ---- this warp's run of pages, and where it starts: every warp for itself.
  // Lane c holds the pages of requests 32c .. 32c + 31 (of each 1024), and how
  // many of them have any.
  int total = 0, some = 0, top = 0, low = 1 << 30, sums = 0, counts = 0;
#pragma unroll 1
  for (int c0 = 0; c0 * 32 < a.B; ++c0) {
    const int x = pages_of(c0 * 32 + lane);
    const int sx = __reduce_add_sync(0xffffffffu, x), nx = __popc(__ballot_sync(0xffffffffu, x > 0));
    total += sx;
    some += nx;
    top = max(top, x);
    low = x > 0 ? min(low, x) : low;
    if (lane == c0) sums = sx, counts = nx;
  }
  top = __reduce_max_sync(0xffffffffu, top);
  low = __reduce_min_sync(0xffffffffu, low);
  const WorkPlan plan = plan_work(total, some, top, low, a.B * a.nkv, a.nkv, gridDim.x, kW);
  const int run = plan.run, pad = plan.pad;
  auto in_list = [&](int pages) { return pages > 0 ? pages + pad : 0; };
  const int u0 = (blockIdx.x * kW + warp) * run;  // first page in the list
  int left = 0;     // of the run (list entries)
  int4 at = make_int4(0, 0, 0, 0);  // request, kv head, page and the pair's pages there
  if (plan.cut == kList) {
    sums += counts * pad;
    left = max(0, min(run, (total + some * pad) * a.nkv - u0));
    if (left > 0) {
      auto scan = [&](int v) {
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int x = __shfl_up_sync(0xffffffffu, v, o);
          if (lane >= o) v += x;
        }
        return v;
      };
      int before = 0, b0 = 0;  // pages of the requests in front; first of the 1024 looked at
      int end = scan(sums);
#pragma unroll 1
      while (__shfl_sync(0xffffffffu, end, 31) * a.nkv <= u0 && b0 < a.B) {
        before = __shfl_sync(0xffffffffu, end, 31);
        b0 += 1024;
        sums = 0;
#pragma unroll 1
        for (int c = 0; c < 32; ++c) {
          const int x = __reduce_add_sync(0xffffffffu, in_list(pages_of(b0 + c * 32 + lane)));
          if (lane == c) sums = x;
        }
        end = before + scan(sums);
      }
      const int c = __popc(__ballot_sync(0xffffffffu, end * a.nkv <= u0));
      before = __shfl_sync(0xffffffffu, end - sums, c);
      const int n = in_list(pages_of(b0 + c * 32 + lane));
      end = before + scan(n);
      const int r = __popc(__ballot_sync(0xffffffffu, end * a.nkv <= u0));
      at.x = b0 + c * 32 + r;
      const int len = __shfl_sync(0xffffffffu, n, r);
      const int off = u0 - __shfl_sync(0xffffffffu, end - n, r) * a.nkv;
      at.y = quotient(off, len);
      at.z = off - at.y * len;
      at.w = len - pad;
      if (at.x >= a.B) left = 0;
    }
  } else {
    const int pair = plan.cut == kCta ? blockIdx.x : blockIdx.x * kW + warp;
    at.x = quotient(pair, a.nkv);
    at.y = pair - at.x * a.nkv;
    at.z = plan.cut == kCta ? warp * run : 0;
    at.w = pages_of(at.x);
    left = max(0, min(run, at.w - at.z));
  }

  const uint32_t ring = smem_addr(smem) + warp * S::kWarpBytes;
  if (left > 0) {
    // cursors: the pages being used, and the ones being fetched
    struct Cursor {
      int b, kvh, p, pages, left;
    };
    Cursor use{at.x, at.y, at.z, at.w, left};
    int pos = u0;  // use's place in the list
    auto pages_in = [&](int keys) { return (min(max(keys, 0), max_keys) + PAGE - 1) / PAGE; };
    auto keys_of = [&](int b) { return b < a.B ? a.kv_len[b] : 0; };
    // to the next pair (there is one), with the length of the next request in hand
    auto next_pair = [&](Cursor& c, int next_keys) {
      c.p = 0;
      if (++c.kvh < a.nkv) return false;
      c.kvh = 0;
      ++c.b;
      c.pages = pages_in(next_keys);
#pragma unroll 1
      while (c.pages == 0 && ++c.b < a.B) c.pages = pages_of(c.b);
      if (c.b >= a.B) c.left = 0;  // only where another stream shortened a length meanwhile
      return true;
    };
    if (use.p >= use.pages) {  // the run starts in the room behind a pair
      use.left -= use.pages + pad - use.p;
      pos += use.pages + pad - use.p;
      if (use.left > 0) next_pair(use, keys_of(use.b + 1));
    }
    Cursor in = use;
    // What the cursors will need is loaded ahead: lane i holds the block of page
    // win + i of the request being fetched, of page win + 32 + i, of page i of
    // it and of the next request, whose length next_keys is.
    auto ids_of = [&](int b, int p) {
      return b < a.B && p + lane < a.max_blocks ? a.block_table[b * a.bt_s + p + lane] : -1;
    };
    int win = in.p, id = ids_of(in.b, win), id_next = ids_of(in.b, win + 32);
    int first = ids_of(in.b, 0), next_first = ids_of(in.b + 1, 0), next_keys = keys_of(in.b + 1);
    typename HeadState<NT>::Query query;
    auto load_query = [&](int b, int kvh) { query.load(a.q + ((int64_t)b * a.nq + kvh * G) * D, G, lane); };
    if (use.left > 0) load_query(use.b, use.kvh);
    int keys = keys_of(use.b), use_next_keys = next_keys;
    // Each copy instruction reads 512 contiguous bytes (four rows, lane l the
    // l-th 16) and places them where pages() reads them.
    uint32_t k_dst[2], v_dst[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int row = i * 4 + (lane >> 3), ch = lane & 7;
      k_dst[i] = k_place(row, ch);
      v_dst[i] = 2048 + v_place(row, ch);
    }
    uint32_t bad = 0;  // stages whose page is not in the cache
    auto fetch = [&](int st) {
      if (in.p == in.pages) {
        in.left -= pad;
        if (in.left <= 0) return;
        const int b = in.b;
        if (next_pair(in, next_keys)) {
          first = in.b == b + 1 ? next_first : ids_of(in.b, 0);
          next_first = ids_of(in.b + 1, 0);
          next_keys = keys_of(in.b + 1);
        }
        win = 0;
        id = first;
        id_next = in.pages > 32 ? ids_of(in.b, 32) : -1;
      }
      if (in.left <= 0) return;
      if (in.p == win + 32) {
        win += 32;
        id = id_next;
        id_next = ids_of(in.b, win + 32);
      }
      const int blk = __shfl_sync(0xffffffffu, id, in.p - win);
      const uint32_t dst = ring + st * kStageBytes;
      if (blk >= 0 && blk < a.num_blocks) {
        bad &= ~(1u << st);
        const int64_t base = ((int64_t)blk * a.nkv + in.kvh) * PAGE * D + lane * 16;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          cp_async16(dst + k_dst[i & 1] + (i >> 1) * 1024, a.kv + base + i * 512);
          cp_async16(dst + v_dst[i & 1] + (i >> 1) * 1024, a.vv + base + i * 512);
        }
        if (lane < 8) {
          const uint8_t* e = lane < 4 ? a.ke + blk * a.ke_sb + in.kvh * a.ke_sh + lane * 4
                                      : a.ve + blk * a.ve_sb + in.kvh * a.ve_sh + (lane - 4) * 4;
          cp_async4(dst + 4096 + lane * 4, e);
        }
      } else {
        bad |= 1u << st;
      }
      ++in.p;
      --in.left;
    };
    // groups 0..kSt-1: the first pages; then one group per page used, in order
#pragma unroll 1
    for (int i = 0; i < kSt; ++i) {
      fetch(i);
      cp_async_commit();
    }
    HeadState<NT> st;
    bool fresh = true;
    int seg_p0 = use.p;  // the segment's first page
    int L = 0;
    int stage = 0;
    while (use.left > 0) {
      if (fresh) {
        st.begin(query, a.scale_log2, lane);
        L = min(keys, max_keys);
        seg_p0 = use.p;
        fresh = false;
        // the next pair's query, where this warp will come to it
        if (NT == 1 && use.left > use.pages - use.p + pad) {
          const bool same = use.kvh + 1 < a.nkv;
          load_query(same ? use.b : min(use.b + 1, a.B - 1), same ? use.kvh + 1 : 0);
        }
      }
      cp_async_wait<kSt - 2>();
      __syncwarp();
      const int stage1 = stage + 1 == kSt ? 0 : stage + 1;
      const uint8_t* const src[2] = {smem + warp * S::kWarpBytes + stage * kStageBytes,
                                     smem + warp * S::kWarpBytes + stage1 * kStageBytes};
      const bool two = use.left > 1 && use.p + 1 < use.pages;
      const int live[2] = {(bad >> stage) & 1 ? 0 : min(PAGE, L - use.p * PAGE),
                           !two || ((bad >> stage1) & 1) ? 0 : min(PAGE, L - use.p * PAGE - PAGE)};
      st.pages(src, live, lane);
      __syncwarp();
#pragma unroll 1
      for (int u = two ? 2 : 1; u > 0; --u) {
        fetch(stage);
        cp_async_commit();
        stage = stage + 1 == kSt ? 0 : stage + 1;
        ++pos;
        ++use.p;
        --use.left;
      }
      const bool ends = use.p == use.pages;
      if (!ends && use.left > 0) continue;
      // ---- the segment is done
      st.end();
      // Rows are divided by their sum here, partial ones too, and the weights' 2^d
      // is taken out in two halves: nothing on the way leaves fp32's normal range
      // where the result does not.
      if (seg_p0 == 0 && ends) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const int head = n * 8 + 2 * t + c;
            if (head >= G) continue;
            const int d = st.d23[n][c] >> 23;
            const float vs = pow2(-(d >> 1)), inv = inverse(st.l[n][c]) * pow2((d >> 1) - d);
            float f[16];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              f[2 * j] = st.o[n][j][c] * inv * vs;
              f[2 * j + 1] = st.o[n][j][2 + c] * inv * vs;
            }
            __nv_bfloat16* dst = a.o + ((int64_t)use.b * a.nq + use.kvh * G + head) * D + g * 16;
            *reinterpret_cast<uint4*>(dst) = pack_from<__nv_bfloat16>(f);
            *reinterpret_cast<uint4*>(dst + 8) = pack_from<__nv_bfloat16>(f + 8);
          }
      } else {
        // began earlier: slot 0; begins here and goes on behind the run, whose
        // ring is free then: slot 1
        const int slot = seg_p0 == 0 ? 1 : 0;
        float* po = reinterpret_cast<float*>(smem + (slot == 0 ? S::kPart + warp * S::kPartBytes : warp * S::kWarpBytes));
        float2* ml = reinterpret_cast<float2*>(smem + S::kMl) + (slot * kW + warp) * S::kHeads;
        __syncwarp();
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const int head = n * 8 + 2 * t + c;
            if (head >= G) continue;
            const int d = st.d23[n][c] >> 23;
            const float vs = pow2(-(d >> 1)), inv = inverse(st.l[n][c]) * pow2((d >> 1) - d);
#pragma unroll
            for (int j = 0; j < 8; ++j)
              *reinterpret_cast<float2*>(po + head * kRow + g * 16 + 2 * j) =
                  make_float2(st.o[n][j][c] * inv * vs, st.o[n][j][2 + c] * inv * vs);
            if (g == 0) ml[head] = make_float2(st.m[n][c], st.l[n][c]);
          }
        if (lane == 0) {
          flags[slot][warp] = kHere | (ends ? kEnds : 0);
          pairs[slot][warp] = make_int4(use.b, use.kvh, pos - use.p, use.pages);
        }
      }
      fresh = true;
      if (!ends) break;
      use.left -= pad;
      pos += pad;
      if (use.left <= 0) break;
      const int b = use.b;
      if (next_pair(use, use_next_keys)) {
        keys = use.b == b + 1 ? use_next_keys : keys_of(use.b);
        use_next_keys = keys_of(use.b + 1);
      }
      if (use.left > 0 && (NT > 1 || use.b > b + 1)) load_query(use.b, use.kvh);
    }
  }
  // requests without keys: zeros, by the CTAs in turn
#pragma unroll 1
  for (int b = blockIdx.x + gridDim.x * warp; b < a.B; b += gridDim.x * kW) {
    if (pages_of(b) > 0) continue;
    uint4* dst = reinterpret_cast<uint4*>(a.o + (int64_t)b * a.nq * D);
#pragma unroll 1
    for (int i = lane; i < a.nq * D / 8; i += 32) dst[i] = make_uint4(0, 0, 0, 0);
  }
  __syncthreads();

  // ---- merges. Level 0, the warps' partials: chain 0 entered the CTA's run,
  // chain c + 1 begins in warp c's; it goes on through the first segments of the
  // warps that follow, up to the first that ends. Level 1, by the last CTA to
  // arrive: the CTAs' partials of a pair that reaches over CTAs. One code for
  // both (what runs once a launch waits for its instructions, too): partial 0
  // lies by itself, the others a stride apart. A warp per (chain, head): lane i
  // has partial i's (m, l), so that the weights 2^(m_i - M) l_i come at once and the
  // rows (lane l: dims 4l..4l+3) are independent loads.
  const int f0 = lane < kW ? flags[0][lane] : 0, f1 = lane < kW ? flags[1][lane] : 0;
  const uint32_t held = __ballot_sync(0xffffffffu, f0 != 0), ended = __ballot_sync(0xffffffffu, f0 & kEnds),
                 begun = __ballot_sync(0xffffffffu, f1 != 0);
  float* part_ml = a.part + (int64_t)gridDim.x * 2 * S::kHeads * D;
  const int span = kW * run;     // pages per CTA
  const bool out0 = held & 1;    // chain 0 is one of several CTAs'
  int out1 = -1;                 // the warp in whose run a pair begins that goes on in the next CTA
  uint32_t todo = (begun << 1) | (held & 1);
#pragma unroll 1
  for (int level = 0; level < 2; ++level) {
    int turn = warp;
#pragma unroll 1
    for (; todo != 0; todo &= todo - 1) {
      const int c = __ffs(todo) - 2;  // -1, or the warp whose run the pair begins in
      const int begins = c >= 0;
      const int4 pair = begins ? pairs[1][c] : pairs[0][0];
      int n;
      bool whole = true;
      const float *row0, *row1, *ml0, *ml1;  // rows and (m, l) of partials 0 and 1 of head 0
      int row_step, ml_step, head_step;      // in floats
      if (level == 0) {
        const uint32_t ends = ended >> (c + 1);
        n = begins + (ends ? __ffs(ends) : __popc(held >> (c + 1)));
        whole = begins && ends;
        if (begins && !ends) out1 = c;
        const float* const parts = reinterpret_cast<const float*>(smem + S::kPart);
        const float* const ml = reinterpret_cast<const float*>(smem + S::kMl);
        row_step = S::kPartBytes / 4;
        row1 = parts + (c + 1 + !begins) * row_step;
        row0 = begins ? reinterpret_cast<const float*>(smem + c * S::kWarpBytes) : parts;
        ml_step = 2 * S::kHeads;
        ml1 = ml + (c + 1 + !begins) * ml_step;
        ml0 = ml + (begins ? kW + c : 0) * ml_step;
        head_step = kRow;
      } else {
        const int c0 = s_last[begins];
        n = quotient(pair.z + pair.w - 1, span) - c0 + 1;
        row_step = 2 * S::kHeads * D;
        row0 = a.part + (int64_t)(2 * c0 + 1) * S::kHeads * D;
        row1 = row0 + S::kHeads * D;
        ml_step = 4 * S::kHeads;
        ml0 = part_ml + (2 * c0 + 1) * S::kHeads * 2;
        ml1 = ml0 + 2 * S::kHeads;
        head_step = D;
      }
#pragma unroll 1
      for (; turn < G; turn += kW) {
        const int head = turn;
        float M = -INFINITY, l = 0.f;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
        constexpr int kBlock = 8;  // partials loaded at once
#pragma unroll 1
        for (int i0 = 0; i0 < n; i0 += kBlock) {
          const int mine = i0 + lane;
          const bool has = lane < kBlock && mine < n;
          float2 x = make_float2(-INFINITY, 0.f);
          if (has) x = ld_partial2((mine == 0 ? ml0 : ml1 + (mine - 1) * ml_step) + 2 * head);
          float4 y[kBlock];
#pragma unroll
          for (int j = 0; j < kBlock; ++j) {
            const int i = min(i0 + j, n - 1);
            y[j] = ld_partial4((i == 0 ? row0 : row1 + (int64_t)(i - 1) * row_step) + head * head_step + lane * 4);
          }
          const float nm = fmaxf(M, warp_max(x.x));
          const float keep = merge_weight(M, nm);
          const float part = has ? merge_weight(x.x, nm) * x.y : 0.f;
          const float sum = l * keep + warp_sum(part), inv = inverse(sum);
          const float w = part * inv, old = l * keep * inv;
          M = nm;
          l = sum;
          o = make_float4(o.x * old, o.y * old, o.z * old, o.w * old);
#pragma unroll
          for (int j = 0; j < kBlock; ++j)  // behind the last partial: its row again, weight 0
            add_scaled(o, __shfl_sync(0xffffffffu, w, j), y[j]);
        }
        if (whole) {
          const __nv_bfloat162 lo = __floats2bfloat162_rn(o.x, o.y);
          const __nv_bfloat162 hi = __floats2bfloat162_rn(o.z, o.w);
          uint2 y;
          y.x = *reinterpret_cast<const uint32_t*>(&lo);
          y.y = *reinterpret_cast<const uint32_t*>(&hi);
          *reinterpret_cast<uint2*>(a.o + ((int64_t)pair.x * a.nq + pair.y * G + head) * D + lane * 4) = y;
        } else {
          const int to = (blockIdx.x * 2 + begins) * S::kHeads + head;
          *reinterpret_cast<float4*>(a.part + (int64_t)to * D + lane * 4) = o;
          if (lane == 0) *reinterpret_cast<float2*>(part_ml + 2 * to) = make_float2(M, l);
        }
      }
      turn -= G;
    }
    if (level == 1 || (!out0 && out1 < 0)) return;
    __syncthreads();
    if (threadIdx.x < 2) {
      int last = -1;
      if (threadIdx.x == 0 ? out0 : out1 >= 0) {
        const int4 pair = threadIdx.x == 0 ? pairs[0][0] : pairs[1][out1];
        const int c0 = quotient(pair.z, span), c1 = quotient(pair.z + pair.w - 1, span);
        // this CTA's partials before the count, the count before the others' partials
        int seen;
        asm volatile("atom.acq_rel.gpu.global.add.s32 %0, [%1], 1;" : "=r"(seen) : "l"(a.counters + c0) : "memory");
        if (seen == c1 - c0) {
          a.counters[c0] = 0;  // for the next launch
          last = c0;
        }
      }
      s_last[threadIdx.x] = last;
    }
    __syncthreads();
    todo = (s_last[0] >= 0 ? 1u : 0u) | (s_last[1] >= 0 ? 2u << out1 : 0u);
  }
}

}  // namespace

void rope_and_cache_kv8_launch(const void* qkv, const int* pos, const float* cos_sin, int64_t max_pos,
                               const int64_t* slots, void* q_out, const Kv8Cache& c, int64_t T, int nq, int nkv,
                               cudaStream_t s, const void* q_norm, const void* k_norm, double eps) {
  if (T == 0) return;
  AppendArgs a;
  a.qkv = static_cast<const __nv_bfloat16*>(qkv);
  a.pos = pos;
  a.cos_sin = cos_sin;
  a.slots = slots;
  a.q_out = static_cast<__nv_bfloat16*>(q_out);
  a.kv = c.kv;
  a.vv = c.vv;
  a.ke = c.ke;
  a.ve = c.ve;
  a.ke_sb = c.ke_sb;
  a.ke_sh = c.ke_sh;
  a.ve_sb = c.ve_sb;
  a.ve_sh = c.ve_sh;
  a.q_norm = static_cast<const __nv_bfloat16*>(q_norm);
  a.k_norm = static_cast<const __nv_bfloat16*>(k_norm);
  a.eps = eps;
  a.T = T;
  a.n_slots = c.blocks * PAGE;
  a.max_pos = (int)max_pos;
  a.nq = nq;
  a.nkv = nkv;
  // Tokens per k/v CTA: one where there are few (64 tokens of 32 + 2 x 8 heads:
  // 3.0 us, two 3.6, four 5.2); more for many, since every CTA looks through all
  // later slots for its own (8005 tokens of 64 + 2 x 8: 2 tokens 88 us, 16
  // tokens 65). q passes per warp share the angles: one, two and four measure
  // 81, 69 and 65 us there, and 10.2, 8.0 and 8.6 at 1024 tokens of 32 heads.
  const int tokens = T <= 128 ? 1 : (int)std::min<int64_t>(kMaxTokens, std::max<int64_t>(2, (T + 511) / 512));
  const int passes = T * nq >= 1 << 18 ? 4 : T * nq >= 1 << 14 ? 2 : 1;
  const int64_t kv_ctas = (T + tokens - 1) / tokens;
  const int64_t q_tasks = T * ((nq + 4 * passes - 1) / (4 * passes));
  const dim3 grid((unsigned)(kv_ctas + (q_tasks + kAppendWarps - 1) / kAppendWarps));
  if (q_norm != nullptr)
    launch_k(append_kernel<true>, grid, dim3(kAppendWarps * 32), 0, s, a, (int)kv_ctas, tokens, passes);
  else
    launch_k(append_kernel<false>, grid, dim3(kAppendWarps * 32), 0, s, a, (int)kv_ctas, tokens, passes);
  MBX_CUDA_CHECK(cudaGetLastError());
}

void read_pages_kv8_launch(const Kv8Cache& c, int nkv, const int* block_table, int64_t bt_stride, const int* out_table,
                           int64_t ot_stride, const int* kv_len, int R, int max_blocks, void* k_out, void* v_out,
                           int64_t out_pages, cudaStream_t s) {
  if (R == 0 || max_blocks == 0) return;
  ReadArgs a{c.kv, c.vv, c.ke, c.ve, c.ke_sb, c.ke_sh, c.ve_sb, c.ve_sh, block_table, out_table, kv_len,
             bt_stride, ot_stride, static_cast<__nv_bfloat16*>(k_out), static_cast<__nv_bfloat16*>(v_out), out_pages,
             max_blocks, nkv, (int)c.blocks};
  const int tasks = R * max_blocks * nkv;
  launch_k(read_pages_kernel, dim3((tasks + kReadWarps - 1) / kReadWarps), dim3(kReadWarps * 32), 0, s, a, tasks);
  MBX_CUDA_CHECK(cudaGetLastError());
}

int decode_kv8_grid(int B, int nkv, int max_blocks) {
  static std::atomic<int> sms_of[64];  // 0: not asked yet
  int dev = 0;
  MBX_CUDA_CHECK(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64) throw std::runtime_error("decode: device index out of range");
  int sms = sms_of[dev].load(std::memory_order_relaxed);
  if (sms == 0) {
    MBX_CUDA_CHECK(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
    sms_of[dev].store(sms, std::memory_order_relaxed);
  }
  const int64_t pages = (int64_t)B * nkv * max_blocks;
  return (int)std::max<int64_t>(1, std::min<int64_t>(sms, (pages + kWarps - 1) / kWarps));
}

size_t decode_kv8_part_floats(int grid) { return (size_t)grid * 2 * 16 * (D + 2); }

void decode_attention_kv8_launch(const void* q, const Kv8Cache& c, void* o, const int* kv_len, const int* block_table,
                                 int64_t bt_stride, int max_blocks, int B, int nq, int nkv, int grid, float* part,
                                 int* counters, float scale, cudaStream_t s) {
  if (B == 0) return;
  if (nq % nkv != 0 || nq / nkv > 16) throw std::runtime_error("decode: group size must be <= 16");
  Kv8DecodeArgs a{static_cast<const __nv_bfloat16*>(q), c.kv, c.vv, c.ke, c.ve, c.ke_sb, c.ke_sh, c.ve_sb, c.ve_sh,
                  static_cast<__nv_bfloat16*>(o), part, counters, kv_len, block_table, bt_stride, B, max_blocks,
                  (int)c.blocks, nq, nkv, scale * 1.4426950408889634f};
  if (nq / nkv <= 8) {
    static SmemLimit limit;
    limit.ensure((const void*)decode_kv8_kernel<1>, DecodeSmem<1>::kTotal);
    launch_k(decode_kv8_kernel<1>, dim3(grid), dim3(kWarps * 32), DecodeSmem<1>::kTotal, s, a);
  } else {
    static SmemLimit limit;
    limit.ensure((const void*)decode_kv8_kernel<2>, DecodeSmem<2>::kTotal);
    launch_k(decode_kv8_kernel<2>, dim3(grid), dim3(kWarps * 32), DecodeSmem<2>::kTotal, s, a);
  }
  MBX_CUDA_CHECK(cudaGetLastError());
}

}  // namespace mbx
