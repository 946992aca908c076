// The paged KV cache in 8 bits: writing it, reading it back, and attention of
// one new token per request over it (head_dim 128, pages of 16 tokens).
//
// A cached row x (one token, one kv head) is held as e4m3 numbers with one
// power-of-two scale:
//   e = the smallest integer with max|x_i| <= 448 * 2^e, at least -117
//   values_i = round_to_nearest_even_e4m3(x_i / 2^e),  exps = e + 127
// and stands for values_i * 2^e. e4m3 is a floating format, so a scale finer
// than a power of two would buy at most one exponent of range and no
// accuracy, while a power of two makes every scaling exact: a stored row is
// exact in bf16 and in fp32 products, and which e4m3 number a value rounds to
// does not depend on a division. Elements that are not finite are stored as
// NaN and do not take part in the maximum.
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

// A row's exponent from the largest magnitude of its finite elements (fp32):
// 448 = 1.75 * 2^8.
MBX_DEVICE int row_exp(float top) {
  const uint32_t b = __float_as_uint(top);
  const int e = (int)(b >> 23) - 127 - 8 + ((b & 0x7fffffu) > 0x600000u ? 1 : 0);
  return max(e, kMinExp);
}

// 2^e for e in [-126, 127].
MBX_DEVICE float pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// Two e4m3 numbers from lo and hi (lo in the low byte); what is not finite becomes NaN.
MBX_DEVICE uint32_t e4m3x2(float lo, float hi) {
  uint16_t r;
  const float nan = __uint_as_float(0x7fffffffu);
  lo = fabsf(lo) <= 3.4e38f ? lo : nan;
  hi = fabsf(hi) <= 3.4e38f ? hi : nan;
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
// rounding x itself: x cut to 24 bits, the last one set if anything was cut.
MBX_DEVICE float round_to_odd(double x) {
  const float f = __double2float_rz(x);
  return (double)f != x ? __uint_as_float(__float_as_uint(f) | 1u) : f;
}

MBX_DEVICE float finite_abs(float x) {
  const float a = fabsf(x);
  return a <= 3.4e38f ? a : 0.f;
}

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

// One warp per (token, head of [q | k | v]). Lane l holds dims 2l, 2l + 1 and
// their rotation partners 2l + 64, 2l + 65. k is normalised and rotated in 64
// bits, so that the stored byte is the one of the real number.
__global__ void __launch_bounds__(128) append_kernel(AppendArgs a) {
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int heads = a.nq + 2 * a.nkv;
  const int64_t task = (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  if (task >= a.T * heads) return;
  const int64_t t = task / heads;
  const int h = (int)(task % heads);
  const int j = 2 * lane;
  const __nv_bfloat16* src = a.qkv + task * D;
  float2 x = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(src + j));
  float2 y = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(src + 64 + j));
  const int p = min(max(a.pos[t], 0), a.max_pos - 1);
  const float* cs = a.cos_sin + (int64_t)p * D;
  const float c0 = cs[j], c1 = cs[j + 1], s0 = cs[64 + j], s1 = cs[64 + j + 1];
  if (h < a.nq) {
    if (a.q_norm != nullptr) {
      const float r = rsqrtf(warp_sum(x.x * x.x + x.y * x.y + y.x * y.x + y.y * y.y) * (1.f / D) + (float)a.eps);
      x.x = x.x * r * __bfloat162float(a.q_norm[j]);
      x.y = x.y * r * __bfloat162float(a.q_norm[j + 1]);
      y.x = y.x * r * __bfloat162float(a.q_norm[64 + j]);
      y.y = y.y * r * __bfloat162float(a.q_norm[64 + j + 1]);
    }
    __nv_bfloat16* dst = a.q_out + (t * a.nq + h) * D;
    *reinterpret_cast<__nv_bfloat162*>(dst + j) = __floats2bfloat162_rn(x.x * c0 - y.x * s0, x.y * c1 - y.y * s1);
    *reinterpret_cast<__nv_bfloat162*>(dst + 64 + j) = __floats2bfloat162_rn(y.x * c0 + x.x * s0, y.y * c1 + x.y * s1);
    return;
  }
  const int64_t slot = a.slots[t];
  if (slot < 0 || slot >= a.n_slots) return;
  // a slot that a later token names as well holds that token's row
  bool later = false;
  for (int64_t u = t + 1 + lane; u < a.T; u += 32) later |= a.slots[u] == slot;
  if (__any_sync(0xffffffffu, later)) return;
  const bool is_k = h < a.nq + a.nkv;
  const int kh = is_k ? h - a.nq : h - a.nq - a.nkv;
  float v[4] = {x.x, x.y, y.x, y.y};
  if (is_k) {
    double d[4] = {x.x, x.y, y.x, y.y};
    if (a.k_norm != nullptr) {
      double ss = d[0] * d[0] + d[1] * d[1] + d[2] * d[2] + d[3] * d[3];
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      const double r = 1.0 / sqrt(ss * (1.0 / D) + a.eps);
      d[0] *= r * __bfloat162float(a.k_norm[j]);
      d[1] *= r * __bfloat162float(a.k_norm[j + 1]);
      d[2] *= r * __bfloat162float(a.k_norm[64 + j]);
      d[3] *= r * __bfloat162float(a.k_norm[64 + j + 1]);
    }
    v[0] = round_to_odd(d[0] * c0 - d[2] * s0);
    v[1] = round_to_odd(d[1] * c1 - d[3] * s1);
    v[2] = round_to_odd(d[2] * c0 + d[0] * s0);
    v[3] = round_to_odd(d[3] * c1 + d[1] * s1);
  }
  float top = fmaxf(fmaxf(finite_abs(v[0]), finite_abs(v[1])), fmaxf(finite_abs(v[2]), finite_abs(v[3])));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  const int e = row_exp(top);
  const float inv = pow2(-e);
  const int64_t blk = slot / PAGE;
  const int off = (int)(slot % PAGE);
  uint8_t* dst = (is_k ? a.kv : a.vv) + ((blk * a.nkv + kh) * PAGE + off) * D;
  *reinterpret_cast<uint16_t*>(dst + j) = (uint16_t)e4m3x2(v[0] * inv, v[1] * inv);
  *reinterpret_cast<uint16_t*>(dst + 64 + j) = (uint16_t)e4m3x2(v[2] * inv, v[3] * inv);
  if (lane == 0) {
    if (is_k) a.ke[blk * a.ke_sb + kh * a.ke_sh + off] = (uint8_t)(e + 127);
    else a.ve[blk * a.ve_sb + kh * a.ve_sh + off] = (uint8_t)(e + 127);
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

// 16 e4m3 numbers to bf16, times 2^e (exact).
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
  *reinterpret_cast<uint4*>(dst) = pack_from<__nv_bfloat16>(f);
  *reinterpret_cast<uint4*>(dst + 8) = pack_from<__nv_bfloat16>(f + 8);
}

// One block of 128 threads per (page, kv head, request): a thread per 16
// elements. Rows behind the length are written as zeros, so that whatever
// reads whole pages never meets what an earlier user of the page left there.
__global__ void __launch_bounds__(128) read_pages_kernel(ReadArgs a) {
  pdl_wait();
  const int i = blockIdx.x, h = blockIdx.y, r = blockIdx.z;
  const int L = a.kv_len[r];
  if (i * PAGE >= L) return;
  const int blk = a.block_table[r * a.bt_s + i];
  const int64_t to = a.out_table ? a.out_table[r * a.ot_s + i] : (int64_t)r * a.max_blocks + i;
  if (to < 0 || to >= a.out_pages) return;
  const int row = threadIdx.x >> 3;
  const bool live = i * PAGE + row < L && blk >= 0 && blk < a.num_blocks;
  const int64_t src = live ? ((int64_t)blk * a.nkv + h) * PAGE * D + threadIdx.x * 16 : 0;
  const int64_t dst = (to * a.nkv + h) * PAGE * D + threadIdx.x * 16;
  uint4 k = make_uint4(0, 0, 0, 0), v = k;
  float ks = 0.f, vs = 0.f;
  if (live) {
    k = ld_v4(a.kv + src);
    v = ld_v4(a.vv + src);
    ks = __uint_as_float((uint32_t)a.ke[blk * a.ke_sb + h * a.ke_sh + row] << 23);
    vs = __uint_as_float((uint32_t)a.ve[blk * a.ve_sb + h * a.ve_sh + row] << 23);
  }
  emit16(k, ks, a.k_out + dst);
  emit16(v, vs, a.v_out + dst);
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
//  * softmax in base 2 with a running maximum m. The value exponents join the
//    weights: w = 2^(s - m) * 2^(ve - vr + 8) in f16 with vr a running maximum
//    of ve, so weights down to 2^-22 of the largest keep 11 bits (bf16 would
//    keep 8). m and vr only move when a page exceeds them by more than 2^4 and
//    2^3: then w <= 2^15 stays inside f16. The row sum uses the fp32 weights.
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
  float* part_o;           // [B, nq, splits, D]
  float* part_lse;         // [B, nq, splits]
  const int* kv_len;       // [B]
  const int* block_table;  // [B, max_blocks], row stride bt_s
  int64_t bt_s;
  int max_blocks, num_blocks, nq, nkv, splits;
  float scale_log2;
};

constexpr int kNoExp = -1000;  // value exponent of a masked key, and vr before the first page

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
  int vr;

  MBX_DEVICE void begin(const __nv_bfloat16* q, int G, float scale_log2, int lane) {
    const int g = lane >> 2, t = lane & 3;
    vr = kNoExp;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int head = n * 8 + g;
      float x[2][16];
      float top = 0.f;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          uint4 w = make_uint4(0, 0, 0, 0);
          if (head < G) w = ld_v4(q + head * D + (t + 4 * h) * 16 + c * 8);
          float f[8] = {};
          unpack_add<__nv_bfloat16>(w, f);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            x[h][c * 8 + i] = f[i];
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
        m[n][c] = -INFINITY;
        l[n][c] = 0.f;
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) o[n][i][0] = o[n][i][1] = o[n][i][2] = o[n][i][3] = 0.f;
    }
  }

  // k[0..1]: row g, chunks t and t + 4; k[2..3]: row g + 8. v[i]: chunk g of
  // keys 2t, 2t + 1, 2t + 8, 2t + 9. ke, ve: exponent bytes of keys g, g + 8.
  // Only the page's first `live` keys count.
  MBX_DEVICE void page(const uint4 (&k)[4], uint4 (&v)[4], const int (&ke)[2], const int (&ve)[2], int live,
                       int lane) {
    const int g = lane >> 2, t = lane & 3;
    float s[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
    const uint32_t kw[4][4] = {{k[0].x, k[0].y, k[0].z, k[0].w},
                               {k[1].x, k[1].y, k[1].z, k[1].w},
                               {k[2].x, k[2].y, k[2].z, k[2].w},
                               {k[3].x, k[3].y, k[3].z, k[3].w}};
#pragma unroll
    for (int ks = 0; ks < 8; ++ks) {
      const uint32_t r0 = kw[ks >> 2][ks & 3], r8 = kw[2 + (ks >> 2)][ks & 3];
      const uint32_t af[4] = {f16x2_of(r0, 0), f16x2_of(r8, 0), f16x2_of(r0, 1), f16x2_of(r8, 1)};
#pragma unroll
      for (int n = 0; n < NT; ++n) mma_f16(s[n], af, qf[n][ks][0], qf[n][ks][1]);
    }
    const bool on[2] = {g < live, g + 8 < live};
    int vx[2];
    bool grow = false;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      vx[r] = on[r] ? ve[r] - 127 : kNoExp;
      grow |= vx[r] > vr + 3;
      const float kf = __uint_as_float((uint32_t)ke[r] << 23);
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const float x = on[r] ? s[n][2 * r + c] * (kf * qs[n][c]) : -INFINITY;
          s[n][2 * r + c] = x;
          grow |= x > m[n][c] + 4.f;
        }
    }
    if (__any_sync(0xffffffffu, grow)) {
      int nv = max(vr, max(vx[0], vx[1]));
#pragma unroll
      for (int off = 4; off < 32; off <<= 1) nv = max(nv, __shfl_xor_sync(0xffffffffu, nv, off));
      const float vc = ex2((float)(vr - nv));
      vr = nv;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float corr[2];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float nm = fmaxf(m[n][c], fmaxf(s[n][c], s[n][2 + c]));
#pragma unroll
          for (int off = 4; off < 32; off <<= 1) nm = fmaxf(nm, __shfl_xor_sync(0xffffffffu, nm, off));
          corr[c] = nm == -INFINITY ? 1.f : ex2(m[n][c] - nm);
          m[n][c] = nm;
          l[n][c] *= corr[c];
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          o[n][i][0] *= corr[0] * vc;
          o[n][i][1] *= corr[1] * vc;
          o[n][i][2] *= corr[0] * vc;
          o[n][i][3] *= corr[1] * vc;
        }
      }
    }
    uint32_t pf[NT][2];
    const float vf[2] = {pow2(max(vx[0] - vr + 8, -126)), pow2(max(vx[1] - vr + 8, -126))};
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        float w[2];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const float p = ex2(s[n][2 * r + c] - (m[n][c] == -INFINITY ? 0.f : m[n][c]));
          l[n][c] += p;
          w[c] = p * vf[r];
        }
        pf[n][r] = transpose8x8(pack_f16(w[0], w[1]));
      }
    if (live < PAGE) {  // rows behind the length may hold anything: 0 * NaN would not be 0
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (2 * t + (i & 1) + 8 * (i >> 1) >= live) v[i] = make_uint4(0, 0, 0, 0);
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
      for (int n = 0; n < NT; ++n) mma_f16(o[n][i], af, pf[n][0], pf[n][1]);
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

// One warp per (split, kv head, request), pages straight from global memory.
template <int NT>
__global__ void __launch_bounds__(32) decode_kv8_kernel(Kv8DecodeArgs a) {
  pdl_wait();
  const int split = blockIdx.x, kvh = blockIdx.y, b = blockIdx.z;
  const int lane = threadIdx.x, g = lane >> 2, t = lane & 3;
  const int G = a.nq / a.nkv;
  const int L = min(max(a.kv_len[b], 0), a.max_blocks * PAGE);
  const int pages = (L + PAGE - 1) / PAGE;
  const int per = (pages + a.splits - 1) / a.splits;
  HeadState<NT> st;
  st.begin(a.q + ((int64_t)b * a.nq + kvh * G) * D, G, a.scale_log2, lane);
  for (int p = split * per; p < min(pages, split * per + per); ++p) {
    const int blk = a.block_table[b * a.bt_s + p];
    if (blk < 0 || blk >= a.num_blocks) continue;
    const int64_t base = ((int64_t)blk * a.nkv + kvh) * PAGE * D;
    uint4 k[4], v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      k[i] = ld_v4(a.kv + base + (g + 8 * (i >> 1)) * D + (t + 4 * (i & 1)) * 16);
      v[i] = ld_v4(a.vv + base + (2 * t + (i & 1) + 8 * (i >> 1)) * D + g * 16);
    }
    const uint8_t* kep = a.ke + blk * a.ke_sb + kvh * a.ke_sh;
    const uint8_t* vep = a.ve + blk * a.ve_sb + kvh * a.ve_sh;
    const int ke[2] = {kep[g], kep[g + 8]}, ve[2] = {vep[g], vep[g + 8]};
    st.page(k, v, ke, ve, min(PAGE, L - p * PAGE), lane);
  }
  st.end();
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int head = n * 8 + 2 * t + c;
      if (head >= G) continue;
      const int64_t row = ((int64_t)b * a.nq + kvh * G + head) * a.splits + split;
      const float l = st.l[n][c];
      const float inv = l == 0.f ? 0.f : pow2(max(st.vr, -118) - 8) / l;
#pragma unroll
      for (int i = 0; i < 8; ++i)
        *reinterpret_cast<float2*>(a.part_o + row * D + g * 16 + 2 * i) =
            make_float2(st.o[n][i][c] * inv, st.o[n][i][2 + c] * inv);
      if (g == 0) a.part_lse[row] = l == 0.f ? -INFINITY : st.m[n][c] + log2f(l);
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
  const int64_t tasks = T * (nq + 2 * nkv);
  launch_k(append_kernel, dim3((unsigned)((tasks + 3) / 4)), dim3(128), 0, s, a);
  MBX_CUDA_CHECK(cudaGetLastError());
}

void read_pages_kv8_launch(const Kv8Cache& c, int nkv, const int* block_table, int64_t bt_stride, const int* out_table,
                           int64_t ot_stride, const int* kv_len, int R, int max_blocks, void* k_out, void* v_out,
                           int64_t out_pages, cudaStream_t s) {
  if (R == 0 || max_blocks == 0) return;
  ReadArgs a{c.kv, c.vv, c.ke, c.ve, c.ke_sb, c.ke_sh, c.ve_sb, c.ve_sh, block_table, out_table, kv_len,
             bt_stride, ot_stride, static_cast<__nv_bfloat16*>(k_out), static_cast<__nv_bfloat16*>(v_out), out_pages,
             max_blocks, nkv, (int)c.blocks};
  launch_k(read_pages_kernel, dim3(max_blocks, nkv, R), dim3(128), 0, s, a);
  MBX_CUDA_CHECK(cudaGetLastError());
}

void decode_attention_kv8_launch(const void* q, const Kv8Cache& c, void* o, const int* kv_len, const int* block_table,
                                 int64_t bt_stride, int max_blocks, int B, int nq, int nkv, int splits, float* part_o,
                                 float* part_lse, float scale, cudaStream_t s) {
  if (B == 0) return;
  if (nq % nkv != 0 || nq / nkv > 16) throw std::runtime_error("decode: group size must be <= 16");
  Kv8DecodeArgs a{static_cast<const __nv_bfloat16*>(q), c.kv, c.vv, c.ke, c.ve, c.ke_sb, c.ke_sh, c.ve_sb, c.ve_sh,
                  static_cast<__nv_bfloat16*>(o), part_o, part_lse, kv_len, block_table, bt_stride, max_blocks,
                  (int)c.blocks, nq, nkv, splits, scale * 1.4426950408889634f};
  const dim3 grid(splits, nkv, B);
  if (nq / nkv <= 8) launch_k(decode_kv8_kernel<1>, grid, dim3(32), 0, s, a);
  else launch_k(decode_kv8_kernel<2>, grid, dim3(32), 0, s, a);
  MBX_CUDA_CHECK(cudaGetLastError());
  attn_combine_launch(part_o, part_lse, (int64_t)B * nq, splits, o, s);
}

}  // namespace mbx
