// The key/value cache held in 4 bits: writing it (with RoPE), reading it back, and attention over it.
//
// Format. A value is code * s: code in [-7, 7] held as the nibble code + 8, s one bf16 scale per 32 dims of a (position,
// kv head): s = bf16(max|x| / 7), code = rint(x / s) clamped to [-7, 7] (0 where s is 0). x is bf16, so x / s in fp32
// decides exactly: a border (n + 1/2) s has at most 12 significant bits and x has 8, two unequal ones differ by more
// than 2^-13 of themselves, and a correctly rounded quotient cannot fall on a border that x is not on. A group that holds
// an infinity or a NaN gets the scale NaN: it reads back as NaN, its codes stay finite. 4.5 bits an element.
//
// Layout. buf: [layers][cache rows][kv heads][ceil(cache_len / 16)] records of 16 positions, 18 hd bytes each:
//   K codes [16][hd / 2 bytes] | V codes [16][hd / 2 bytes] | K scales [16 G] bf16 | V scales [16 G] bf16,  G = hd / 32
// so any run of positions is one contiguous, 16-byte aligned piece (one bulk copy) with its scales beside its codes. The
// order inside a record is the one in which tensor-core fragments (m16n8k16) are read from shared memory without bank
// conflicts (position j = 4 i + (t ^ (3 if i odd)) is the i-th of the four positions that lane-in-quad t owns):
//   K word (t', slot): dims 32 g + 8 t' .. + 7 at byte  j hd / 2 + (t' G + slot) 4, the first in the lowest nibble
//   V half (q, slot):  dims 32 g + 4 q .. + 3 at byte   j hd / 2 + ((q ^ sw) G + slot) 2,  sw = 4 (j >> 1 & 1) at hd 128
//   scale (j, slot):   element (4 t + i) G + slot
// slot orders the groups so that group g and g + G / 2 (the two dims of a RoPE pair) are neighbours: 0, 2, 1, 3 at hd 128.
#include <atomic>
#include <type_traits>

#include "common.cuh"

namespace a8 {

constexpr int KERNEL_ID_KV4_STORE = 9;
constexpr int KERNEL_ID_KV4_LOAD = 10;
constexpr int KERNEL_ID_KV4_ATTN = 11;
constexpr int KV4_BLK = 16;                              // positions a record holds

struct Kv4View {
  uint8_t* base;          // this layer's first record
  int cache_rows, nkv, cache_len, nblk;
};

template <int HD>
struct Kv4 {
  static constexpr int G = HD / 32;                      // scale groups of a head
  static constexpr int REC = 18 * HD;
  static constexpr int V0 = 8 * HD, KS0 = 16 * HD, VS0 = 17 * HD;
  __device__ static __forceinline__ int slot(int grp) { return (grp % (G / 2)) * 2 + grp / (G / 2); }
  __device__ static __forceinline__ int kword(int j, int t8, int s) { return j * (HD / 2) + (t8 * G + s) * 4; }
  __device__ static __forceinline__ int vsw(int j) { return G == 4 ? ((j >> 1) & 1) * 4 : 0; }
  __device__ static __forceinline__ int vhalf(int j, int q, int s) {
    return V0 + j * (HD / 2) + ((q ^ vsw(j)) * G + s) * 2;
  }
  __device__ static __forceinline__ int scale(int j, int s) {
    const int i = j >> 2, t = (j & 3) ^ ((i & 1) * 3);
    return ((t * 4 + i) * G + s) * 2;                    // + KS0 or VS0
  }
};

__device__ __forceinline__ uint8_t* kv4_rec(const Kv4View& c, int rec, int row, int h, int blk) {
  return c.base + (((size_t)row * c.nkv + h) * c.nblk + blk) * (size_t)rec;
}

// ------------------------------------------------------------------------------------------------ store
struct Kv4StoreArgs {
  Kv4View c;
  const __nv_bfloat16* qkv;
  int ld, nq;
  const __nv_bfloat16 *cos, *sin;   // [npos, hd], or null: no rotation
  int npos;
  const int *pos, *slot;
  int rows, ring;
  __nv_bfloat16* q;
  int ldq;
};

// Bound: at many rows by memory with the quantiser's instructions right behind it (16,381 rows of 48 heads, hd 128: 354 MB in
// 73 us, 4.8 TB/s); a tick's 192 rows by the launch, 2.4 us. Warps of query heads alone skip the quantiser.

// The 8 codes of this thread's dims (w: bf16 pairs; nibble n = dim n) and the scale of the group that they share with the
// other three lanes of the aligned four. rint(x / s) without a division an element: x (1 / s) is off by under 2^-21 of
// itself, and snapped to a multiple of 2^-10 it is on the right side of every border: a quotient that is not on the
// border n + 1/2 is at least 2^-9.9 from it (x - (n + 1/2) s is a whole multiple of a 12-bit grid), one that is on it snaps
// to it exactly.
__device__ __forceinline__ uint32_t kv4_quant8(const uint32_t* w, uint32_t& scale_bits) {
  // (as whole numbers the magnitudes order infinities and NaN above all)
  uint32_t mm = __vmaxu2(__vmaxu2(w[0] & 0x7FFF7FFFu, w[1] & 0x7FFF7FFFu), __vmaxu2(w[2] & 0x7FFF7FFFu, w[3] & 0x7FFF7FFFu));
  mm = __vmaxu2(mm, __shfl_xor_sync(0xffffffffu, mm, 1));
  mm = __vmaxu2(mm, __shfl_xor_sync(0xffffffffu, mm, 2));
  const uint32_t top = max(mm & 0xFFFFu, mm >> 16);
  if (top >= 0x7F80u) {
    scale_bits = 0x7FFFu;
    return 0x88888888u;
  }
  const __nv_bfloat16 sb = __float2bfloat16_rn(__fdiv_rn(__uint_as_float(top << 16), 7.0f));
  scale_bits = __bfloat16_as_ushort(sb);
  float s = __bfloat162float(sb);
  if (s == 0.f) return 0x88888888u;
  float x[8];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const float2 d = unpack_bf16(w[k]);
    x[2 * k] = d.x;
    x[2 * k + 1] = d.y;
  }
  if (s < 0x1p-100f) {
    // a scale of few bits may be well below max|x| / 7: clamp; and keep 1 / s finite (both exact)
    s *= 0x1p100f;
#pragma unroll
    for (int n = 0; n < 8; ++n) x[n] = fminf(fmaxf(x[n] * 0x1p100f, -7.f * s), 7.f * s);
  }
  const float inv = __fdiv_rn(1.f, s);
  uint32_t c = 0;
#pragma unroll
  for (int n = 0; n < 8; ++n) {
    const float y = fmaf(x[n], inv, 12288.f) - 12288.f;                     // 1.5 x 2^13: whole multiples of 2^-10
    c |= (__float_as_uint(y + 12582920.f) & 15u) << (4 * n);                // 1.5 x 2^23 + 8: rint(y) + 8 in the low bits
  }
  return c;
}

// The (row, head, part of TPH) of this thread in the row-major sequence of all; false behind the last (the row is clamped).
// The 64-bit division is the block's, the thread's is of a small number.
template <int TPH>
__device__ __forceinline__ bool kv4_item(int heads, int rows, int& row, int& head, int& sub) {
  const unsigned per = (unsigned)heads * TPH;
  const unsigned long long first = (unsigned long long)blockIdx.x * blockDim.x;
  const unsigned long long r0 = first / per;
  const unsigned t = unsigned(first - r0 * per) + threadIdx.x, up = t / per, in = t - up * per;
  const unsigned long long r = r0 + up;
  sub = in % TPH;
  head = in / TPH;
  row = int(min(r, (unsigned long long)rows - 1));
  return r < (unsigned long long)rows;
}

// One thread: 8 dims of a head and the 8 dims hd / 2 further (a RoPE pair each) of one row's q, k or v head; the scale of
// a 32-dim group needs the maximum over four neighbouring threads.
template <int HD>
__global__ void __launch_bounds__(256) k_kv4_store(const Kv4StoreArgs a) {
  using F = Kv4<HD>;
  constexpr int TPH = HD / 16;
  pdl_launch();
  pdl_wait();
  const int heads = a.nq + 2 * a.c.nkv;
  int row, head, sub;
  bool live = kv4_item<TPH>(heads, a.rows, row, head, sub);
  const int d0 = sub * 8;
  const __nv_bfloat16* x = a.qkv + (size_t)row * a.ld + head * HD + d0;
  uint32_t lo[4], hi[4];                                 // (on their way while the position is read)
  *reinterpret_cast<uint4*>(lo) = *reinterpret_cast<const uint4*>(x);
  *reinterpret_cast<uint4*>(hi) = *reinterpret_cast<const uint4*>(x + HD / 2);
  const int pos = a.pos[row];
  const int slot = a.slot != nullptr ? a.slot[row] : row;
  const int at = a.ring > 0 ? pos % a.ring : pos;
  live = live && pos >= 0;                               // a row at a negative position is padding
  if (live && (at >= a.c.cache_len || slot < 0 || slot >= a.c.cache_rows || (a.cos != nullptr && pos >= a.npos))) {
    if (sub == 0 && head == 0) set_error(ERR_BOUNDS, KERNEL_ID_KV4_STORE, row);
    live = false;
  }
  if (live && a.cos != nullptr && head < a.nq + a.c.nkv) {
    uint32_t cw[4], sw[4];
    *reinterpret_cast<uint4*>(cw) = *reinterpret_cast<const uint4*>(a.cos + (size_t)pos * HD + d0);
    *reinterpret_cast<uint4*>(sw) = *reinterpret_cast<const uint4*>(a.sin + (size_t)pos * HD + d0);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      // products of two bf16 are exact in fp32: the rotation is one fp32 rounding and one to bf16, what a bf16 cache
      // would hold
      const float2 u = unpack_bf16(lo[k]), v = unpack_bf16(hi[k]), c = unpack_bf16(cw[k]), s = unpack_bf16(sw[k]);
      lo[k] = pack_bf16(u.x * c.x - v.x * s.x, u.y * c.y - v.y * s.y);
      hi[k] = pack_bf16(v.x * c.x + u.x * s.x, v.y * c.y + u.y * s.y);
    }
  }
  if (live && head < a.nq) {
    __nv_bfloat16* y = a.q + (size_t)row * a.ldq + head * HD + d0;
    *reinterpret_cast<uint4*>(y) = *reinterpret_cast<const uint4*>(lo);
    *reinterpret_cast<uint4*>(y + HD / 2) = *reinterpret_cast<const uint4*>(hi);
  }
  // (a group's maximum takes every lane of its warp; warps of query heads alone are done)
  if (!__any_sync(0xffffffffu, live && head >= a.nq)) return;
  uint32_t slo, shi;
  const uint32_t wlo = kv4_quant8(lo, slo), whi = kv4_quant8(hi, shi);
  if (!live || head < a.nq) return;
  const bool isv = head >= a.nq + a.c.nkv;
  const int h = head - a.nq - (isv ? a.c.nkv : 0);
  const int t8 = sub & 3, s0 = (sub >> 2) * 2, j = at % KV4_BLK;
  uint8_t* rec = kv4_rec(a.c, F::REC, slot, h, at / KV4_BLK);
  if (!isv) {
    *reinterpret_cast<uint2*>(rec + F::kword(j, t8, s0)) = make_uint2(wlo, whi);
  } else {
    *reinterpret_cast<uint32_t*>(rec + F::vhalf(j, 2 * t8, s0)) = (wlo & 0xFFFFu) | (whi << 16);
    *reinterpret_cast<uint32_t*>(rec + F::vhalf(j, 2 * t8 + 1, s0)) = (wlo >> 16) | (whi & 0xFFFF0000u);
  }
  if (t8 == 0)
    *reinterpret_cast<uint32_t*>(rec + (isv ? F::VS0 : F::KS0) + F::scale(j, s0)) = slo | (shi << 16);
}

// ------------------------------------------------------------------------------------------------ load
struct Kv4LoadArgs {
  Kv4View c;
  const int *pos, *slot;
  int rows;
  __nv_bfloat16 *k, *v;   // either may be null
  int ldk, ldv;
};

// Codes n of the two 16-bit halves of w as bf16: the nibble u is the low mantissa bits of 128 + u; less 136 is exact.
template <int N>
__device__ __forceinline__ uint32_t kv4_pair(uint32_t w) {
  uint32_t d;
  asm("{\n\t.reg .b32 t;\n\tlop3.b32 t, %1, 0x000F000F, 0x43004300, 0xEA;\n\tadd.rn.bf16x2 %0, t, %2;\n\t}"
      : "=r"(d)
      : "r"(w >> (4 * N)), "r"(0xC308C308u));
  return d;
}
// bf16(code * s) of the 8 nibbles of w: a product of bf16 numbers rounded once
__device__ __forceinline__ uint4 kv4_deq8(uint32_t w, uint32_t s_low) {
  const uint32_t ss = __byte_perm(s_low, 0, 0x1010);
  const __nv_bfloat162 s2 = *reinterpret_cast<const __nv_bfloat162*>(&ss);
  const uint32_t c[4] = {kv4_pair<0>(w), kv4_pair<1>(w), kv4_pair<2>(w), kv4_pair<3>(w)};   // dims (n, n + 4)
  uint32_t v[4];
#pragma unroll
  for (int n = 0; n < 4; ++n) {
    const __nv_bfloat162 x = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&c[n]), s2);
    v[n] = *reinterpret_cast<const uint32_t*>(&x);
  }
  return make_uint4(__byte_perm(v[0], v[1], 0x5410), __byte_perm(v[2], v[3], 0x5410), __byte_perm(v[0], v[1], 0x7632),
                    __byte_perm(v[2], v[3], 0x7632));
}

// The inverse map, one thread the same 8 + 8 dims of a row's K and V head: bound by memory (65,533 rows x 8 heads, hd 128:
// 344 MB in 57 us, 6.1 TB/s, 0.93 of a copy's rate); streaming stores and more rows a thread changed nothing.
template <int HD>
__global__ void __launch_bounds__(256) k_kv4_load(const Kv4LoadArgs a) {
  using F = Kv4<HD>;
  constexpr int TPH = HD / 16;
  pdl_launch();
  pdl_wait();
  int row, h, sub;
  if (!kv4_item<TPH>(a.c.nkv, a.rows, row, h, sub)) return;
  const int pos = a.pos[row];
  const int slot = a.slot != nullptr ? a.slot[row] : row;
  if (pos < 0) return;
  if (pos >= a.c.cache_len || slot < 0 || slot >= a.c.cache_rows) {
    if (sub == 0 && h == 0) set_error(ERR_BOUNDS, KERNEL_ID_KV4_LOAD, row);
    return;
  }
  const int t8 = sub & 3, s0 = (sub >> 2) * 2, j = pos % KV4_BLK;
  const uint8_t* rec = kv4_rec(a.c, F::REC, slot, h, pos / KV4_BLK);
  // both heads' words and scales are on their way before the first is used
  uint2 w = make_uint2(0, 0);
  uint32_t u0 = 0, u1 = 0, ks = 0, vs = 0;
  if (a.k != nullptr) {
    w = *reinterpret_cast<const uint2*>(rec + F::kword(j, t8, s0));
    ks = *reinterpret_cast<const uint32_t*>(rec + F::KS0 + F::scale(j, s0));
  }
  if (a.v != nullptr) {
    u0 = *reinterpret_cast<const uint32_t*>(rec + F::vhalf(j, 2 * t8, s0));
    u1 = *reinterpret_cast<const uint32_t*>(rec + F::vhalf(j, 2 * t8 + 1, s0));
    vs = *reinterpret_cast<const uint32_t*>(rec + F::VS0 + F::scale(j, s0));
  }
  if (a.k != nullptr) {
    __nv_bfloat16* y = a.k + (size_t)row * a.ldk + h * HD + sub * 8;
    *reinterpret_cast<uint4*>(y) = kv4_deq8(w.x, ks);
    *reinterpret_cast<uint4*>(y + HD / 2) = kv4_deq8(w.y, ks >> 16);
  }
  if (a.v != nullptr) {
    __nv_bfloat16* y = a.v + (size_t)row * a.ldv + h * HD + sub * 8;
    *reinterpret_cast<uint4*>(y) = kv4_deq8((u0 & 0xFFFFu) | (u1 << 16), vs);
    *reinterpret_cast<uint4*>(y + HD / 2) = kv4_deq8((u0 >> 16) | (u1 & 0xFFFF0000u), vs >> 16);
  }
}

// ------------------------------------------------------------------------------------------------ decode attention
struct Kv4AttnArgs {
  Kv4View c;
  const __nv_bfloat16* q;
  int q_stride, nq, group;
  const int *lens, *rowmap;   // decode: keys of row r: lens[r] + lens_add; cache row of row r (null: r)
  int lens_add;
  const int* blocks;          // packed prompts: [nblocks][4] = (q0, n, slot, pos0)
  int rows, max_len;
  float scale_log2;
  __nv_bfloat16* out;
  int out_stride;
  float* ws;                  // [CTAs][2][part]: a CTA's share of the units it cuts: O [group][hd], then (max, sum) [group]
  int part;
  int* counters;              // [rows * nkv] tickets, zero between calls
};

constexpr int KV4_CTAS = 148;         // one a SM
constexpr int KV4_STEP = 32;           // positions a warp takes at a time: two records
// Fewer steps than CTAs x this: fewer CTAs, so that short work is joined within a CTA. Measured with 12, 16, 24, 36, 48: one
// row of 733 keys (two heads of 23 steps) 12.8, 12.9, 9.9, 9.9, 11.3 us; 192 rows x 8 heads of 1 to 128 keys 15.9, 16.0, 16.0,
// 16.8, 19.6; long ones the same. The other side of it: one row of 768 keys (48 steps, 2 CTAs, nothing cut) takes 10.3 us, one of
// 769 (50 steps, 3 CTAs, both units cut between them) 14.7, one of 2,047 (6 CTAs) 13.6.
constexpr int KV4_CTA_STEPS = 24;
constexpr int KV4_WHOLE = 8;          // a unit of at most so many steps is not cut between warps
constexpr float KV4_LAZY = 8.f;       // a running maximum moves when a logit passes it by 2^8

template <int HD, int NT>
struct Kv4DecSmem {
  // Warps: as many as their registers (O [hd][8 NT], the queries, a record's scores) leave with little or no spilling.
  // hd 64, 192 rows of 1 to 2,047 keys: 16 warps (128 registers) 22 us, 20, 24 and 28 no better. hd 128, 3 rows x 8 heads of
  // 40,009 to 131,071 keys: 8 warps 106 us, 10 123 (the SM's quarters are uneven), 12 101, 14 121 and 16 114 (spills).
  // More than 8 query heads a kv head (NT 2), hd 64, 1,000 rows x 2 heads of 1 to 2,047 keys: 12 warps 67.4 us, 16 69.6 (spills).
  static constexpr int NW = HD == 64 ? (NT == 1 ? 16 : 12) : NT == 1 ? 12 : 8;
  // Steps in flight a warp: 148 SMs x 16 x 4 x 2.3 KB or 12 x 3 x 4.6 KB are 22 to 24 MB, well above what 6.5 TB/s times
  // the latency of a load (about 1 us) asks for; what shared memory holds beside the partials.
  static constexpr int NST = HD == 64 ? 4 : 3;
  static constexpr int RING = NST * 2 * Kv4<HD>::REC;
  static constexpr int PART = (8 * NT * HD + 16 * NT) * 4;        // bytes: O [8 NT][hd], (max, sum) [8 NT]
  static constexpr int HEADP = NW * RING;                         // first partials; the last ones go into the rings
  static constexpr int PRE = HEADP + NW * PART;                   // prefix of the rows' steps by thread
  static constexpr int META = PRE + (NW * 32 + 4) * 4;            // int [2 NW][4]: a piece's unit, its first and end step
  static constexpr int RUNS = META + 2 * NW * 4 * 4;              // int [2 NW] x 4: a unit's pieces [from, to); the pieces in
                                                                  // order; their runs
  static constexpr int WGT = RUNS + 2 * NW * 4 * 4;               // float [2 NW][8 NT]: a piece's weight in its unit
  static constexpr int BARS = WGT + 2 * NW * 8 * NT * 4;
  static constexpr int TOTAL = BARS + NW * NST * 8 + 16;
  static_assert(PART <= RING && TOTAL <= 227 * 1024 && BARS % 8 == 0, "");
};

// Two waits of a warp at once: the second barrier's state is on its way while the first one's is looked at.
__device__ __forceinline__ bool kv4_wait2(uint64_t* a, uint32_t pa, uint64_t* b, uint32_t pb, int err, int where) {
  const bool ra = mbar_try_wait(a, pa), rb = mbar_try_wait(b, pb);
  if (__all_sync(0xffffffffu, ra && rb)) return true;
  return mbar_wait_all(a, pa, err, where) && mbar_wait_all(b, pb, err, where);
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// As they stand, nibbles 0 and 2 of a half are the fp16 subnormals u 2^-24, 1 and 3 (in bits 4-7) 16 u 2^-24: exact operands
// of a product, one mask each.
constexpr uint32_t KV4_LO = 0x000F000Fu, KV4_HI = 0x00F000F0u;
constexpr float KV4_OFF_LO = 8.f * 0x1p-24f, KV4_OFF_HI = 128.f * 0x1p-24f;     // code 0 in the two forms
// The codes n of the two 16-bit halves of w (n = 0, 2: w >> 4 n; n = 1, 3: w >> 4 (n - 1)) as bf16, times 2^-6: the masked
// bits are the bf16 subnormals u 2^-133 and 16 u 2^-133, one fused multiply-add (exact) makes them (u - 8) 2^-6.
__device__ __forceinline__ uint32_t kv4_code_lo(uint32_t w) {
  uint32_t d;
  asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(w & KV4_LO), "r"(0x7F007F00u), "r"(0xBE00BE00u));   // x 2^127, - 2^-3
  return d;
}
__device__ __forceinline__ uint32_t kv4_code_hi(uint32_t w) {
  uint32_t d;
  asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(w & KV4_HI), "r"(0x7D007D00u), "r"(0xBE00BE00u));   // x 2^123, - 2^-3
  return d;
}
constexpr float KV4_O_UNIT = 64.f;    // what O is held in

__device__ __forceinline__ void kv4_mma_bf16(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// d = a b (+ c): fp16 products of one 16-dim step
__device__ __forceinline__ void mma_f16_first(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ void mma_f16(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Row r's keys and cache row; (0, -) for a row that attends nothing.
__device__ __forceinline__ int kv4_row(const Kv4AttnArgs& a, int r, int& crow) {
  crow = a.rowmap != nullptr ? a.rowmap[r] : r;
  const int n = max(0, min(a.lens[r] + a.lens_add, a.max_len));
  return crow >= 0 && crow < a.c.cache_rows ? n : 0;
}

// A place in the steps of all units (row-major, then kv head): row r, head h, step blk of nb; len keys.
struct Kv4Cursor {
  int r, h, blk, nb, len;
  const uint8_t* at;            // the step's first record
};

template <int HD>
__device__ __forceinline__ void kv4_cursor_unit(const Kv4AttnArgs& a, Kv4Cursor& c, int crow) {
  c.nb = (c.len + KV4_STEP - 1) / KV4_STEP;
  c.at = kv4_rec(a.c, Kv4<HD>::REC, crow, c.h, 2 * c.blk);
}
// On to the next unit's first step (there is one).
template <int HD>
__device__ __forceinline__ void kv4_cursor_next(const Kv4AttnArgs& a, Kv4Cursor& c) {
  int crow;
  if (++c.h == a.c.nkv) {
    c.h = 0;
    do {
      ++c.r;
      c.len = c.r < a.rows ? kv4_row(a, c.r, crow) : 1;
    } while (c.len == 0);
    if (c.r >= a.rows) return;
  } else {
    c.len = kv4_row(a, c.r, crow);
  }
  c.blk = 0;
  kv4_cursor_unit<HD>(a, c, crow);
}

// The steps (32 positions, two records) of all rows and kv heads form one sequence; CTA b of G takes the b-th of G equal
// parts of it, its warps equal parts of that: the work is even whatever the lengths. A warp runs through its steps alone
// (its own ring of bulk copies, no barrier with the others) and writes the units (a row's kv head) that lie wholly in its
// part; what it has of the unit it begins and the unit it ends within goes to shared memory, where the CTA joins its warps'
// pieces, and units that span CTAs are joined, in order, by the CTA that comes last.
//   S = Q K^T (M: the query heads of the kv head, N: 8 keys), O^T = V^T P^T (M: 16 dims, K: 16 keys): the accumulator
//   layout of S is the B operand of the second product, no exchange between lanes. Codes are operands as they stand: K's
//   nibbles are masked to fp16 subnormals u 2^-24 (code + 8 = u: 8 times the query's sum is taken off each group's product
//   in fp32, then it is scaled by s_k); V's become bf16 by a mask and a fused multiply-add; P is multiplied by s_v in fp32
//   before its rounding to bf16, whose range holds the product whatever the scale (fp16 would take a running power of two of
//   the scales); it is the rounding that the bf16 cache's decode attention gives its weights. The query is fp16, scaled by a
//   power of two (8 bits in 11).
//   Running maximum per head, moved only when a logit passes it by 2^8 (then O and the sum are rescaled); sums and O fp32.
// Why mma.sync and not tcgen05: up to 16 query heads share a kv head, a 128-row tile would be an eighth full at best, and
// its operands would have to be written to shared memory as 16-bit values; here they never leave registers.
// Bound: at long lengths by the instructions that unpack and scale and by their latency at four (three) warps a scheduler,
//   not by memory: about 240 warp instructions a record at hd 64, 330 at hd 128; 56 % of the issue slots of the serving call
//   below and 59 % of the long one's are taken (ALU 46 and 53 %, tensor pipe 22 and 34 %), the rest is latency. 3 rows x 8
//   heads of 40,009 to 131,071 keys, hd 128: 407 MB in 99 us, 4.1 TB/s; 1,408 rows x 2 heads of 97 to 911 keys, hd 64: 106 MB
//   in 41 us, 2.6 TB/s. 16 query heads a kv head instead of 8 (two tiles of 8, 12 warps at hd 64 and 8 at hd 128 by
//   registers): 1,000 rows x 2 heads of 1 to 2,047 keys, hd 64, 68 us against 52; 500 rows, hd 128, 71 against 54.
//   Short ones by latency: launch 2.5 us, lengths and the split 2.5, first records and queries 1.5, joining 2.5, a cut unit's
//   join 3 to 5: 192 rows of 1 to 2,047 keys 22 us, one row of 733 keys 9.9, 192 rows x 8 heads of 1 to 128 keys (hd 128)
//   14.8.
template <int HD, int NT>
__global__ void __launch_bounds__(Kv4DecSmem<HD, NT>::NW * 32, 1) k_kv4_attn(const Kv4AttnArgs a) {
  using F = Kv4<HD>;
  using SM = Kv4DecSmem<HD, NT>;
  constexpr int NW = SM::NW, NST = SM::NST, G = F::G, NTHR = NW * 32;
  extern __shared__ __align__(128) uint8_t smem[];
  int* pre = reinterpret_cast<int*>(smem + SM::PRE);
  int* meta = reinterpret_cast<int*>(smem + SM::META);
  __shared__ int s_sum[32], s_runs, s_pieces, s_last[2], s_split[4], s_lost;
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31, g = lane >> 2, t = lane & 3;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + SM::BARS) + warp * NST;
  uint8_t* ring = smem + warp * SM::RING;
  pdl_launch();
  if (lane == 0)
    for (int s = 0; s < NST; ++s) mbar_init(&full[s], 1);
  fence_mbar_init();
  if (tid < 2 * NW) meta[4 * tid] = -1;
  if (tid == 0) s_lost = 0;
  pdl_wait();

  // ---- how many steps every row has: a prefix by thread (rows in equal runs), and zeros into rows without keys
  const int run = (a.rows + NTHR - 1) / NTHR;
  int mine = 0;
  bool none = false;
#pragma unroll 4
  for (int r = tid * run; r < min(a.rows, (tid + 1) * run); ++r) {
    int crow;
    const int n = kv4_row(a, r, crow);
    mine += (n + KV4_STEP - 1) / KV4_STEP;
    none = none || n == 0;
  }
  if (none)
    for (int r = tid * run; r < min(a.rows, (tid + 1) * run); ++r) {
      int crow;
      if (r % gridDim.x != blockIdx.x || kv4_row(a, r, crow) != 0) continue;
      if (a.lens[r] + a.lens_add > 0) set_error(ERR_BOUNDS, KERNEL_ID_KV4_ATTN, r);
      uint4* o = reinterpret_cast<uint4*>(a.out + (size_t)r * a.out_stride);
      for (int i = 0; i < a.nq * HD / 8; ++i) o[i] = make_uint4(0, 0, 0, 0);
    }
  int inc = mine;
#pragma unroll
  for (int k = 1; k < 32; k <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, inc, k);
    if (lane >= k) inc += up;
  }
  if (lane == 31) s_sum[warp] = inc;
  __syncthreads();
  int sums = lane < NW ? s_sum[lane] : 0;
#pragma unroll
  for (int k = 1; k < 32; k <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, sums, k);
    if (lane >= k) sums += up;
  }
  const int total = __shfl_sync(0xffffffffu, sums, 31), upto = __shfl_sync(0xffffffffu, sums, warp);
  pre[tid] = upto - s_sum[warp] + inc - mine;
  if (tid == 0) pre[NTHR] = total;
  __syncthreads();
  int T = total * a.c.nkv;                             // steps of all units
  int ctas = min((int)gridDim.x, (T + KV4_CTA_STEPS - 1) / KV4_CTA_STEPS);
  if ((int)blockIdx.x >= ctas) return;
  // the row that holds step x: its first step (at) and its steps a head (nb)
  auto locate = [&](int x, int& at, int& nb) {
    // the last thread whose rows begin at or before x, the warp looking together: every NW-th, then the NW of one
    uint32_t le = __ballot_sync(0xffffffffu, pre[lane * NW] * a.c.nkv <= x);
    int lo = (31 - __clz(le)) * NW;
    le = __ballot_sync(0xffffffffu, lane < NW && pre[lo + min(lane, NW - 1)] * a.c.nkv <= x);
    lo += 31 - __clz(le);
    int r = lo * run;
    at = pre[lo] * a.c.nkv;
    nb = pre[lo + 1] - pre[lo];
    if (run > 1)
      for (;; ++r) {
        int crow;
        nb = (kv4_row(a, r, crow) + KV4_STEP - 1) / KV4_STEP;
        if (at + nb * a.c.nkv > x) break;
        at += nb * a.c.nkv;
      }
    return r;
  };
  // Where CTA b's part begins: an equal share, moved to the nearer end of a unit that is small against it (at most half a
  // share). A cut unit costs a pass through global memory and a ticket, 3 to 5 us, an uneven share less: measured at 192
  // rows of 1 to 2,047 keys, 1,408 rows of 97 to 911 and 192 rows x 8 heads of 1 to 128: never moved 23.6, 45.1 and
  // 20.7 us; up to an eighth of a share 24.0, 41.7, 20.1; a quarter 22.5, 41.7, 16.0; half 22.1, 41.6, 15.9.
  // Then warp w's: the CTA's part in equal shares, moved likewise where units are few steps (joining a unit's pieces costs
  // about 2.5 us, a step too many in a warp 0.5): 192 rows x 8 heads of 1 to 128 keys 15.9 us cut, 14.6 whole.
  // (No part is empty: places a share apart move by at most a quarter of one.)
  const int share = T / ctas;
  auto moved = [&](int x, int most) {
    int at, nb;
    locate(x, at, nb);
    const int in = (x - at) % nb;
    return nb > most ? x : 2 * in < nb ? x - in : x - in + nb;
  };
  auto begin = [&](int b) {
    const int x = int((long long)T * b / ctas);
    return b == 0 || b == ctas ? x : moved(x, share / 2);
  };
  int b0 = begin(blockIdx.x), b1 = begin(blockIdx.x + 1), w0, w1;
  auto own = [&](int& w0, int& w1) {
    w0 = b0 + int((long long)(b1 - b0) * warp / NW);
    w1 = b0 + int((long long)(b1 - b0) * (warp + 1) / NW);
    if (T <= (long long)KV4_WHOLE * a.rows * a.c.nkv) {
      if (warp > 0) w0 = max(b0, moved(w0, KV4_WHOLE));
      if (warp < NW - 1) w1 = min(b1, moved(w1, KV4_WHOLE));
    }
  };
  own(w0, w1);
  if (tid == 0) {                                      // (not in registers until the join)
    s_split[0] = b0;
    s_split[1] = b1;
    s_split[2] = T;
    s_split[3] = ctas;
  }
  const int n = w1 - w0;
  bool pieces = false;                                 // of units that other warps share

  if (n > 0) {
    // ---- where the warp's part begins
    Kv4Cursor cc;
    {
      int at, crow;
      cc.r = locate(w0, at, cc.nb);
      cc.len = kv4_row(a, cc.r, crow);
      cc.h = (w0 - at) / cc.nb;
      cc.blk = (w0 - at) % cc.nb;
      kv4_cursor_unit<HD>(a, cc, crow);
    }
    Kv4Cursor pc = cc;
    int issued = 0;
    auto issue = [&](int s) {
      if (lane == 0) {
        const uint32_t bytes = (pc.len - pc.blk * KV4_STEP > KV4_BLK ? 2 : 1) * F::REC;
        mbar_arrive_expect_tx(&full[s], bytes);
        bulk_load(ring + s * 2 * F::REC, pc.at, bytes, &full[s]);
      }
      ++issued;
      pc.at += 2 * F::REC;
      if (++pc.blk == pc.nb && issued < n) kv4_cursor_next<HD>(a, pc);
    };
    for (int s = 0; s < NST && s < n; ++s) issue(s);

    uint32_t qa[G][2][4];                              // A operands; with one tile of heads rows 8-15 repeat rows 0-7
    float o[NT][G][2][4], m[NT], l[NT], qs[NT], off[NT][G];
    int slot = 0, ph = 0;                              // ring position of the next step
    bool ok = true;
    // this lane's places in a record: K words of its key in the first half (the second: 8 positions on), scales, and V
    // words of its even and odd positions
    const int kw = (4 * (g & 1) + ((g & 1) ? (g >> 1) ^ 3 : g >> 1)) * (HD / 2) + t * (4 * G);
    const int ve = F::vhalf(t, g, 0), vo = F::vhalf(4 + (t ^ 3), g, 0), sc0 = t * (8 * G);
    auto sf2 = [](uint32_t x, uint32_t y, int s) {     // two bf16 scales as fp32
      return (s & 1) ? make_float2(__uint_as_float(x & 0xFFFF0000u), __uint_as_float(y & 0xFFFF0000u))
                     : make_float2(__uint_as_float(x << 16), __uint_as_float(y << 16));
    };
    // S of a record: v[u][h] of query head g + 8 u and this lane's keys (2 h, 2 h + 1), in units of qs
    auto scores = [&](const uint8_t* rec, float2 (&v)[NT][2]) {
      uint32_t ks[4][G / 2];
      if constexpr (G == 4) {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const uint4 x = *reinterpret_cast<const uint4*>(rec + sc0 + F::KS0 + k * 16);
          ks[2 * k][0] = x.x; ks[2 * k][1] = x.y; ks[2 * k + 1][0] = x.z; ks[2 * k + 1][1] = x.w;
        }
      } else {
        const uint4 x = *reinterpret_cast<const uint4*>(rec + sc0 + F::KS0);
        ks[0][0] = x.x; ks[1][0] = x.y; ks[2][0] = x.z; ks[3][0] = x.w;
      }
#pragma unroll
      for (int nb = 0; nb < 2; ++nb) {
        uint32_t w[G];
        if constexpr (G == 4) {
          const uint4 x = *reinterpret_cast<const uint4*>(rec + kw + nb * 8 * (HD / 2));
          w[0] = x.x; w[1] = x.y; w[2] = x.z; w[3] = x.w;
        } else {
          const uint2 x = *reinterpret_cast<const uint2*>(rec + kw + nb * 8 * (HD / 2));
          w[0] = x.x; w[1] = x.y;
        }
#pragma unroll
        for (int s = 0; s < G; ++s) {
          float acc[4];
          mma_f16_first(acc, qa[s][0], w[s] & KV4_LO, w[s] & KV4_HI);
          const uint32_t w8 = w[s] >> 8;
          mma_f16(acc, qa[s][1], w8 & KV4_LO, w8 & KV4_HI);
          const float2 sc = sf2(ks[2 * nb][s >> 1], ks[2 * nb + 1][s >> 1], s);
#pragma unroll
          for (int u = 0; u < NT; ++u) {
            const float2 d = make_float2(acc[2 * u] - off[u][s], acc[2 * u + 1] - off[u][s]);
            v[u][nb] = s == 0 ? fmul2(d, sc) : ffma2(d, sc, v[u][nb]);
          }
        }
      }
    };
    // the running maximum m (in logits of base 2) moves only when a logit passes it by 2^8: p stays below 2^8
    auto raise = [&](const float2 (&v)[2][NT][2]) {
      bool over = false;
      float mx[NT];
#pragma unroll
      for (int u = 0; u < NT; ++u) {
        mx[u] = fmaxf(fmaxf(fmaxf(v[0][u][0].x, v[0][u][0].y), fmaxf(v[0][u][1].x, v[0][u][1].y)),
                      fmaxf(fmaxf(v[1][u][0].x, v[1][u][0].y), fmaxf(v[1][u][1].x, v[1][u][1].y))) * qs[u];
        over = over || mx[u] > m[u] + KV4_LAZY;
      }
      if (__any_sync(0xffffffffu, over)) {
#pragma unroll
        for (int u = 0; u < NT; ++u) {
          mx[u] = fmaxf(mx[u], __shfl_xor_sync(0xffffffffu, mx[u], 1));
          mx[u] = fmaxf(mx[u], __shfl_xor_sync(0xffffffffu, mx[u], 2));
          const float nm = fmaxf(m[u], mx[u]);
          const float al = m[u] == -INFINITY ? 0.f : ex2(m[u] - nm);
          m[u] = nm;
          l[u] *= al;
          const float c0 = __shfl_sync(0xffffffffu, al, 8 * t), c1 = __shfl_sync(0xffffffffu, al, 8 * t + 4);
#pragma unroll
          for (int s = 0; s < G; ++s)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              o[u][s][k][0] *= c0;
              o[u][s][k][1] *= c1;
              o[u][s][k][2] *= c0;
              o[u][s][k][3] *= c1;
            }
        }
      }
    };
    // O^T += V^T P^T of a record; CUT: only its first `keys` positions count
    auto values = [&](auto cut, const uint8_t* rec, float2 (&v)[NT][2], int keys) {
#pragma unroll
      for (int u = 0; u < NT; ++u)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          v[u][k].x = ex2(fmaf(v[u][k].x, qs[u], -m[u]));
          v[u][k].y = ex2(fmaf(v[u][k].y, qs[u], -m[u]));
          l[u] += v[u][k].x + v[u][k].y;
        }
      uint32_t vs[4][G / 2], vw[4][G / 2];             // this lane's scales; dims 4 g .. + 3 of every group of its keys
      if constexpr (G == 4) {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const uint4 y = *reinterpret_cast<const uint4*>(rec + sc0 + F::VS0 + k * 16);
          vs[2 * k][0] = y.x; vs[2 * k][1] = y.y; vs[2 * k + 1][0] = y.z; vs[2 * k + 1][1] = y.w;
        }
      } else {
        const uint4 y = *reinterpret_cast<const uint4*>(rec + sc0 + F::VS0);
        vs[0][0] = y.x; vs[1][0] = y.y; vs[2][0] = y.z; vs[3][0] = y.w;
      }
      if constexpr (decltype(cut)::value) {
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (4 * k + ((k & 1) ? t ^ 3 : t) >= keys)
#pragma unroll
            for (int s = 0; s < G / 2; ++s) vs[k][s] = 0u;
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint8_t* at = rec + ((k & 1) ? vo : ve) + (k >> 1) * 8 * (HD / 2);
        if constexpr (G == 4) {
          const uint2 x = *reinterpret_cast<const uint2*>(at);
          vw[k][0] = x.x;
          vw[k][1] = x.y;
        } else {
          vw[k][0] = *reinterpret_cast<const uint32_t*>(at);
        }
      }
#pragma unroll
      for (int s = 0; s < G; ++s) {
        const uint32_t u01 = __byte_perm(vw[0][s >> 1], vw[1][s >> 1], (s & 1) ? 0x7632 : 0x5410);
        const uint32_t u23 = __byte_perm(vw[2][s >> 1], vw[3][s >> 1], (s & 1) ? 0x7632 : 0x5410);
        uint32_t b[NT][2];
#pragma unroll
        for (int u = 0; u < NT; ++u) {
          const float2 p0 = fmul2(v[u][0], sf2(vs[0][s >> 1], vs[1][s >> 1], s)),
                       p1 = fmul2(v[u][1], sf2(vs[2][s >> 1], vs[3][s >> 1], s));
          b[u][0] = pack_bf16(p0.x, p0.y);
          b[u][1] = pack_bf16(p1.x, p1.y);
        }
        const uint32_t lo[4] = {kv4_code_lo(u01), kv4_code_hi(u01), kv4_code_lo(u23), kv4_code_hi(u23)};
        const uint32_t hi[4] = {kv4_code_lo(u01 >> 8), kv4_code_hi(u01 >> 8), kv4_code_lo(u23 >> 8), kv4_code_hi(u23 >> 8)};
#pragma unroll
        for (int u = 0; u < NT; ++u) {
          kv4_mma_bf16(o[u][s][0], lo, b[u][0], b[u][1]);
          kv4_mma_bf16(o[u][s][1], hi, b[u][0], b[u][1]);
        }
      }
    };
    auto arrived = [&] { return mbar_wait_all(&full[slot], ph, ERR_TIMEOUT_FULL, KERNEL_ID_KV4_ATTN); };
    auto step = [&] {
      if (++slot == NST) {
        slot = 0;
        ph ^= 1;
      }
    };

    for (int i = 0; i < n && ok;) {
      // ---- a segment: the warp's steps of one unit. The query heads as fp16: scaled by a power of two so that the
      // largest is in [2^7, 2^8) (exact down to 2^-18 of it), every other dim divided by 16 against its 16 u, and what
      // the offsets of the codes add up to in each group
      const int first = cc.blk, seg = min(cc.nb - cc.blk, n - i);
#pragma unroll
      for (int u = 0; u < NT; ++u) {
        m[u] = -INFINITY;
        l[u] = 0.f;
        const bool have = g + 8 * u < a.group;
        const __nv_bfloat16* qr = a.q + (size_t)cc.r * a.q_stride + (cc.h * a.group + g + 8 * u) * HD + 8 * t;
        uint4 x[G];
        uint32_t top = 0;
#pragma unroll
        for (int s = 0; s < G; ++s) {
          x[s] = have ? *reinterpret_cast<const uint4*>(qr + 32 * ((s & 1) * (G / 2) + s / 2)) : make_uint4(0, 0, 0, 0);
          const uint32_t e[4] = {x[s].x, x[s].y, x[s].z, x[s].w};
#pragma unroll
          for (int k = 0; k < 4; ++k) top = max(top, max(e[k] & 0x7FFFu, (e[k] >> 16) & 0x7FFFu));
        }
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const uint32_t ex = max(top >> 7, 8u);
        const float up = __uint_as_float((261u - ex) << 23);
        // (never 0, which would make a masked -infinity NaN)
        qs[u] = fmaxf(a.scale_log2 * 0x1p24f * __uint_as_float((ex - 7u) << 23), 0x1p-126f);
#pragma unroll
        for (int s = 0; s < G; ++s) {
          const float2 d01 = unpack_bf16(x[s].x), d23 = unpack_bf16(x[s].y), d45 = unpack_bf16(x[s].z),
                       d67 = unpack_bf16(x[s].w);
          // dims (n, n + 4) of the word's eight
#pragma unroll
          for (int w = u; w < 2; w += NT) {
            qa[s][0][w] = pack_f16(d01.x * up, d45.x * up);
            qa[s][0][2 + w] = pack_f16(d01.y * up * 0.0625f, d45.y * up * 0.0625f);
            qa[s][1][w] = pack_f16(d23.x * up, d67.x * up);
            qa[s][1][2 + w] = pack_f16(d23.y * up * 0.0625f, d67.y * up * 0.0625f);
          }
          const float2 e0 = unpack_f16(qa[s][0][u]), e1 = unpack_f16(qa[s][1][u]), h0 = unpack_f16(qa[s][0][2 + u]),
                       h1 = unpack_f16(qa[s][1][2 + u]);
          float f = KV4_OFF_LO * ((e0.x + e0.y) + (e1.x + e1.y)) + KV4_OFF_HI * ((h0.x + h0.y) + (h1.x + h1.y));
          f += __shfl_xor_sync(0xffffffffu, f, 1);
          f += __shfl_xor_sync(0xffffffffu, f, 2);
          off[u][s] = f;
#pragma unroll
          for (int k = 0; k < 2; ++k) o[u][s][k][0] = o[u][s][k][1] = o[u][s][k][2] = o[u][s][k][3] = 0.f;
        }
      }
      // (only the last step can hold positions past the row's end; the others are spared the masks)
      auto one = [&](auto cut, int keys) {
        if (!(ok = arrived())) return;
        const uint8_t* rec = ring + slot * 2 * F::REC;
        float2 v[2][NT][2];
        scores(rec, v[0]);
        scores(rec + F::REC, v[1]);
        if constexpr (decltype(cut)::value) {
          // whatever the records hold there (their scales may be NaN) counts for nothing
#pragma unroll
          for (int r = 0; r < 2; ++r)
#pragma unroll
            for (int k = 0; k < 4; ++k)
              if (r * KV4_BLK + 4 * k + ((k & 1) ? t ^ 3 : t) >= keys)
#pragma unroll
                for (int u = 0; u < NT; ++u) ((k & 1) ? v[r][u][k >> 1].y : v[r][u][k >> 1].x) = -INFINITY;
        }
        raise(v);
        values(cut, rec, v[0], keys);
        values(cut, rec + F::REC, v[1], keys - KV4_BLK);
        __syncwarp();
        if (issued < n) issue(slot);
        step();
      };
      for (int j = 1; ok && j < seg; ++j) one(std::false_type(), KV4_STEP);
      if (ok) one(std::true_type(), cc.len - (first + seg - 1) * KV4_STEP);
      if (!ok) break;
      // ---- the segment's result: the unit's, or a piece of it
      i += seg;
      cc.blk += seg;
#pragma unroll
      for (int u = 0; u < NT; ++u) {
        l[u] += __shfl_xor_sync(0xffffffffu, l[u], 1);
        l[u] += __shfl_xor_sync(0xffffffffu, l[u], 2);
      }
      const bool whole = seg == cc.nb;
      pieces = pieces || !whole;
      const int piece = i == seg ? 0 : 1;              // the warp's first segment, or a later one (then its last)
      float* part = reinterpret_cast<float*>(piece == 0 ? smem + SM::HEADP + warp * SM::PART : ring);
#pragma unroll
      for (int u = 0; u < NT; ++u) {
        const float l0 = __shfl_sync(0xffffffffu, l[u], 8 * t), l1 = __shfl_sync(0xffffffffu, l[u], 8 * t + 4);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int qh = 2 * t + e + 8 * u;
          if (qh >= a.group) continue;
          const float inv = KV4_O_UNIT / (e ? l1 : l0);
#pragma unroll
          for (int s = 0; s < G; ++s) {
            const int d = 32 * ((s & 1) * (G / 2) + s / 2) + 4 * g;
            const float4 x = make_float4(o[u][s][0][e], o[u][s][0][2 + e], o[u][s][1][e], o[u][s][1][2 + e]);
            if (whole)
              *reinterpret_cast<uint2*>(a.out + (size_t)cc.r * a.out_stride + (cc.h * a.group + qh) * HD + d) =
                  make_uint2(pack_bf16(x.x * inv, x.y * inv), pack_bf16(x.z * inv, x.w * inv));
            else
              *reinterpret_cast<float4*>(part + qh * HD + d) = x;
          }
        }
        if (!whole && t == 0) {
          part[8 * NT * HD + 2 * (g + 8 * u)] = m[u];
          part[8 * NT * HD + 2 * (g + 8 * u) + 1] = l[u];
        }
      }
      if (!whole && lane == 0) {
        int* e = meta + 4 * (2 * warp + piece);
        e[0] = cc.r * a.c.nkv + cc.h;
        e[1] = w0 + i - cc.blk;                        // the unit's first step, and its end
        e[2] = e[1] + cc.nb;
      }
      if (i < n) kv4_cursor_next<HD>(a, cc);
    }
    if (!ok) {                                         // a copy did not arrive: wait (bounded) for what is in flight
      for (int s = 0; s < NST; ++s) mbar_wait_all(&full[s], ph ^ (s < slot), ERR_TIMEOUT_FULL, KERNEL_ID_KV4_ATTN);
      pieces = true;
      if (lane == 0) s_lost = 1;
    }
  }
  if (!__syncthreads_or(pieces)) return;
  b0 = s_split[0];
  b1 = s_split[1];
  T = s_split[2];
  ctas = s_split[3];
  if (s_lost) {
    // Units that warps share still get every warp's piece, a NaN from one that gave up: every CTA takes its tickets, and the
    // counters come back to zero.
    own(w0, w1);
    for (int piece = 0; piece < 2 && w0 < w1; ++piece) {
      const int x = piece == 0 ? w0 : w1 - 1;
      int at, nb, *e = meta + 4 * (2 * warp + piece);
      const int r = locate(x, at, nb), h = (x - at) / nb, us = at + h * nb;
      if ((us >= w0 && us + nb <= w1) || e[0] >= 0 || (piece == 1 && us <= w0)) continue;      // (whole, there, the first again)
      float* part = reinterpret_cast<float*>(piece == 0 ? smem + SM::HEADP + warp * SM::PART : ring) + 8 * NT * HD;
      if (lane < 8 * NT) *reinterpret_cast<float2*>(part + 2 * lane) = make_float2(0.f, __int_as_float(0x7FFFFFFF));
      __syncwarp();
      if (lane == 0) {
        e[0] = r * a.c.nkv + h;
        e[1] = us;
        e[2] = us + nb;
      }
    }
    __syncthreads();
  }

  // ---- join the warps' pieces of each unit, in key order: the runs of pieces of one unit, each piece's weight
  int *runs = reinterpret_cast<int*>(smem + SM::RUNS), *list = runs + 4 * NW, *rof = list + 2 * NW;
  float* wgt = reinterpret_cast<float*>(smem + SM::WGT);
  auto piece_at = [&](int e) {
    return reinterpret_cast<const float*>((e & 1) ? smem + (e >> 1) * SM::RING : smem + SM::HEADP + (e >> 1) * SM::PART);
  };
  constexpr int ML = 8 * NT * HD;                      // (max, sum) behind a piece's O
  if (warp == 0) {
    static_assert(2 * NW <= 64, "");
    uint64_t valid = 0, heads = 0;
    bool starts[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int e = lane + 32 * k;
      valid |= uint64_t(__ballot_sync(0xffffffffu, e < 2 * NW && meta[4 * min(e, 2 * NW - 1)] >= 0)) << (32 * k);
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int e = lane + 32 * k;
      const uint64_t before = valid & ((1ull << e) - 1);
      starts[k] = (valid >> e & 1) && (before == 0 || meta[4 * (63 - __clzll(before))] != meta[4 * e]);
      heads |= uint64_t(__ballot_sync(0xffffffffu, starts[k])) << (32 * k);
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int e = lane + 32 * k;
      const uint64_t below = (1ull << e) - 1;
      const int at = __popcll(valid & below);
      if (valid >> e & 1) {
        list[at] = e;
        rof[at] = __popcll(heads & (2 * below + 1)) - 1;
      }
      if (starts[k]) {
        const uint64_t later = heads & ~(2 * below + 1);
        const int r = __popcll(heads & below);
        runs[2 * r] = at;
        runs[2 * r + 1] = later ? __popcll(valid & ((1ull << (__ffsll(later) - 1)) - 1)) : __popcll(valid);
      }
    }
    if (lane == 0) {
      s_runs = __popcll(heads);
      s_pieces = __popcll(valid);
    }
  }
  __syncthreads();
  const int nruns = s_runs;
  for (int i = tid; i < s_pieces * a.group; i += NTHR) {
    const int p = i / a.group, qh = i % a.group, from = runs[2 * rof[p]], to = runs[2 * rof[p] + 1];
    float M = -INFINITY;
#pragma unroll 4
    for (int e = from; e < to; ++e) M = fmaxf(M, piece_at(list[e])[ML + 2 * qh]);
    wgt[p * 8 * NT + qh] = ex2(piece_at(list[p])[ML + 2 * qh] - M);
  }
  __syncthreads();
  auto cta_of = [&](int x) { return int(((long long)(x + 1) * ctas - 1) / T); };    // by equal shares
  const int nel = a.group * HD / 4;                    // float4 elements of a unit
  // few elements: 2 or 4 neighbouring lanes share one, each every 2nd or 4th piece of it
  const int share_ = nruns * nel * 4 <= NTHR ? 4 : nruns * nel * 2 <= NTHR ? 2 : 1, part_ = tid & (share_ - 1);
  for (int i0 = 0; i0 < nruns * nel; i0 += NTHR / share_) {
    const int i = i0 + tid / share_;
    const bool live = i < nruns * nel;
    const int k = live ? i / nel : 0, el = live ? i % nel : 0, qh = el / (HD / 4), from = runs[2 * k], to = runs[2 * k + 1];
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
    float L = 0.f, M = -INFINITY;
    if (live) {
#pragma unroll 4
      for (int p = from + part_; p < to; p += share_) {
        const float* src = piece_at(list[p]);
        const float f = wgt[p * 8 * NT + qh];
        const float4 y = reinterpret_cast<const float4*>(src)[el];
        const float2 ml = *reinterpret_cast<const float2*>(src + ML + 2 * qh);
        x.x += f * y.x;
        x.y += f * y.y;
        x.z += f * y.z;
        x.w += f * y.w;
        L += f * ml.y;
        M = fmaxf(M, ml.x);
      }
    }
    for (int d = 1; d < share_; d <<= 1) {
      x.x += __shfl_xor_sync(0xffffffffu, x.x, d);
      x.y += __shfl_xor_sync(0xffffffffu, x.y, d);
      x.z += __shfl_xor_sync(0xffffffffu, x.z, d);
      x.w += __shfl_xor_sync(0xffffffffu, x.w, d);
      L += __shfl_xor_sync(0xffffffffu, L, d);
      M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, d));
    }
    if (!live || part_ != 0) continue;
    const int* e = meta + 4 * list[from];
    const int u = e[0], us = e[1], ue = e[2];
    if (us >= b0 && ue <= b1) {
      const float inv = KV4_O_UNIT / L;
      *reinterpret_cast<uint2*>(a.out + (size_t)(u / a.c.nkv) * a.out_stride + (u % a.c.nkv * a.group) * HD + 4 * el) =
          make_uint2(pack_bf16(x.x * inv, x.y * inv), pack_bf16(x.z * inv, x.w * inv));
    } else {                                           // cut: in the unit's first CTA place 1, in later ones place 0
      float* dst = a.ws + ((size_t)blockIdx.x * 2 + (cta_of(us) == (int)blockIdx.x)) * a.part;
      reinterpret_cast<float4*>(dst)[el] = x;
      if (el % (HD / 4) == 0) *reinterpret_cast<float2*>(dst + a.group * HD + 2 * qh) = make_float2(M, L);
    }
  }
  // only the first and the last run can belong to a unit that other CTAs share
  int cut_from[2] = {nruns > 0 ? list[runs[0]] : -1, nruns > 1 ? list[runs[2 * nruns - 2]] : -1};
#pragma unroll
  for (int k = 0; k < 2; ++k)
    if (cut_from[k] >= 0 && meta[4 * cut_from[k] + 1] >= b0 && meta[4 * cut_from[k] + 2] <= b1) cut_from[k] = -1;
  if (cut_from[0] < 0 && cut_from[1] < 0) return;
  __threadfence();
  __syncthreads();

  // ---- units that span CTAs: the last of their CTAs joins them, in order
  if (tid < 2) {
    const int e = cut_from[tid];
    s_last[tid] = 0;
    if (e >= 0) {
      const unsigned others = cta_of(meta[4 * e + 2] - 1) - cta_of(meta[4 * e + 1]);
      s_last[tid] = atomicInc(reinterpret_cast<unsigned*>(&a.counters[meta[4 * e]]), others) == others;
    }
  }
  __syncthreads();
  __threadfence();
#pragma unroll 1
  for (int k = 0; k < 2; ++k) {
    if (!s_last[k]) continue;
    const int e = cut_from[k], u = meta[4 * e], c0 = cta_of(meta[4 * e + 1]), np = cta_of(meta[4 * e + 2] - 1) - c0 + 1;
    // thread groups take every splits-th part, four loads in flight each, and join through shared memory (the rings)
    const int splits = max(1, min(NTHR / nel, np)), step = splits > 1 ? NTHR / splits : max(nel, 1);
    float4* red = reinterpret_cast<float4*>(smem);                    // [splits][nel], then (max, sum) [splits][nel]
    float2* redm = reinterpret_cast<float2*>(red + splits * nel);
    for (int i = tid; i < step * splits; i += NTHR) {
      const int sp = i / step, el = i % step, qh = el / (HD / 4);
      if (el >= nel) continue;
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
      float M = -INFINITY, L = 0.f;
      for (int p = sp; p < np; p += 4 * splits) {
        float2 ml[4];
        float4 y[4];
        float nm = M;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int pp = p + j * splits;
          const float* src = a.ws + ((size_t)(c0 + pp) * 2 + (pp == 0)) * a.part;
          ml[j] = pp < np ? __ldcg(reinterpret_cast<const float2*>(src + a.group * HD) + qh) : make_float2(-INFINITY, 0.f);
          y[j] = pp < np ? __ldcg(reinterpret_cast<const float4*>(src) + el) : make_float4(0.f, 0.f, 0.f, 0.f);
          nm = fmaxf(nm, ml[j].x);
        }
        const float f0 = p == sp ? 0.f : ex2(M - nm);
        x = make_float4(x.x * f0, x.y * f0, x.z * f0, x.w * f0);
        L *= f0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float f = p + j * splits < np ? ex2(ml[j].x - nm) : 0.f;
          x.x += f * y[j].x;
          x.y += f * y[j].y;
          x.z += f * y[j].z;
          x.w += f * y[j].w;
          L += f * ml[j].y;
        }
        M = nm;
      }
      red[sp * nel + el] = x;
      redm[sp * nel + el] = make_float2(M, L);
    }
    __syncthreads();
    for (int el = tid; el < nel; el += NTHR) {
      float M = -INFINITY, L = 0.f;
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int sp = 0; sp < splits; ++sp) M = fmaxf(M, redm[sp * nel + el].x);
      for (int sp = 0; sp < splits; ++sp) {
        const float f = ex2(redm[sp * nel + el].x - M);
        const float4 y = red[sp * nel + el];
        x.x += f * y.x;
        x.y += f * y.y;
        x.z += f * y.z;
        x.w += f * y.w;
        L += f * redm[sp * nel + el].y;
      }
      const float inv = KV4_O_UNIT / L;
      *reinterpret_cast<uint2*>(a.out + (size_t)(u / a.c.nkv) * a.out_stride + (u % a.c.nkv * a.group) * HD + 4 * el) =
          make_uint2(pack_bf16(x.x * inv, x.y * inv), pack_bf16(x.z * inv, x.w * inv));
    }
    __syncthreads();
  }
}

// ------------------------------------------------------------------------------------------------ host
static cudaError_t kv4_launch(const void* fn, dim3 grid, int threads, size_t smem, void** args, cudaStream_t s) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  ++g_launches;
  return cudaLaunchKernelExC(&cfg, fn, args);
}

// Dynamic shared memory above 48 KB is a kernel's attribute on each device: set once a device (bit of `ready`), and the
// registers that the kernel was compiled to looked at, where it depends on them.
static bool kv4_ready(std::atomic<uint64_t>& ready, const void* fn, int bytes, bool (*registers)(int) = nullptr) {
  int dev = -1;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return false;
  if (ready.load(std::memory_order_relaxed) >> dev & 1) return true;
  if (registers != nullptr) {
    cudaFuncAttributes fa;
    if (cudaFuncGetAttributes(&fa, fn) != cudaSuccess || !registers(fa.numRegs)) return false;
  }
  if (cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) return false;
  ready.fetch_or(1ull << dev, std::memory_order_relaxed);
  return true;
}

static bool kv4_shape_ok(const A8KV4* c) {
  return c != nullptr && c->layers > 0 && c->cache_rows > 0 && c->nkv > 0 && (c->hd == 64 || c->hd == 128) &&
         c->cache_len > 0 && c->cache_len <= (1 << 30);
}
// records of the whole cache: below 2^40, so that no byte offset leaves 64 bits
static long long kv4_records(const A8KV4* c) {
  const long long nblk = ((long long)c->cache_len + KV4_BLK - 1) / KV4_BLK;
  const unsigned __int128 n = (unsigned __int128)c->layers * c->cache_rows * c->nkv * nblk;
  return n < ((unsigned __int128)1 << 40) ? (long long)n : -1;
}
static int kv4_check(const A8KV4* c, int layer) {
  if (!kv4_shape_ok(c) || c->buf == nullptr || layer < 0 || layer >= c->layers) return A8_ERR_ARG;
  if (kv4_records(c) < 0) return A8_ERR_SIZE;
  if (reinterpret_cast<uintptr_t>(c->buf) & 15) return A8_ERR_ALIGN;
  return A8_OK;
}
static Kv4View kv4_view(const A8KV4* c, int layer) {
  Kv4View v;
  v.cache_rows = c->cache_rows;
  v.nkv = c->nkv;
  v.cache_len = c->cache_len;
  v.nblk = (c->cache_len + KV4_BLK - 1) / KV4_BLK;
  v.base = reinterpret_cast<uint8_t*>(c->buf) + (size_t)layer * c->cache_rows * c->nkv * v.nblk * (size_t)(18 * c->hd);
  return v;
}
static bool kv4_misaligned(const void* p, int ld) { return (reinterpret_cast<uintptr_t>(p) & 15) || (ld % 8); }

}  // namespace a8

using namespace a8;

extern "C" long long a8_kv4_bytes(const A8KV4* c) {
  if (!kv4_shape_ok(c)) return -1;
  const long long n = kv4_records(c);
  return n < 0 ? -1 : n * 18 * c->hd;
}

extern "C" int a8_kv4_store(const A8KV4* c, int layer, const void* qkv, int ld, int nq, const void* cos,
                            const void* sin, int npos, const int* pos, const int* slot, int rows, int ring, void* q,
                            int ldq, a8_stream_t stream) {
  int rc = kv4_check(c, layer);
  if (rc) return rc;
  if (qkv == nullptr || pos == nullptr || rows <= 0 || nq < 0 || ring < 0 || (nq > 0 && q == nullptr)) return A8_ERR_ARG;
  if ((cos == nullptr) != (sin == nullptr) || (cos != nullptr && npos <= 0)) return A8_ERR_ARG;
  const long long heads = (long long)nq + 2ll * c->nkv;
  if (ld < heads * c->hd || (nq > 0 && ldq < (long long)nq * c->hd) || ring > c->cache_len) return A8_ERR_ARG;
  if (kv4_misaligned(qkv, ld) || (nq > 0 && kv4_misaligned(q, ldq)) || kv4_misaligned(cos, 0) || kv4_misaligned(sin, 0))
    return A8_ERR_ALIGN;
  if (nq > 0 && q == qkv && ldq != ld) return A8_ERR_ARG;     // (in place: every thread rewrites what it read)
  Kv4StoreArgs a;
  a.c = kv4_view(c, layer);
  a.qkv = reinterpret_cast<const __nv_bfloat16*>(qkv);
  a.ld = ld;
  a.nq = nq;
  a.cos = reinterpret_cast<const __nv_bfloat16*>(cos);
  a.sin = reinterpret_cast<const __nv_bfloat16*>(sin);
  a.npos = npos;
  a.pos = pos;
  a.slot = slot;
  a.rows = rows;
  a.ring = ring;
  a.q = reinterpret_cast<__nv_bfloat16*>(q);
  a.ldq = ldq;
  const long long blocks = ((long long)rows * heads * (c->hd / 16) + 255) / 256;
  if (blocks >= (1ll << 31)) return A8_ERR_SIZE;
  void* args[] = {&a};
  return kv4_launch(c->hd == 64 ? (const void*)k_kv4_store<64> : (const void*)k_kv4_store<128>, dim3((unsigned)blocks),
                    256, 0, args, reinterpret_cast<cudaStream_t>(stream)) == cudaSuccess ? A8_OK : A8_ERR_CUDA;
}

extern "C" int a8_kv4_load(const A8KV4* c, int layer, const int* pos, const int* slot, int rows, void* k, int ldk,
                           void* v, int ldv, a8_stream_t stream) {
  int rc = kv4_check(c, layer);
  if (rc) return rc;
  if (pos == nullptr || rows <= 0 || (k == nullptr && v == nullptr)) return A8_ERR_ARG;
  const long long w = (long long)c->nkv * c->hd;
  if ((k != nullptr && ldk < w) || (v != nullptr && ldv < w)) return A8_ERR_ARG;
  if ((k != nullptr && kv4_misaligned(k, ldk)) || (v != nullptr && kv4_misaligned(v, ldv))) return A8_ERR_ALIGN;
  Kv4LoadArgs a;
  a.c = kv4_view(c, layer);
  a.pos = pos;
  a.slot = slot;
  a.rows = rows;
  a.k = reinterpret_cast<__nv_bfloat16*>(k);
  a.v = reinterpret_cast<__nv_bfloat16*>(v);
  a.ldk = ldk;
  a.ldv = ldv;
  const long long blocks = ((long long)rows * c->nkv * (c->hd / 16) + 255) / 256;
  if (blocks >= (1ll << 31)) return A8_ERR_SIZE;
  void* args[] = {&a};
  return kv4_launch(c->hd == 64 ? (const void*)k_kv4_load<64> : (const void*)k_kv4_load<128>, dim3((unsigned)blocks),
                    256, 0, args, reinterpret_cast<cudaStream_t>(stream)) == cudaSuccess ? A8_OK : A8_ERR_CUDA;
}

// The checks and arguments that the decode and the prompt form share.
static int kv4_attn_args(Kv4AttnArgs* a, const A8KV4* c, int layer, const void* q, int q_stride, int nq, int rows,
                         float scale, void* out, int out_stride) {
  int rc = kv4_check(c, layer);
  if (rc) return rc;
  if (q == nullptr || out == nullptr || rows <= 0 || nq <= 0 || nq % c->nkv != 0 || nq / c->nkv > 16) return A8_ERR_ARG;
  if (q_stride < (long long)nq * c->hd || out_stride < (long long)nq * c->hd || !(scale < INFINITY)) return A8_ERR_ARG;
  if (kv4_misaligned(q, q_stride) || kv4_misaligned(out, out_stride)) return A8_ERR_ALIGN;
  *a = {};
  a->c = kv4_view(c, layer);
  a->q = reinterpret_cast<const __nv_bfloat16*>(q);
  a->q_stride = q_stride;
  a->nq = nq;
  a->group = nq / c->nkv;
  a->rows = rows;
  a->max_len = c->cache_len;
  a->scale_log2 = (scale > 0 ? scale : 1.0f / sqrtf((float)c->hd)) * 1.4426950408889634f;
  a->out = reinterpret_cast<__nv_bfloat16*>(out);
  a->out_stride = out_stride;
  return A8_OK;
}

// CTAs of a decode call: one an SM, fewer when the rows cannot hold enough steps.
static int kv4_ctas(const A8KV4* c, int rows, int max_len) {
  const long long steps = (long long)rows * c->nkv * ((max_len + KV4_STEP - 1) / KV4_STEP);
  return (int)std::min<long long>(KV4_CTAS, (steps + KV4_CTA_STEPS - 1) / KV4_CTA_STEPS);
}
static int kv4_part(const A8KV4* c, int nq) { return (nq / c->nkv * (c->hd + 2) + 3) / 4 * 4; }

extern "C" int a8_kv4_attention_workspace(const A8KV4* c, int nq, int rows, int max_len, long long* ws_floats,
                                          int* n_counters) {
  if (!kv4_shape_ok(c) || nq <= 0 || nq % c->nkv != 0 || nq / c->nkv > 16 || rows <= 0 || rows > (1 << 24) ||
      max_len <= 0 || max_len > c->cache_len || (long long)rows * c->nkv >= (1ll << 31))
    return A8_ERR_ARG;
  if (ws_floats) *ws_floats = 2ll * kv4_ctas(c, rows, max_len) * kv4_part(c, nq);
  if (n_counters) *n_counters = rows * c->nkv;
  return A8_OK;
}

template <int HD, int NT>
static int kv4_attn_launch(Kv4AttnArgs& a, int ctas, cudaStream_t s) {
  using SM = Kv4DecSmem<HD, NT>;
  const void* fn = (const void*)k_kv4_attn<HD, NT>;
  static std::atomic<uint64_t> ready{0};
  if (!kv4_ready(ready, fn, SM::TOTAL)) return A8_ERR_CUDA;
  void* args[] = {&a};
  return kv4_launch(fn, dim3(ctas), SM::NW * 32, SM::TOTAL, args, s) == cudaSuccess ? A8_OK : A8_ERR_CUDA;
}

// a8_kv4_attention with row r's keys counted from lens[r] + lens_add (a stack gives its positions and 1).
static int kv4_attention(const A8KV4* c, int layer, const void* q, int q_stride, int nq, const int* lens, int lens_add,
                         const int* rowmap, int rows, int max_len, float scale, void* out, int out_stride, float* ws,
                         long long ws_floats, int* counters, int n_counters, cudaStream_t s) {
  Kv4AttnArgs a;
  int rc = kv4_attn_args(&a, c, layer, q, q_stride, nq, rows, scale, out, out_stride);
  if (rc) return rc;
  // (in place: a unit's result is written after its last read of the queries it stands in)
  if (lens == nullptr || max_len <= 0 || max_len > c->cache_len || (out == q && out_stride != q_stride)) return A8_ERR_ARG;
  // the steps of all rows are counted in 32 bits, and rounded up to CTAs' shares there
  const long long steps = (long long)rows * c->nkv * ((max_len + KV4_STEP - 1) / KV4_STEP);
  if (rows > (1 << 24) || steps >= (1ll << 31) - KV4_CTA_STEPS) return A8_ERR_SIZE;
  const int ctas = kv4_ctas(c, rows, max_len);
  a.part = kv4_part(c, nq);
  if (ws == nullptr || ws_floats < 2ll * ctas * a.part || counters == nullptr || n_counters < (long long)rows * c->nkv)
    return A8_ERR_SIZE;
  if (reinterpret_cast<uintptr_t>(ws) & 15) return A8_ERR_ALIGN;
  a.lens = lens;
  a.lens_add = lens_add;
  a.rowmap = rowmap;
  a.max_len = max_len;
  a.ws = ws;
  a.counters = counters;
  if (a.group <= 8) return c->hd == 64 ? kv4_attn_launch<64, 1>(a, ctas, s) : kv4_attn_launch<128, 1>(a, ctas, s);
  return c->hd == 64 ? kv4_attn_launch<64, 2>(a, ctas, s) : kv4_attn_launch<128, 2>(a, ctas, s);
}

extern "C" int a8_kv4_attention(const A8KV4* c, int layer, const void* q, int q_stride, int nq, const int* lens,
                                const int* rowmap, int rows, int max_len, float scale, void* out, int out_stride,
                                float* ws, long long ws_floats, int* counters, int n_counters, a8_stream_t stream) {
  return kv4_attention(c, layer, q, q_stride, nq, lens, 0, rowmap, rows, max_len, scale, out, out_stride, ws, ws_floats,
                       counters, n_counters, reinterpret_cast<cudaStream_t>(stream));
}
