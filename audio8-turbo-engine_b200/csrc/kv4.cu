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
//   K word (t', slot): dims 32 g + 8 t' .. + 7 at byte  j hd / 2 + (t' G + slot) 4
//   V half (q, slot):  dims 32 g + 4 q .. + 3 at byte   j hd / 2 + ((q ^ sw) G + slot) 2,  sw = 4 (j >> 1 & 1) at hd 128
//   scale (j, slot):   element (4 t + i) G + slot
// slot orders the groups so that group g and g + G / 2 (the two dims of a RoPE pair) are neighbours: 0, 2, 1, 3 at hd 128.
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

__device__ __forceinline__ void ld8f(const __nv_bfloat16* p, float* f) {
  const uint4 u = *reinterpret_cast<const uint4*>(p);
  const float2 a = unpack_bf16(u.x), b = unpack_bf16(u.y), c = unpack_bf16(u.z), d = unpack_bf16(u.w);
  f[0] = a.x; f[1] = a.y; f[2] = b.x; f[3] = b.y; f[4] = c.x; f[5] = c.y; f[6] = d.x; f[7] = d.y;
}

// The 8 codes of this thread's dims (nibble n = dim n) and the scale of the group they share with the other three lanes
// of the aligned four.
__device__ __forceinline__ uint32_t kv4_quant8(const float* x, uint32_t& scale_bits) {
  uint32_t m = 0;
#pragma unroll
  for (int n = 0; n < 8; ++n) m = max(m, __float_as_uint(x[n]) & 0x7FFFFFFFu);   // (orders inf and NaN above all)
  m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
  m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
  uint32_t w = 0x88888888u;
  if (m >= 0x7F800000u) {
    scale_bits = 0x7FFFu;
    return w;
  }
  const __nv_bfloat16 sb = __float2bfloat16_rn(__fdiv_rn(__uint_as_float(m), 7.0f));
  scale_bits = __bfloat16_as_ushort(sb);
  const float s = __bfloat162float(sb);
  if (s > 0.f) {
    w = 0;
#pragma unroll
    for (int n = 0; n < 8; ++n)
      w |= uint32_t(min(max(__float2int_rn(__fdiv_rn(x[n], s)), -7), 7) + 8) << (4 * n);
  }
  return w;
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
  const long long idx = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  const int sub = int(idx % TPH);
  const long long rh = idx / TPH;
  const int head = int(rh % heads);
  const int row = int(min(rh / heads, (long long)a.rows - 1));
  bool live = rh / heads < a.rows;
  const int pos = a.pos[row];
  const int slot = a.slot != nullptr ? a.slot[row] : row;
  const int at = a.ring > 0 ? pos % a.ring : pos;
  live = live && pos >= 0;                               // a row at a negative position is padding
  if (live && (at >= a.c.cache_len || slot < 0 || slot >= a.c.cache_rows || (a.cos != nullptr && pos >= a.npos))) {
    if (sub == 0 && head == 0) set_error(ERR_BOUNDS, KERNEL_ID_KV4_STORE, row);
    live = false;
  }
  const int d0 = sub * 8;
  float lo[8], hi[8];
#pragma unroll
  for (int n = 0; n < 8; ++n) lo[n] = hi[n] = 0.f;
  if (live) {
    const __nv_bfloat16* x = a.qkv + (size_t)row * a.ld + head * HD;
    ld8f(x + d0, lo);
    ld8f(x + d0 + HD / 2, hi);
    if (a.cos != nullptr && head < a.nq + a.c.nkv) {
      float c[8], s[8];
      ld8f(a.cos + (size_t)pos * HD + d0, c);
      ld8f(a.sin + (size_t)pos * HD + d0, s);
#pragma unroll
      for (int n = 0; n < 8; ++n) {
        // products of two bf16 are exact in fp32: the rotation is one fp32 rounding and one to bf16, what a bf16 cache
        // would hold
        const float u = lo[n], v = hi[n];
        lo[n] = bf16r(u * c[n] - v * s[n]);
        hi[n] = bf16r(v * c[n] + u * s[n]);
      }
    }
    if (head < a.nq) {
      __nv_bfloat16* y = a.q + (size_t)row * a.ldq + head * HD + d0;
      *reinterpret_cast<uint4*>(y) = make_uint4(pack_bf16(lo[0], lo[1]), pack_bf16(lo[2], lo[3]),
                                                pack_bf16(lo[4], lo[5]), pack_bf16(lo[6], lo[7]));
      *reinterpret_cast<uint4*>(y + HD / 2) = make_uint4(pack_bf16(hi[0], hi[1]), pack_bf16(hi[2], hi[3]),
                                                         pack_bf16(hi[4], hi[5]), pack_bf16(hi[6], hi[7]));
    }
  }
  // (every lane takes part in the group maximum)
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

// bf16(code * s) of the 8 nibbles of w
__device__ __forceinline__ uint4 kv4_deq8(uint32_t w, float s) {
  float f[8];
#pragma unroll
  for (int n = 0; n < 8; ++n) f[n] = float(int((w >> (4 * n)) & 15u) - 8) * s;
  return make_uint4(pack_bf16(f[0], f[1]), pack_bf16(f[2], f[3]), pack_bf16(f[4], f[5]), pack_bf16(f[6], f[7]));
}

template <int HD>
__global__ void __launch_bounds__(256) k_kv4_load(const Kv4LoadArgs a) {
  using F = Kv4<HD>;
  constexpr int TPH = HD / 16;
  pdl_launch();
  pdl_wait();
  const long long idx = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  const int sub = int(idx % TPH);
  const long long rh = idx / TPH;
  const int h = int(rh % a.c.nkv);
  if (rh / a.c.nkv >= a.rows) return;
  const int row = int(rh / a.c.nkv);
  const int pos = a.pos[row];
  const int slot = a.slot != nullptr ? a.slot[row] : row;
  if (pos < 0) return;
  if (pos >= a.c.cache_len || slot < 0 || slot >= a.c.cache_rows) {
    if (sub == 0 && h == 0) set_error(ERR_BOUNDS, KERNEL_ID_KV4_LOAD, row);
    return;
  }
  const int t8 = sub & 3, s0 = (sub >> 2) * 2, j = pos % KV4_BLK;
  const uint8_t* rec = kv4_rec(a.c, F::REC, slot, h, pos / KV4_BLK);
  if (a.k != nullptr) {
    const uint2 w = *reinterpret_cast<const uint2*>(rec + F::kword(j, t8, s0));
    const float2 s = unpack_bf16(*reinterpret_cast<const uint32_t*>(rec + F::KS0 + F::scale(j, s0)));
    __nv_bfloat16* y = a.k + (size_t)row * a.ldk + h * HD + sub * 8;
    *reinterpret_cast<uint4*>(y) = kv4_deq8(w.x, s.x);
    *reinterpret_cast<uint4*>(y + HD / 2) = kv4_deq8(w.y, s.y);
  }
  if (a.v != nullptr) {
    const uint32_t u0 = *reinterpret_cast<const uint32_t*>(rec + F::vhalf(j, 2 * t8, s0));
    const uint32_t u1 = *reinterpret_cast<const uint32_t*>(rec + F::vhalf(j, 2 * t8 + 1, s0));
    const float2 s = unpack_bf16(*reinterpret_cast<const uint32_t*>(rec + F::VS0 + F::scale(j, s0)));
    __nv_bfloat16* y = a.v + (size_t)row * a.ldv + h * HD + sub * 8;
    *reinterpret_cast<uint4*>(y) = kv4_deq8((u0 & 0xFFFFu) | (u1 << 16), s.x);
    *reinterpret_cast<uint4*>(y + HD / 2) = kv4_deq8((u0 >> 16) | (u1 & 0xFFFF0000u), s.y);
  }
}

// ------------------------------------------------------------------------------------------------ attention
struct Kv4AttnArgs {
  Kv4View c;
  const __nv_bfloat16* q;
  int q_stride, nq;
  const int *lens, *rowmap;   // decode: keys of row r; cache row of row r (null: r)
  const int* blocks;          // packed prompts: [nblocks][4] = (q0, n, slot, pos0)
  int rows, max_len;
  float scale_log2;
  __nv_bfloat16* out;
  int out_stride;
};

// One warp a (query row, query head): a lane holds hd / 32 dims, the keys come one after another.
template <int HD>
__global__ void __launch_bounds__(128) k_kv4_attn_simple(const Kv4AttnArgs a) {
  using F = Kv4<HD>;
  constexpr int D = HD / 32;
  pdl_launch();
  pdl_wait();
  const int lane = threadIdx.x & 31, head = blockIdx.y * 4 + (threadIdx.x >> 5);
  if (head >= a.nq) return;
  int r = blockIdx.x, len, crow;
  if (a.blocks != nullptr) {
    const int* b = a.blocks + 4 * (blockIdx.x / 64);
    const int i = blockIdx.x % 64;
    if (i >= b[1]) return;
    if (b[0] < 0 || b[1] > 64 || b[0] > a.rows - b[1] || b[2] < 0 || b[2] >= a.c.cache_rows || b[3] < 0 ||
        b[3] > a.c.cache_len - b[1]) {
      if (i == 0 && lane == 0) set_error(ERR_BOUNDS, KERNEL_ID_KV4_ATTN, blockIdx.x / 64);
      return;
    }
    r = b[0] + i;
    crow = b[2];
    len = b[3] + i + 1;
  } else {
    len = a.lens[r];
    crow = a.rowmap != nullptr ? a.rowmap[r] : r;
  }
  len = max(0, min(len, a.max_len));
  if (crow < 0 || crow >= a.c.cache_rows) {
    if (lane == 0 && head == 0) set_error(ERR_BOUNDS, KERNEL_ID_KV4_ATTN, r);
    len = 0;
  }
  const int h = head / (a.nq / a.c.nkv);
  float q[D], o[D], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int d = 0; d < D; ++d) {
    q[d] = __bfloat162float(a.q[(size_t)r * a.q_stride + head * HD + lane * D + d]) * a.scale_log2;
    o[d] = 0.f;
  }
  const int dim = lane * D, grp = dim / 32, s = F::slot(grp);
  for (int p = 0; p < len; ++p) {
    const int j = p % KV4_BLK;
    const uint8_t* rec = kv4_rec(a.c, F::REC, crow, h, p / KV4_BLK);
    const uint32_t kw = *reinterpret_cast<const uint32_t*>(rec + F::kword(j, (dim % 32) / 8, s)) >> (4 * (dim % 8));
    const uint32_t vw = *reinterpret_cast<const uint16_t*>(rec + F::vhalf(j, (dim % 32) / 4, s)) >> (4 * (dim % 4));
    const float ks = __bfloat162float(*reinterpret_cast<const __nv_bfloat16*>(rec + F::KS0 + F::scale(j, s)));
    const float vs = __bfloat162float(*reinterpret_cast<const __nv_bfloat16*>(rec + F::VS0 + F::scale(j, s)));
    float x = 0.f;
#pragma unroll
    for (int d = 0; d < D; ++d) x += q[d] * (float(int((kw >> (4 * d)) & 15u) - 8) * ks);
#pragma unroll
    for (int k = 16; k > 0; k >>= 1) x += __shfl_xor_sync(0xffffffffu, x, k);
    const float n = fmaxf(m, x), al = m == -INFINITY ? 0.f : exp2f(m - n), e = exp2f(x - n);
    m = n;
    l = l * al + e;
#pragma unroll
    for (int d = 0; d < D; ++d) o[d] = o[d] * al + e * (float(int((vw >> (4 * d)) & 15u) - 8) * vs);
  }
#pragma unroll
  for (int d = 0; d < D; ++d)
    a.out[(size_t)r * a.out_stride + head * HD + dim + d] = __float2bfloat16_rn(len > 0 ? o[d] / l : 0.f);
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
  a->rows = rows;
  a->max_len = c->cache_len;
  a->scale_log2 = (scale > 0 ? scale : 1.0f / sqrtf((float)c->hd)) * 1.4426950408889634f;
  a->out = reinterpret_cast<__nv_bfloat16*>(out);
  a->out_stride = out_stride;
  return A8_OK;
}

extern "C" int a8_kv4_attention_workspace(const A8KV4* c, int nq, int rows, int max_len, long long* ws_floats,
                                          int* n_counters) {
  if (!kv4_shape_ok(c) || nq <= 0 || nq % c->nkv != 0 || nq / c->nkv > 16 || rows <= 0 || max_len <= 0 ||
      max_len > c->cache_len)
    return A8_ERR_ARG;
  if (ws_floats) *ws_floats = 0;
  if (n_counters) *n_counters = 0;
  return A8_OK;
}

extern "C" int a8_kv4_attention(const A8KV4* c, int layer, const void* q, int q_stride, int nq, const int* lens,
                                const int* rowmap, int rows, int max_len, float scale, void* out, int out_stride,
                                float* ws, long long ws_floats, int* counters, int n_counters, a8_stream_t stream) {
  Kv4AttnArgs a;
  int rc = kv4_attn_args(&a, c, layer, q, q_stride, nq, rows, scale, out, out_stride);
  if (rc) return rc;
  if (lens == nullptr || max_len <= 0 || max_len > c->cache_len) return A8_ERR_ARG;
  a.lens = lens;
  a.rowmap = rowmap;
  a.max_len = max_len;
  void* args[] = {&a};
  return kv4_launch(c->hd == 64 ? (const void*)k_kv4_attn_simple<64> : (const void*)k_kv4_attn_simple<128>,
                    dim3(rows, (nq + 3) / 4), 128, 0, args, reinterpret_cast<cudaStream_t>(stream)) == cudaSuccess
             ? A8_OK : A8_ERR_CUDA;
}

extern "C" int a8_kv4_prefill_attention(const A8KV4* c, int layer, const void* q, int q_stride, int nq,
                                        const int* blocks, int nblocks, int rows, float scale, void* out,
                                        int out_stride, a8_stream_t stream) {
  Kv4AttnArgs a;
  int rc = kv4_attn_args(&a, c, layer, q, q_stride, nq, rows, scale, out, out_stride);
  if (rc) return rc;
  if (blocks == nullptr || nblocks <= 0 || nblocks > (1 << 24)) return A8_ERR_ARG;
  a.blocks = blocks;
  void* args[] = {&a};
  return kv4_launch(c->hd == 64 ? (const void*)k_kv4_attn_simple<64> : (const void*)k_kv4_attn_simple<128>,
                    dim3(nblocks * 64, (nq + 3) / 4), 128, 0, args, reinterpret_cast<cudaStream_t>(stream)) ==
                 cudaSuccess ? A8_OK : A8_ERR_CUDA;
}
