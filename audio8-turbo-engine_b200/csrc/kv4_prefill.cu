// Packed causal prompt attention over the 4-bit cache on the tensor cores (tcgen05).
//
// A query block is up to 64 consecutive positions of one request (q0, n, slot, pos0). One CTA takes a block, a kv head and
// up to four of its query heads: two 128-row tiles (64 positions x 2 heads each) share every 64-key tile, which is
// brought to 16 bits once.
//   warps 0-7   softmax, one query vector a thread (its TMEM lane): tile warp / 4
//   warps 8-11  K: codes -> fp16 [64 keys][hd], K-major, 128-byte swizzle
//   warps 12-15 V: codes -> fp16 V^T [hd][64 keys]
//   warp 16     bulk copies of the key tiles' records (a tile is four records, one copy)
//   warp 17     issue of S = Q K^T     warp 18  issue of O += P V     warp 19  each tile's exponents ek, E
// fp16, not bf16: code * s has 8 + 3 significant bits, so K and V are exact in fp16's 11 where bf16 would round each to 8.
// Its narrow range is met by powers of two: a tile's K is divided by 2^ek (its largest scale in [1, 2)), which the softmax
// multiplies back into its logit scale; V by 2^E, the largest scale met so far, which joins the running maximum's factor
// on O when it grows; a query vector by its own largest element. In a block's own tiles, the last ones, keys behind a row may
// be far above those that it attends: where a tile's scales there lie more than 2^14 apart (past what fp16 holds exactly) each
// key is divided by its own exponents, and each row brings its logits and weights to the largest that it attends, so that
// keys behind a row cost it no bits (such tiles throughout: 8 to 33 % slower). P is fp16 with weights up to 2^15 (the running
// maximum is moved where a logit passes it by 2^8, and only looked at where a tile's weights of a row sum to more than 2^15),
// rounded to 11 bits; sums and O in fp32.
// Bound: 8,189 positions, 32 heads over 8, hd 128: 549 GFLOP in 576 to 617 us, 900 to 950 TFLOP/s, 0.55 of a library product's
// rate. A key tile takes its CTA about 1.3 us, 2,500 cycles, and no unit is full in them: a tile's chain, unpacking -> S ->
// softmax -> P V, two stages of S deep, waits on itself. The tile's time hardly depends on hd or on the heads it serves: 14 heads
// over 2, hd 64, 1.26 us (8,189 positions 281 us, 427 TFLOP/s); one head a kv head, where 64 of the 256 query vectors are used,
// 1.0 us (8 over 8, hd 128, 445 us, 309 TFLOP/s). An admission (2,048 ragged rows behind prefixes of 317, 14 heads over 2, hd 64)
// takes 20 to 29 us, as long as its longest prompt's last block, a second wave where there are more than 148 CTAs, and the
// filling of the pipeline.
// Measured and not kept: exponentials as polynomials on the FMA pipe for 1/4, 1/2, 3/4 of the weights (707, 740, 998 us
// against 693 then). On the way: S and P V issued by one warp 905 us, by two 693; every tile's maximum before its weights 693,
// only where their sum asks for it 673; warp indexes that the compiler cannot see are uniform 650, shuffled from one lane 620;
// the second half of S fetched behind the first half's weights 684 against 646; the two tiles' softmax started half a tile
// apart no gain; masks and wide scales in a loop of their own for the block's own tiles 576 against 607, where a test more
// between the other tiles' instructions gave 617 to 730.
// Within a chunk of eight dims Q and K keep the order 0 4 1 5 2 6 3 7, in which the codes come out of their words.
#include "common.cuh"

namespace a8 {

constexpr int KERNEL_ID_KV4_PREFILL = 12;
constexpr int KV4P_SOFT = 8, KV4P_DEQ = 4;               // softmax warps; warps of each of K and V
constexpr int KV4P_THREADS = (KV4P_SOFT + 2 * KV4P_DEQ + 4) * 32;   // five warpgroups (the last: warps 16 to 19)
// Registers a thread after the warpgroups' redistribution: 256 x 144 + 256 x 64 + 128 x 64, all of the 640 x 96 = 61,440
// that the block is launched with. A compiler that gave the kernel fewer would leave the softmax warps waiting for registers
// that never come free, so the host looks at what it gave before the first launch.
constexpr int KV4P_REG_SOFT = 144, KV4P_REG_REST = 64;
constexpr bool kv4p_registers_cover(int per_thread) {
  return per_thread * KV4P_THREADS >= KV4P_SOFT * 32 * KV4P_REG_SOFT + (2 * KV4P_DEQ + 4) * 32 * KV4P_REG_REST;
}
static_assert(kv4p_registers_cover(96), "");
#define A8_SETMAXNREG(op, n) asm volatile("setmaxnreg." op ".sync.aligned.u32 %0;" ::"n"(n))
constexpr int KV4P_RAW = 6;                              // raw key tiles in flight
constexpr int KV4P_VST = 3;                              // V tiles at hand
constexpr float KV4P_BIAS = 6.f;                         // p = 2^(x - m + 6)
constexpr int KV4P_WIDE = 256;                           // in ek: the tile's keys have exponents of their own

template <int HD>
struct Kv4PreSmem {
  static constexpr int Q = 0;                            // 2 tiles x HD / 64 atoms x [128 rows][128 B]
  static constexpr int QT = HD / 64 * 16384;
  static constexpr int K = Q + 2 * QT;                   // 2 stages x HD / 64 atoms x [64 keys][128 B]
  static constexpr int KT = HD / 64 * 8192;
  static constexpr int V = K + 2 * KT;                   // KV4P_VST stages x [HD rows][128 B]
  static constexpr int VT = HD * 128;
  static constexpr int RAW = V + KV4P_VST * VT;
  static constexpr int RAWT = 4 * Kv4<HD>::REC;
  static constexpr int SC = RAW + KV4P_RAW * RAWT;       // a raw tile's scales as fp16, divided: K [64 keys][G], V [G][64 keys]
  static constexpr int SCT = 2 * 64 * (HD / 32) * 2;
  static constexpr int MISC = SC + KV4P_RAW * SCT;       // int ek[16], ev[16], nanv[4]
  static constexpr int KEYX = MISC + 144;                // a tile's exponents by key: K [16][64], V [16][64] bytes
  static constexpr int BARS = KEYX + 2 * 16 * 64;
  static constexpr int TOTAL = BARS + 40 * 8 + 16 + 1024;
  static constexpr uint32_t COLS = 512;                  // TMEM: S of tile 0 and 1, two stages of 64 each (P takes
                                                         // the first half of its S); O (HD each)
  static_assert(TOTAL <= 227 * 1024, "");
};

__device__ __forceinline__ void tmem_st32(uint32_t taddr, const float* v) {
  const uint32_t* r = reinterpret_cast<const uint32_t*>(v);
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,"
      "%29,%30,%31};" ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]),
      "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]),
      "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]), "r"(taddr)
      : "memory");
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

__device__ __forceinline__ void tmem_ld4(uint32_t taddr, float* v) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x4.b32 {%0,%1,%2,%3}, [%4];\n\ttcgen05.wait::ld.sync.aligned;"
               : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3])
               : "r"(taddr)
               : "memory");
}
__device__ __forceinline__ void tmem_st4(uint32_t taddr, const float* v) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%4], {%0,%1,%2,%3};\n\ttcgen05.wait::st.sync.aligned;" ::"f"(v[0]),
               "f"(v[1]), "f"(v[2]), "f"(v[3]), "r"(taddr)
               : "memory");
}

// 64 columns at once
__device__ __forceinline__ void tmem_ld64(uint32_t taddr, float* v) {
  uint32_t r[64];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x64.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,"
      "%29,%30,%31,%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,%47,%48,%49,%50,%51,%52,%53,%54,%55,"
      "%56,%57,%58,%59,%60,%61,%62,%63}, [%64];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]), "=r"(r[32]),
        "=r"(r[33]), "=r"(r[34]), "=r"(r[35]), "=r"(r[36]), "=r"(r[37]), "=r"(r[38]), "=r"(r[39]), "=r"(r[40]),
        "=r"(r[41]), "=r"(r[42]), "=r"(r[43]), "=r"(r[44]), "=r"(r[45]), "=r"(r[46]), "=r"(r[47]), "=r"(r[48]),
        "=r"(r[49]), "=r"(r[50]), "=r"(r[51]), "=r"(r[52]), "=r"(r[53]), "=r"(r[54]), "=r"(r[55]), "=r"(r[56]),
        "=r"(r[57]), "=r"(r[58]), "=r"(r[59]), "=r"(r[60]), "=r"(r[61]), "=r"(r[62]), "=r"(r[63])
      : "r"(taddr));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < 64; ++i) v[i] = __uint_as_float(r[i]);
}

// D += A B with A (128 rows x 16 fp16, two a column) in tensor memory, B in shared memory
__device__ __forceinline__ void umma_f16_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc, uint32_t idesc,
                                            uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(tmem_d),
      "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// Codes of the two 16-bit halves of w as fp16 with an offset: nibbles 0 and 2 of a half as 1024 + u, 1 and 3 as
// 1024 + 16 u (one mask with or).
__device__ __forceinline__ uint32_t kv4_lo16(uint32_t w) {
  uint32_t d;
  asm("lop3.b32 %0, %1, 0x000F000F, 0x64006400, 0xEA;" : "=r"(d) : "r"(w));
  return d;
}
__device__ __forceinline__ uint32_t kv4_hi16(uint32_t w) {
  uint32_t d;
  asm("lop3.b32 %0, %1, 0x00F000F0, 0x64006400, 0xEA;" : "=r"(d) : "r"(w));
  return d;
}
// The pairs (n, n + 4) of a word's (or of a key pair's) codes, n = 0..3, as fp16 whole numbers.
__device__ __forceinline__ void kv4_codes_f16(uint32_t w, __half2* c) {
  const __half2 off = __half2half2(__ushort_as_half(0xE408));                     // -1032
  const __half2 sixteenth = __half2half2(__ushort_as_half(0x2C00)), off16 = __half2half2(__ushort_as_half(0xD480));  // 1/16, -72
  const uint32_t w8 = w >> 8;
  uint32_t x;
  x = kv4_lo16(w);
  c[0] = __hadd2(*reinterpret_cast<__half2*>(&x), off);
  x = kv4_hi16(w);
  c[1] = __hfma2(*reinterpret_cast<__half2*>(&x), sixteenth, off16);
  x = kv4_lo16(w8);
  c[2] = __hadd2(*reinterpret_cast<__half2*>(&x), off);
  x = kv4_hi16(w8);
  c[3] = __hfma2(*reinterpret_cast<__half2*>(&x), sixteenth, off16);
}
__device__ __forceinline__ uint32_t h2u(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }
// 2^(e - 127) for a biased exponent e, and its inverse; both normal for e in [1, 253]
__device__ __forceinline__ float pow2_biased(int e) { return __uint_as_float(uint32_t(e) << 23); }
__device__ __forceinline__ float pow2_biased_inv(int e) { return __uint_as_float(uint32_t(254 - e) << 23); }
// 2^(e - of) for e up to of; 0 below 2^-126, and whatever for a larger e (a masked key's) is finite
__device__ __forceinline__ float pow2_diff(int e, int of) { return pow2_biased(max(127 + min(e - of, 0), 0)); }

template <int HD>
__global__ void __launch_bounds__(KV4P_THREADS, 1) k_kv4_prefill(const Kv4AttnArgs a) {
  using F = Kv4<HD>;
  using SM = Kv4PreSmem<HD>;
  constexpr int G = F::G;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  int* ek = reinterpret_cast<int*>(smem + SM::MISC);     // by tile % 16
  int* ev = ek + 16;
  int* nanv = ev + 16;                                   // [4] first position whose V group is NaN
  uint8_t *keyk = smem + SM::KEYX, *keyv = keyk + 16 * 64;
  uint64_t* q_full = reinterpret_cast<uint64_t*>(smem + SM::BARS);
  uint64_t *raw_full = q_full + 1, *raw_free = raw_full + KV4P_RAW, *e_full = raw_free + KV4P_RAW, *k_full = e_full + KV4P_RAW,
           *k_free = k_full + 2, *v_full = k_free + 2, *v_free = v_full + KV4P_VST, *s_full = v_free + KV4P_VST, *p_full = s_full + 4,
           *p_free = p_full + 4;                         // the last three: [tile][stage]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(p_free + 4);

  // (the warp's index from one lane: barrier addresses and branches are uniform to the compiler)
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  pdl_wait();
  // the last blocks first, all their heads together: they attend the most keys of a prompt
  const int hq = (a.group + 3) / 4, per = a.c.nkv * hq;
  const int bi = int(gridDim.x) / per - 1 - int(blockIdx.x) / per, kvh = blockIdx.x % per / hq, hpart = blockIdx.x % hq;
  const int q0 = a.blocks[4 * bi], nrow = a.blocks[4 * bi + 1], crow = a.blocks[4 * bi + 2], pos0 = a.blocks[4 * bi + 3];
  if (nrow <= 0) return;                                 // (uniform over the CTA, before any barrier)
  if (q0 < 0 || nrow > 64 || q0 > a.rows - nrow || crow < 0 || crow >= a.c.cache_rows || pos0 < 0 ||
      pos0 > a.c.cache_len - nrow) {
    if (tid == 0) set_error(ERR_BOUNDS, KERNEL_ID_KV4_PREFILL, bi);
    return;
  }
  const int heads = min(4, a.group - 4 * hpart);
  const int head0 = kvh * a.group + 4 * hpart;
  const int ntx = (heads + 1) / 2;                       // tiles in use
  const int klen = pos0 + nrow, nt = (klen + 63) / 64;
  const int first = (pos0 + 1) / 64;                     // the first tile that some row does not attend to its end

  if (tid == 0) {
    mbar_init(q_full, KV4P_SOFT);
    for (int s = 0; s < KV4P_RAW; ++s) {
      mbar_init(&raw_full[s], 1);
      mbar_init(&raw_free[s], 2 * KV4P_DEQ + 1);
      mbar_init(&e_full[s], 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&k_full[s], KV4P_DEQ);
      mbar_init(&k_free[s], 1);
    }
    for (int s = 0; s < KV4P_VST; ++s) {
      mbar_init(&v_full[s], KV4P_DEQ);
      mbar_init(&v_free[s], 1);
    }
    for (int s = 0; s < 4; ++s) {
      mbar_init(&s_full[s], 2);                          // the MMAs' completion, and the issuer itself (for ek, ev)
      mbar_init(&p_full[s], 4);
      mbar_init(&p_free[s], 1);
    }
    fence_mbar_init();
    for (int g = 0; g < 4; ++g) nanv[g] = 0x7FFFFFFF;
  }
  if (warp == 17) tmem_alloc(tmem_slot, SM::COLS);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  // Only now may the next kernel's CTAs come: one that took tensor memory on this SM first, and then waited for this grid,
  // would leave none for this CTA.
  pdl_launch();

  if (warp < KV4P_SOFT) {
    A8_SETMAXNREG("inc", KV4P_REG_SOFT);
    // ---- softmax: thread = query vector (head 2 x + half, position pos0 + r)
    const int x = warp >> 2, row = (warp & 3) * 32 + lane, r = row & 63, hi = row >> 6;
    const int head = 2 * x + hi;
    const bool live = r < nrow && head < heads;
    const int pos = pos0 + min(r, nrow - 1);
    const uint32_t tS = tmem + x * 128 + (uint32_t((warp & 3) * 32) << 16);
    const uint32_t tO = tmem + 256 + x * HD + (uint32_t((warp & 3) * 32) << 16);
    // the query vector: fp16, divided by the power of two of its largest element
    float qs;
    {
      const uint4* src = reinterpret_cast<const uint4*>(a.q + (size_t)(q0 + r) * a.q_stride + (head0 + head) * HD);
      uint32_t top = 0;
      if (live)
        for (int c = 0; c < HD / 8; ++c) {
          const uint4 w = src[c];
          const uint32_t e[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
          for (int k = 0; k < 4; ++k) top = max(top, max(e[k] & 0x7FFFu, (e[k] >> 16) & 0x7FFFu));
        }
      const int ex = min(max(int(top >> 7), 1), 253);
      const float down = pow2_biased_inv(ex);
      qs = a.scale_log2 * pow2_biased(ex);
      uint8_t* dst = smem + SM::Q + x * SM::QT;
      for (int c = 0; c < HD / 8; ++c) {
        const uint4 w = live ? src[c] : make_uint4(0, 0, 0, 0);
        const float2 d01 = unpack_bf16(w.x), d23 = unpack_bf16(w.y), d45 = unpack_bf16(w.z), d67 = unpack_bf16(w.w);
        *reinterpret_cast<uint4*>(dst + (c >> 3) * 16384 + sw128(row, c & 7)) =
            make_uint4(pack_f16(d01.x * down, d45.x * down), pack_f16(d01.y * down, d45.y * down),
                       pack_f16(d23.x * down, d67.x * down), pack_f16(d23.y * down, d67.y * down));
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(q_full);
    }
    float m = -INFINITY, l = 0.f;
    int E = 0;
    bool ok = true;
    // A key tile (false: no further). own: keys behind a row may be in it, and its scales may be wide.
    auto tile = [&](auto own, const int j) {
      const int b = 2 * x + (j & 1), ph = (j >> 1) & 1;
      if (!(ok = mbar_wait_all(&s_full[b], ph, ERR_TIMEOUT_FULL, KERNEL_ID_KV4_PREFILL))) return false;
      tc_fence_after();
      const int kmax = pos - 64 * j;                     // keys c <= kmax of this tile are causal for this row
      int ex = ek[j & 15], Ej = ev[j & 15];
      bool wide = false;
      if constexpr (decltype(own)::value) {
        wide = ex >= KV4P_WIDE;
        if (kmax < 0) Ej = E;                            // (a row that attends none of them keeps its E)
      }
      if (wide) {
        // each key by its own exponents: the row's are the largest that it attends, and its logits are brought to them
        const uint8_t *kx = keyk + (j & 15) * 64, *vx = keyv + (j & 15) * 64;
        ex = 1;
        Ej = E;
#pragma unroll 1
        for (int c = 0; c < 64; ++c) {
          ex = max(ex, c <= kmax ? int(kx[c]) : 0);
          Ej = max(Ej, c <= kmax ? int(vx[c]) : 0);
        }
#pragma unroll 1
        for (int c = 0; c < 64; c += 4) {
          float z[4];
          tmem_ld4(tS + (j & 1) * 64 + c, z);
#pragma unroll
          for (int k = 0; k < 4; ++k) z[k] *= pow2_diff(kx[c + k], ex);
          tmem_st4(tS + (j & 1) * 64 + c, z);
        }
      }
      float sv[64];
      tmem_ld64(tS + (j & 1) * 64, sv);
      // (never 0, which would make a masked -infinity NaN; at this least value every logit is below 2^-110)
      const float f = fmaxf(qs * pow2_biased(ex), 0x1p-126f);
      if (decltype(own)::value && __any_sync(0xffffffffu, kmax < 63)) {
#pragma unroll
        for (int c = 0; c < 64; ++c) sv[c] = c <= kmax ? sv[c] : -INFINITY;
      }
      // The weights are formed against the maximum at hand; only where their sum says that one may pass fp16's range (or in
      // the first tile, or when E grows) is the tile's own maximum looked for, the running maximum moved where a logit
      // passes it by 2^8, and the weights formed again. (For the whole warp: a row's maximum may move because another row's
      // does, a rounding of its weights apart. A test of each row's own sum spills at hd 128, 633 us against 576.)
      bool full = __any_sync(0xffffffffu, j == 0 || Ej > E);
      uint32_t pk[32];
      float sum;
      for (;;) {
        if (full) {
          float m4[4] = {sv[0], sv[1], sv[2], sv[3]};
#pragma unroll
          for (int c = 4; c < 60; c += 8)
#pragma unroll
            for (int k = 0; k < 4; ++k) m4[k] = fmaxf(fmaxf(m4[k], sv[c + k]), sv[c + 4 + k]);
#pragma unroll
          for (int k = 0; k < 4; ++k) m4[k] = fmaxf(m4[k], sv[60 + k]);
          const float mx = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])) * f;
          const float nm = mx > m + 8.f ? mx : m;
          const float al = m == -INFINITY ? 0.f : ex2(m - nm);
          l *= al;
          m = nm;
          if (j > 0) {
            // O is at rest once the previous tile's product is complete: scale it in place
            const float oa = al * (Ej > E ? pow2_biased(max(127 + E - Ej, 0)) : 1.f);
            if (!(ok = mbar_wait_all(&p_free[b ^ 1], ((j - 1) >> 1) & 1, ERR_TIMEOUT_OTHER, KERNEL_ID_KV4_PREFILL)))
              return false;
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < HD; c += 32) {
              float ov[32];
              tmem_ld32(tO + c, ov);
#pragma unroll
              for (int k = 0; k < 32; ++k) ov[k] *= oa;
              tmem_st32(tO + c, ov);
            }
          }
          E = max(E, Ej);
        }
        const float2 f_2 = f2(f), mb = f2(KV4P_BIAS - m);
        float2 ls[2] = {f2(0.f), f2(0.f)};
#pragma unroll
        for (int c = 0; c < 64; c += 8) {
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float2 z = ffma2(make_float2(sv[c + 2 * k], sv[c + 2 * k + 1]), f_2, mb);
            const float2 p = make_float2(ex2(z.x), ex2(z.y));
            ls[k & 1] = fadd2(ls[k & 1], p);
            pk[c / 2 + k] = pack_f16(p.x, p.y);
          }
        }
        sum = (ls[0].x + ls[0].y) + (ls[1].x + ls[1].y);
        if (full || !__any_sync(0xffffffffu, sum > 32768.f)) break;
        full = true;
      }
      tmem_st32(tS + (j & 1) * 64, reinterpret_cast<const float*>(pk));
      if (wide) {
        // the values stand divided by their keys' exponents, O by the row's E: the weights take the difference
        const uint8_t* vx = keyv + (j & 15) * 64;
#pragma unroll 1
        for (int c = 0; c < 32; c += 4) {
          float z[4];
          tmem_ld4(tS + (j & 1) * 64 + c, z);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float2 p = unpack_f16(__float_as_uint(z[k]));
            z[k] = __uint_as_float(pack_f16(p.x * pow2_diff(vx[2 * (c + k)], E), p.y * pow2_diff(vx[2 * (c + k) + 1], E)));
          }
          tmem_st4(tS + (j & 1) * 64 + c, z);
        }
      }
      l += sum;
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_full[b]);
      return true;
    };
    // (two loops: what the last tiles need is not between the instructions of the others)
    int j = 0;
    while (x < ntx && j < first && tile(std::false_type(), j)) ++j;
    while (x < ntx && ok && j < nt && tile(std::true_type(), j)) ++j;
    if (x < ntx && ok) {
      ok = mbar_wait_all(&p_free[2 * x + ((nt - 1) & 1)], ((nt - 1) >> 1) & 1, ERR_TIMEOUT_ACCUM, KERNEL_ID_KV4_PREFILL);
      tc_fence_after();
      if (ok) {
        const float inv = pow2_biased(E) / l;
        __nv_bfloat16* dst = a.out + (size_t)(q0 + r) * a.out_stride + (head0 + head) * HD;
#pragma unroll 1
        for (int c = 0; c < HD; c += 32) {
          float ov[32];
          tmem_ld32(tO + c, ov);
          const int grp = c / 32, slot = F::slot(grp);
          const float w = nanv[slot] <= pos ? __int_as_float(0x7FFFFFFF) : inv;
          if (live)
#pragma unroll
            for (int k = 0; k < 32; k += 8)
              *reinterpret_cast<uint4*>(dst + c + k) =
                  make_uint4(pack_bf16(ov[k] * w, ov[k + 1] * w), pack_bf16(ov[k + 2] * w, ov[k + 3] * w),
                             pack_bf16(ov[k + 4] * w, ov[k + 5] * w), pack_bf16(ov[k + 6] * w, ov[k + 7] * w));
        }
      }
    }
  } else if (warp < KV4P_SOFT + 2 * KV4P_DEQ) {
    A8_SETMAXNREG("dec", KV4P_REG_REST);
    // ---- codes to fp16: 128 threads for K, 128 for V
    const bool isv = warp >= KV4P_SOFT + KV4P_DEQ;
    const int dw = (warp - KV4P_SOFT) & 3, dt = dw * 32 + lane;
    for (int j = 0; j < nt; ++j) {
      const int rs = j % KV4P_RAW, st = j & 1, rph = (j / KV4P_RAW) & 1;
      if (!kv4_wait2(&raw_full[rs], rph, &e_full[rs], rph, ERR_TIMEOUT_FULL, KERNEL_ID_KV4_PREFILL)) break;
      const uint8_t* raw = smem + SM::RAW + rs * SM::RAWT;
      const __half* table = reinterpret_cast<const __half*>(smem + SM::SC + rs * SM::SCT) + (isv ? 64 * G : 0);
      if (!isv) {
        if (j >= 2 && !mbar_wait_all(&k_free[st], ((j >> 1) - 1) & 1, ERR_TIMEOUT_EMPTY, KERNEL_ID_KV4_PREFILL)) break;
        uint8_t* dst = smem + SM::K + st * SM::KT;
#pragma unroll
        for (int i = 0; i < 2; ++i) {                    // a thread: word t8 of a key, all groups
          const int r = i * 32 + (dt >> 2), t8 = dt & 3;
          const uint8_t* src = raw + (r >> 4) * F::REC + F::kword(r & 15, t8, 0);
          uint32_t w[G], ks[G / 2];
          if constexpr (G == 4) {
            const uint4 u = *reinterpret_cast<const uint4*>(src);
            w[0] = u.x; w[1] = u.y; w[2] = u.z; w[3] = u.w;
            const uint2 v = *reinterpret_cast<const uint2*>(table + r * G);
            ks[0] = v.x; ks[1] = v.y;
          } else {
            const uint2 u = *reinterpret_cast<const uint2*>(src);
            w[0] = u.x; w[1] = u.y;
            ks[0] = *reinterpret_cast<const uint32_t*>(table + r * G);
          }
#pragma unroll
          for (int s = 0; s < G; ++s) {
            const int grp = (s & 1) * (G / 2) + s / 2;
            const uint32_t hb = __byte_perm(ks[s >> 1], 0, (s & 1) ? 0x3232 : 0x1010);
            const __half2 h = *reinterpret_cast<const __half2*>(&hb);
            __half2 c[4];
            kv4_codes_f16(w[s], c);
            *reinterpret_cast<uint4*>(dst + (grp >> 1) * 8192 + sw128(r, (grp & 1) * 4 + t8)) =
                make_uint4(h2u(__hmul2(c[0], h)), h2u(__hmul2(c[1], h)), h2u(__hmul2(c[2], h)), h2u(__hmul2(c[3], h)));
          }
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&k_full[st]);
          mbar_arrive(&raw_free[rs]);
        }
      } else {
        const int part = dw >> 1;                        // this warp's half of the groups
        const int vt = j % KV4P_VST;
        if (j >= KV4P_VST && !mbar_wait_all(&v_free[vt], (j / KV4P_VST - 1) & 1, ERR_TIMEOUT_EMPTY, KERNEL_ID_KV4_PREFILL))
          break;
        uint8_t* dst = smem + SM::V + vt * SM::VT;
        // a thread: dims 4 q .. + 3 of G / 2 groups, of eight keys
        const int oct = lane & 7, q = (dw & 1) * 4 + (lane >> 3);
        uint32_t w[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const int j8 = (oct & 1) * 8 + k;
          const uint8_t* src = raw + (oct >> 1) * F::REC + F::vhalf(j8, q, part * (G / 2));
          w[k] = G == 4 ? *reinterpret_cast<const uint32_t*>(src) : *reinterpret_cast<const uint16_t*>(src);
        }
#pragma unroll
        for (int sl = 0; sl < G / 2; ++sl) {
          const int s = part * (G / 2) + sl, grp = (s & 1) * (G / 2) + s / 2;
          const uint4 hs = *reinterpret_cast<const uint4*>(table + s * 64 + oct * 8);
          const uint32_t hp[4] = {hs.x, hs.y, hs.z, hs.w};
          uint32_t o[4][4];
#pragma unroll
          for (int p = 0; p < 4; ++p) {
            const uint32_t u = __byte_perm(w[2 * p], w[2 * p + 1], sl ? 0x7632 : 0x5410);
            const __half2 h = *reinterpret_cast<const __half2*>(&hp[p]);
            __half2 c[4];
            kv4_codes_f16(u, c);
#pragma unroll
            for (int k = 0; k < 4; ++k) o[k][p] = h2u(__hmul2(c[k], h));
          }
#pragma unroll
          for (int k = 0; k < 4; ++k)
            *reinterpret_cast<uint4*>(dst + sw128(32 * grp + 4 * q + k, oct)) = make_uint4(o[k][0], o[k][1], o[k][2], o[k][3]);
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&v_full[vt]);
          mbar_arrive(&raw_free[rs]);
        }
      }
    }
  } else {
    A8_SETMAXNREG("dec", KV4P_REG_REST);
    if (warp == 16 && lane == 0) {
      const uint8_t* src = kv4_rec(a.c, F::REC, crow, kvh, 0);
      int issued = 0;
      for (int j = 0; j < nt; ++j) {
        const int rs = j % KV4P_RAW;
        if (j >= KV4P_RAW && !mbar_wait(&raw_free[rs], (j / KV4P_RAW - 1) & 1, ERR_TIMEOUT_EMPTY, KERNEL_ID_KV4_PREFILL))
          break;
        const uint32_t bytes = min(4, a.c.nblk - 4 * j) * F::REC;
        mbar_arrive_expect_tx(&raw_full[rs], bytes);
        bulk_load(smem + SM::RAW + rs * SM::RAWT, src + (size_t)j * 4 * F::REC, bytes, &raw_full[rs]);
        issued = j + 1;
      }
      // every requested copy has landed before the CTA can finish (bounded after an error)
      for (int j = max(0, issued - KV4P_RAW); j < issued; ++j)
        mbar_wait(&raw_full[j % KV4P_RAW], (j / KV4P_RAW) & 1, ERR_TIMEOUT_FULL, KERNEL_ID_KV4_PREFILL);
    }
    // a whole warp walks each issue loop (ring positions and descriptors stay warp-uniform), one lane, elected once, issues
    if (warp == 17) {
      constexpr uint32_t idS = umma_idesc(128, 64, 0);
      const uint64_t dQ = umma_desc_sw128(smem + SM::Q), dK = umma_desc_sw128(smem + SM::K);
      const bool lead = elect_one();
      bool ok = mbar_wait_all(q_full, 0, ERR_TIMEOUT_FULL, KERNEL_ID_KV4_PREFILL);
      for (int j = 0; ok && j < nt; ++j) {
        const int st = j & 1, ph = (j >> 1) & 1;
        // K of this tile; the stage's last P (in the columns of S) has been multiplied
        for (int x = 0; x < ntx; ++x) {
          ok = j < 2 ? mbar_wait_all(&k_full[st], ph, ERR_TIMEOUT_FULL, KERNEL_ID_KV4_PREFILL)
                     : kv4_wait2(&k_full[st], ph, &p_free[2 * x + st], ph ^ 1, ERR_TIMEOUT_FULL, KERNEL_ID_KV4_PREFILL);
          if (!ok) break;
          tc_fence_after();
          if (lead) {
            const uint32_t d = tmem + x * 128 + st * 64;
            const uint64_t da = dQ + x * (SM::QT >> 4), db = dK + st * (SM::KT >> 4);
#pragma unroll
            for (int k = 0; k < HD / 16; ++k)
              umma_f16(d, da + (k >> 2) * (16384 >> 4) + 2 * (k & 3), db + (k >> 2) * (8192 >> 4) + 2 * (k & 3), idS, k != 0);
            umma_commit(&s_full[2 * x + st]);
            mbar_arrive(&s_full[2 * x + st]);
            if (x == ntx - 1) umma_commit(&k_free[st]);
          }
          __syncwarp();
        }
      }
    } else if (warp == 18) {
      constexpr uint32_t idO = umma_idesc(128, HD, 0);
      const uint64_t dV = umma_desc_sw128(smem + SM::V);
      const bool lead = elect_one();
      int vt = 0, vph = 0;
      for (int j = 0; j < nt; ++j) {
        const int st = j & 1;
        bool ok = true;
        for (int x = 0; x < ntx; ++x) {
          ok = kv4_wait2(&p_full[2 * x + st], (j >> 1) & 1, &v_full[vt], vph, ERR_TIMEOUT_FULL, KERNEL_ID_KV4_PREFILL);
          if (!ok) break;
          tc_fence_after();
          if (lead) {
            const uint64_t db = dV + vt * (SM::VT >> 4);
            const uint32_t d = tmem + 256 + x * HD, ta = tmem + x * 128 + st * 64;
#pragma unroll
            for (int k = 0; k < 4; ++k) umma_f16_ts(d, ta + 8 * k, db + 2 * k, idO, (j > 0) | (k != 0));
            umma_commit(&p_free[2 * x + st]);
            if (x == ntx - 1) umma_commit(&v_free[vt]);
          }
          __syncwarp();
        }
        if (!ok) break;
        if (++vt == KV4P_VST) {
          vt = 0;
          vph ^= 1;
        }
      }
    } else if (warp == 19) {
      // The exponents of each tile's largest scales (V's only grows), and the scales as fp16, K's divided by 2^ek, V's by
      // 2^E: two positions a lane. (One warp for the other eight: it shares its scheduler with as many of them as any.)
      const int k0 = 2 * lane, off[2] = {(k0 >> 4) * F::REC + F::scale(k0 & 15, 0),
                                         (k0 >> 4) * F::REC + F::scale((k0 + 1) & 15, 0)};
      auto largest = [](const uint32_t (&w)[2][G / 2]) {
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < G / 2; ++i) m = __vmaxu2(m, __vmaxu2(w[0][i], w[1][i]));
        return __reduce_max_sync(0xffffffffu, max(m & 0xFFFFu, m >> 16));
      };
      // the smallest of the lane's scales but zero, less 32,769 (a zero counts as large: as a signed number of 16 bits, w + 0x7FFF)
      auto least = [](const uint32_t (&w)[2][G / 2]) {
        uint32_t m = 0x7FFF7FFFu;
#pragma unroll
        for (int i = 0; i < G / 2; ++i) m = __vmins2(m, __vmins2(w[0][i] + 0x7FFF7FFFu, w[1][i] + 0x7FFF7FFFu));
        return min(int(int16_t(m)), int(m) >> 16);
      };
      auto without_nan = [](const uint32_t (&w)[2][G / 2], uint32_t (&o)[2][G / 2]) {
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
          for (int i = 0; i < G / 2; ++i)
            o[k][i] = ((w[k][i] & 0xFFFFu) < 0x7F80u ? w[k][i] & 0xFFFFu : 0u) | (w[k][i] < 0x7F800000u ? w[k][i] & 0xFFFF0000u : 0u);
      };
      int E = 1;
      for (int j = 0; j < nt; ++j) {
        const int rs = j % KV4P_RAW;
        if (!mbar_wait_all(&raw_full[rs], (j / KV4P_RAW) & 1, ERR_TIMEOUT_FULL, KERNEL_ID_KV4_PREFILL)) break;
        const uint8_t* raw = smem + SM::RAW + rs * SM::RAWT;
        const int left = klen - 64 * j;
        uint32_t kw[2][G / 2], vw[2][G / 2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          if constexpr (G == 4) {
            const uint2 x = *reinterpret_cast<const uint2*>(raw + F::KS0 + off[k]);
            kw[k][0] = x.x; kw[k][1] = x.y;
            const uint2 y = *reinterpret_cast<const uint2*>(raw + F::VS0 + off[k]);
            vw[k][0] = y.x; vw[k][1] = y.y;
          } else {
            kw[k][0] = *reinterpret_cast<const uint32_t*>(raw + F::KS0 + off[k]);
            vw[k][0] = *reinterpret_cast<const uint32_t*>(raw + F::VS0 + off[k]);
          }
          if (k0 + k >= left)                            // behind the last key: whatever the record holds there
#pragma unroll
            for (int i = 0; i < G / 2; ++i) kw[k][i] = vw[k][i] = 0;
        }
        uint32_t topk = largest(kw), topv = largest(vw);
        if (topk >= 0x7F80u) {                           // a NaN scale of K stays NaN but does not count
          uint32_t x[2][G / 2];
          without_nan(kw, x);
          topk = largest(x);
        }
        if (topv >= 0x7F80u) {                           // one of V counts as zero here and is put back at the end
#pragma unroll
          for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int i = 0; i < G / 2; ++i) {
              if ((vw[k][i] & 0xFFFFu) >= 0x7F80u) atomicMin(&nanv[2 * i], 64 * j + k0 + k);
              if (vw[k][i] >= 0x7F800000u) atomicMin(&nanv[2 * i + 1], 64 * j + k0 + k);
            }
          uint32_t x[2][G / 2];
          without_nan(vw, x);
#pragma unroll
          for (int i = 0; i < G / 2; ++i) {
            vw[0][i] = x[0][i];
            vw[1][i] = x[1][i];
          }
          topv = largest(vw);
        }
        const int ex = min(max(int(topk >> 7), 1), 253), before = E;
        E = max(E, min(int(topv >> 7), 253));
        const float dk = pow2_biased_inv(ex), dv = pow2_biased_inv(E);
        // Scales 2^14 below the largest are past what fp16 holds exactly, and in the block's own tiles the largest may be that
        // of a key behind a row.
        const bool wide = 64 * j + 63 > pos0 &&
                          __any_sync(0xffffffffu, least(kw) < (ex - 14) * 128 - 32769 || least(vw) < (E - 14) * 128 - 32769 ||
                                                      (before > 1 && before + 14 < E));
        __half* tk = reinterpret_cast<__half*>(smem + SM::SC + rs * SM::SCT);
        __half* tv = tk + 64 * G;
#pragma unroll
        for (int i = 0; i < G / 2; ++i) {
          float2 v[2];
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const float2 x = unpack_bf16(kw[k][i]), y = unpack_bf16(vw[k][i]);
            *reinterpret_cast<uint32_t*>(tk + (k0 + k) * G + 2 * i) = pack_f16(x.x * dk, x.y * dk);
            v[k] = make_float2(y.x * dv, y.y * dv);
          }
          *reinterpret_cast<uint32_t*>(tv + 2 * i * 64 + k0) = pack_f16(v[0].x, v[1].x);
          *reinterpret_cast<uint32_t*>(tv + (2 * i + 1) * 64 + k0) = pack_f16(v[0].y, v[1].y);
        }
        if (wide) {
          // each key divided by its own largest scale's exponents instead; each row goes by the keys that it attends
#pragma unroll 1
          for (int k = k0; k < k0 + 2; ++k) {
            const uint32_t* ks = reinterpret_cast<const uint32_t*>(raw + F::KS0 + (k >> 4) * F::REC + F::scale(k & 15, 0));
            const uint32_t* vs = ks + (F::VS0 - F::KS0) / 4;
            uint32_t kt = 0, vt = 0;
            auto finite = [](uint32_t h) { return h < 0x7F80u ? h : 0u; };
#pragma unroll
            for (int i = 0; i < G / 2; ++i) {
              kt = max(kt, max(finite(ks[i] & 0xFFFFu), finite(ks[i] >> 16)));
              vt = max(vt, max(finite(vs[i] & 0xFFFFu), finite(vs[i] >> 16)));
            }
            const int ak = k < left ? min(max(int(kt >> 7), 1), 253) : 1, av = k < left ? min(max(int(vt >> 7), 1), 253) : 1;
            keyk[(j & 15) * 64 + k] = uint8_t(ak);
            keyv[(j & 15) * 64 + k] = uint8_t(av);
#pragma unroll
            for (int i = 0; i < G / 2; ++i) {
              const float2 x = unpack_bf16(k < left ? ks[i] : 0u);
              *reinterpret_cast<uint32_t*>(tk + k * G + 2 * i) = pack_f16(x.x * pow2_biased_inv(ak), x.y * pow2_biased_inv(ak));
              const uint32_t w = k < left ? vs[i] : 0u;
              const float2 y = unpack_bf16(finite(w & 0xFFFFu) | finite(w >> 16) << 16);
              tv[2 * i * 64 + k] = __float2half_rn(y.x * pow2_biased_inv(av));
              tv[(2 * i + 1) * 64 + k] = __float2half_rn(y.y * pow2_biased_inv(av));
            }
          }
        }
        __syncwarp();
        if (lane == 0) {
          ek[j & 15] = ex | (wide ? KV4P_WIDE : 0);
          ev[j & 15] = E;
          mbar_arrive(&e_full[rs]);
          mbar_arrive(&raw_free[rs]);
        }
        __syncwarp();
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 17) tmem_dealloc(tmem, SM::COLS);
}

template <int HD>
static int kv4_prefill_launch(Kv4AttnArgs& a, int nblocks, cudaStream_t s) {
  const void* fn = (const void*)k_kv4_prefill<HD>;
  static std::atomic<uint64_t> ready{0};
  if (!kv4_ready(ready, fn, Kv4PreSmem<HD>::TOTAL, kv4p_registers_cover)) return A8_ERR_CUDA;
  const long long per = (long long)a.c.nkv * ((a.group + 3) / 4);
  if (nblocks * per >= (1ll << 31)) return A8_ERR_SIZE;
  void* args[] = {&a};
  return kv4_launch(fn, dim3(unsigned(nblocks * per)), KV4P_THREADS, Kv4PreSmem<HD>::TOTAL, args, s) ==
                 cudaSuccess ? A8_OK : A8_ERR_CUDA;
}

}  // namespace a8

using namespace a8;

extern "C" int a8_kv4_prefill_attention(const A8KV4* c, int layer, const void* q, int q_stride, int nq,
                                        const int* blocks, int nblocks, int rows, float scale, void* out,
                                        int out_stride, a8_stream_t stream) {
  Kv4AttnArgs a;
  int rc = kv4_attn_args(&a, c, layer, q, q_stride, nq, rows, scale, out, out_stride);
  if (rc) return rc;
  // (in place: a CTA reads the queries of its rows and heads before it writes their results)
  if (blocks == nullptr || nblocks <= 0 || (out == q && out_stride != q_stride)) return A8_ERR_ARG;
  a.blocks = blocks;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  return c->hd == 64 ? kv4_prefill_launch<64>(a, nblocks, s) : kv4_prefill_launch<128>(a, nblocks, s);
}
