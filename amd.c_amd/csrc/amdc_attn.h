// amdc_attn.h -- the device code of the paged cache and the attention over it (amdc_kv of amdc_q4.h describes the
// layout); part of amdc_kernels.hip's translation unit.
//
//   amdc_kv_append_{f16,bf16}   rotation, keys and values into the cache, rotated queries
//   amdc_attn_dec_h{64,128,256}_{f16,f16_f32,bf16,bf16_f32}
//                               attention of a few new tokens per sequence
//   amdc_attn_pre_h{64,128,256}_{f16,f16_f32,bf16,bf16_f32}, amdc_attn_join_{f32,f16,bf16}
//                               attention of prompts and prompt chunks

// ------------------------------------------------------------------ helpers

__device__ __forceinline__ u32 uniform(u32 v) { return (u32)__builtin_amdgcn_readfirstlane((int)v); }
// n / d rounded up
__device__ __forceinline__ u32 cdiv(u32 n, u32 d) { return (n + d - 1u) / d; }

__device__ __forceinline__ void kv_bad(const amdc_kv_dev &kv, u32 why) { __hip_atomic_store(kv.bad, why, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }

// The largest b of 0 .. n - 1 with base(b) <= u, of values that do not decrease with base(0) <= u; every lane of the
// wave gets it. 64 candidates a step: one load for up to 64 sequences, two for 4096. Whatever base() gives, the
// result is in range.
template <class F>
__device__ __forceinline__ u32 find_seq(u32 n, u32 u, F base) {
  const u32 lane = threadIdx.x & 63u;
  u32 lo = 0u, span = n;
  while (span > 1u) {
    const u32 step = cdiv(span, 64u);
    const bool in = lane * step < span;
    const u64 hit = __ballot(in && base(lo + (in ? lane * step : 0u)) <= u);
    const u32 c = hit ? (u32)__popcll(hit) - 1u : 0u;
    lo += c * step;
    span = span - c * step < step ? span - c * step : step;
  }
  return (u32)__builtin_amdgcn_readfirstlane((int)lo);
}

// The new rows of sequence b: first row and count, and its length. m = 0: none, or the sequence takes no part, or
// (after the flag is set) they cannot be trusted.
struct SeqRows {
  u32 row0, m, len;
  bool bad;
};
__device__ __forceinline__ SeqRows seq_rows(const amdc_kv_dev &kv, const int *cu, u32 T, u32 b) {
  SeqRows s = {b * T, T, 0u, false};
  const int L = kv.len[b];
  if (cu) {
    const int c0 = cu[b], c1 = cu[b + 1u];
    if (c0 < 0 || c1 < c0 || (u32)c1 > T) {
      kv_bad(kv, AMDC_BAD_ROWS);
      return {0u, 0u, 0u, true};
    }
    s.row0 = (u32)c0, s.m = (u32)(c1 - c0);
  }
  if (s.m == 0u || L == 0) return s; // len 0: no part
  if (L < 0 || (u32)L > kv.cap || (u32)L < s.m) {
    kv_bad(kv, AMDC_BAD_LEN);
    s.bad = true;
    return s;
  }
  s.len = (u32)L;
  return s;
}

// two f32 -> two f16 or bf16 in one register, rounded to nearest even
template <bool BF>
__device__ __forceinline__ u32 pack2(float a, float b) {
  if constexpr (BF) {
    return __builtin_bit_cast(u32, __builtin_convertvector((v2f){a, b}, b2)); // v_cvt_pk_bf16_f32
  } else {
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(u32, (h2){(_Float16)a, (_Float16)b});
  }
}
template <bool BF>
__device__ __forceinline__ float lo16(u32 v) { return BF ? __builtin_bit_cast(float, v << 16) : h2f(v); }
template <bool BF>
__device__ __forceinline__ float hi16(u32 v) { return BF ? __builtin_bit_cast(float, v & 0xFFFF0000u) : h2f(v >> 16); }

// sin and cos of `a` in 64 bits: the quadrant by Cody and Waite's two-part pi / 2, then the Taylor polynomials, off by
// under 2^-40 on |r| <= pi / 4, so that the f32 results are those of the exact angle. a is at most 2^31 times a
// frequency: 64 bits keep the fraction of a turn that f32 loses from positions of some thousand on.
__device__ __forceinline__ void sincos64(double a, float &s, float &c) {
  const double k = __builtin_rint(a * 0.63661977236758134308);
  double r = __builtin_fma(-k, 1.57079632679489655800, a);
  r = __builtin_fma(-k, 6.12323399573676603587e-17, r);
  const double z = r * r;
  double p = 1.0 / 6227020800.0;
  p = __builtin_fma(p, z, -1.0 / 39916800.0);
  p = __builtin_fma(p, z, 1.0 / 362880.0);
  p = __builtin_fma(p, z, -1.0 / 5040.0);
  p = __builtin_fma(p, z, 1.0 / 120.0);
  p = __builtin_fma(p, z, -1.0 / 6.0);
  p = __builtin_fma(p * z, r, r);
  double q = 1.0 / 479001600.0;
  q = __builtin_fma(q, z, -1.0 / 3628800.0);
  q = __builtin_fma(q, z, 1.0 / 40320.0);
  q = __builtin_fma(q, z, -1.0 / 720.0);
  q = __builtin_fma(q, z, 1.0 / 24.0);
  q = __builtin_fma(q, z, -0.5);
  q = __builtin_fma(q, z, 1.0);
  const double quad = k - 4.0 * __builtin_rint(k * 0.25); // -2 .. 2: k mod 4, exact
  const int n = (int)quad & 3;
  const double sn = n & 1 ? q : p, cn = n & 1 ? p : q;
  s = (float)(n & 2 ? -sn : sn);
  c = (float)((n + 1) & 2 ? -cn : cn);
}

// ------------------------------------------------------------------ append

// Eight values of a row from p (16-byte aligned where vec)
__device__ __forceinline__ void load8(const float *p, bool vec, float (&x)[8]) {
  if (vec) {
    const v4f a = ((const v4f *)p)[0], b = ((const v4f *)p)[1];
#pragma unroll
    for (int i = 0; i < 4; i++) x[i] = a[i], x[4 + i] = b[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; i++) x[i] = p[i];
  }
}

// Reading and writing bound it. Queries and keys: the first nrw workgroups, a wave to a row (or gq waves, where the rows are few). The
// row's n_rot / 2 angles once, into the wave's part of the LDS, then eight values a lane, whole heads at a time: a key's eight are 16
// bytes of the cache. Where the pairs are halves apart a lane reads the other eight as well (from the L1) instead of trading them.
// Values: the other workgroups, gv of them to a group of eight positions of a sequence, aligned as the cache is (for ragged rows,
// cu[b] / 8 + 2 b is a first group of b's that leaves room for its floor(m / 8) + 2 at most). A thread reads one value (four, where the
// rows are aligned) of up to eight rows and stores each value's positions as 16 bytes, or where the group is not full the new ones alone.
// Measured on MI355X: 8657 rows of 32 + 8 + 8 heads of 128 (319 MB) 79 us; a workgroup to a row 87, three to a row 110.
template <bool BF>
__device__ __forceinline__ void append_body(const amdc_kv_dev &kv, const amdc_append_args &a) {
  __shared__ float s_cos[4][128], s_sin[4][128];
  const u32 hd = 1u << a.lghd, tid = threadIdx.x, nrw = cdiv(a.rows * a.gq, 4u);
  const u64 gb = 32ull << a.lghd, lgg = kv.lgp - 4u; // bytes of 16 positions of a head, log2 of such groups in a page
  if (blockIdx.x < nrw) {
    const u32 lane = tid & 63u, wv = uniform(tid >> 6), w = 4u * blockIdx.x + wv, row = w / a.gq, part = w - row * a.gq;
    if (row >= a.rows) return;
    const u32 b = a.cu ? find_seq(kv.n_seq, row, [&](u32 i) { const int c = a.cu[i]; return c < 0 ? 0u : (u32)c; }) : row / a.T;
    const SeqRows s = seq_rows(kv, a.cu, a.T, b);
    if (!s.len || row < s.row0 || row - s.row0 >= s.m) return;
    const u32 pos = s.len - s.m + (row - s.row0);
    const int id = kv.pages[(u64)b * kv.max_pages + (pos >> kv.lgp)];
    const bool ok = (u32)id < kv.n_pages;
    if (!ok) kv_bad(kv, AMDC_BAD_PAGE);
    const u32 half = a.n_rot >> 1;
    if (a.rope) {
      for (u32 i = lane; i < half; i += 64u) sincos64((double)pos * (double)a.freq[i], s_sin[wv][i], s_cos[wv][i]);
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront"); // the wave's own LDS: in order, once the compiler keeps them so
      __builtin_amdgcn_wave_barrier();
    }
    const u32 nq = a.q ? a.n_q : 0u, nh = nq + kv.n_kv, hpi = 512u >> a.lghd;
    const u32 slot = pos & ((1u << kv.lgp) - 1u), c = lane & ((hd >> 3) - 1u);
    for (u32 h0 = part * hpi; h0 < nh; h0 += a.gq * hpi) {
      const u32 h = h0 + (lane >> (a.lghd - 3u));
      if (h >= nh) break;
      float x[8];
      const float *src = h < nq ? a.q + (u64)row * a.qs + (u64)h * hd : a.k + (u64)row * a.ks + (u64)(h - nq) * hd;
      load8(src + 8u * c, a.vec & (h < nq ? 1u : 2u), x);
      if (a.rope == 1u) { // pairs
#pragma unroll
        for (u32 i = 0; i < 8u; i += 2u) {
          const u32 e = 8u * c + i;
          if (e < a.n_rot) {
            const float cs = s_cos[wv][e >> 1], sn = s_sin[wv][e >> 1], u = x[i], v = x[i + 1u];
            x[i] = u * cs - v * sn, x[i + 1u] = u * sn + v * cs;
          }
        }
      } else if (a.rope == 2u && 8u * c < a.n_rot) { // halves
        float o[8];
        if (!(half & 7u)) load8(src + (8u * c < half ? 8u * c + half : 8u * c - half), a.vec & (h < nq ? 1u : 2u), o);
        else
#pragma unroll
          for (u32 i = 0; i < 8u; i++) {
            const u32 e = 8u * c + i;
            o[i] = e < a.n_rot ? src[e < half ? e + half : e - half] : 0.0f;
          }
#pragma unroll
        for (u32 i = 0; i < 8u; i++) {
          const u32 e = 8u * c + i;
          if (e < a.n_rot) {
            const u32 f = e < half ? e : e - half;
            const float cs = s_cos[wv][f], sn = s_sin[wv][f];
            x[i] = e < half ? x[i] * cs - o[i] * sn : o[i] * sn + x[i] * cs;
          }
        }
      }
      // queries in place: a head is one wave's, in one pass, and all of the wave's reads are back before its first write
      if (a.q == (const float *)a.qo) __builtin_amdgcn_s_waitcnt(0x0F70);
      if (h >= nq) {
        if (!ok) continue;
        const u32x4 v = {pack2<BF>(x[0], x[1]), pack2<BF>(x[2], x[3]), pack2<BF>(x[4], x[5]), pack2<BF>(x[6], x[7])};
        *(u32x4 *)(kv.k + (((((u64)(u32)id * kv.n_kv + (h - nq)) << lgg) + (slot >> 4)) * gb + 256u * c + 16u * (slot & 15u))) = v;
      } else if (a.qt == 0u) {
        float *d = (float *)a.qo + (u64)row * a.qos + (u64)h * hd + 8u * c;
        if (a.vec & 4u) ((v4f *)d)[0] = (v4f){x[0], x[1], x[2], x[3]}, ((v4f *)d)[1] = (v4f){x[4], x[5], x[6], x[7]};
        else
#pragma unroll
          for (int i = 0; i < 8; i++) d[i] = x[i];
      } else {
        const u32x4 v = {pack2<BF>(x[0], x[1]), pack2<BF>(x[2], x[3]), pack2<BF>(x[4], x[5]), pack2<BF>(x[6], x[7])};
        unsigned short *d = (unsigned short *)a.qo + (u64)row * a.qos + (u64)h * hd + 8u * c;
        if (a.vec & 4u) *(u32x4 *)d = v;
        else
#pragma unroll
          for (int i = 0; i < 8; i++) d[i] = (unsigned short)(v[i >> 1] >> (16 * (i & 1)));
      }
    }
    return;
  }
  const u32 vb = blockIdx.x - nrw, u = vb / a.gv, part = vb - u * a.gv;
  u32 b, gi;
  if (a.cu) {
    auto base = [&](u32 i) { const int c = a.cu[i]; return (c < 0 ? 0u : (u32)c >> 3) + 2u * i; };
    b = find_seq(kv.n_seq, u, base);
    gi = u - base(b);
  } else
    b = u / a.upb, gi = u - b * a.upb;
  const SeqRows s = seq_rows(kv, a.cu, a.T, b);
  if (!s.len) return;
  const u32 start = s.len - s.m, grp = (start >> 3) + gi;
  if (8ull * grp >= s.len) return;
  const u32 p0 = 8u * grp, j0 = p0 < start ? start - p0 : 0u, j1 = s.len - p0 < 8u ? s.len - p0 : 8u;
  const int id = kv.pages[(u64)b * kv.max_pages + (p0 >> kv.lgp)];
  if ((u32)id >= kv.n_pages) return; // flagged by the row's own workgroup
  const u32 g = (p0 & ((1u << kv.lgp) - 1u)) >> 3, n = kv.n_kv << a.lghd;
  const float *src = a.v + (u64)(s.row0 + (p0 + j0 - start)) * a.vs;
  auto put8 = [&](uint8_t *to, u32x4 w) { // a value's eight positions, or the new ones of them
    if (j1 - j0 == 8u) *(u32x4 *)to = w;
    else
#pragma unroll
      for (u32 j = 0; j < 8u; j++)
        if (j >= j0 && j < j1) ((unsigned short *)to)[j] = (unsigned short)(w[j >> 1] >> (16u * (j & 1u)));
  };
  if (a.vec & 8u) { // four values a thread
    for (u32 i = 4u * (part * 256u + tid); i < n; i += a.gv * 1024u) {
      const u32 h = i >> a.lghd, d = i & (hd - 1u);
      v4f x[8];
#pragma unroll
      for (u32 j = 0; j < 8u; j++) x[j] = j >= j0 && j < j1 ? *(const v4f *)(src + (u64)(j - j0) * a.vs + i) : (v4f){0.0f, 0.0f, 0.0f, 0.0f};
      uint8_t *to = kv.v + (((((u64)(u32)id * kv.n_kv + h) << (lgg + 1u)) + g) * (gb >> 1) + 16u * d);
#pragma unroll
      for (u32 e = 0; e < 4u; e++) {
        const u32x4 w = {pack2<BF>(x[0][e], x[1][e]), pack2<BF>(x[2][e], x[3][e]), pack2<BF>(x[4][e], x[5][e]), pack2<BF>(x[6][e], x[7][e])};
        put8(to + 16u * e, w);
      }
    }
    return;
  }
  for (u32 i = part * 256u + tid; i < n; i += a.gv * 256u) {
    const u32 h = i >> a.lghd, d = i & (hd - 1u);
    float x[8];
#pragma unroll
    for (u32 j = 0; j < 8u; j++) x[j] = j >= j0 && j < j1 ? src[(u64)(j - j0) * a.vs + i] : 0.0f;
    const u32x4 w = {pack2<BF>(x[0], x[1]), pack2<BF>(x[2], x[3]), pack2<BF>(x[4], x[5]), pack2<BF>(x[6], x[7])};
    put8(kv.v + (((((u64)(u32)id * kv.n_kv + h) << (lgg + 1u)) + g) * (gb >> 1) + 16u * d), w);
  }
}

#define APPEND_KERNEL(KN, BF) \
  extern "C" __global__ __launch_bounds__(256) void amdc_kv_append_##KN(amdc_kv_dev kv, amdc_append_args a) { append_body<BF>(kv, a); }
APPEND_KERNEL(f16, false)
APPEND_KERNEL(bf16, true)
#undef APPEND_KERNEL

// ------------------------------------------------------------------ attention of a few new tokens

typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef short s4 __attribute__((ext_vector_type(4)));

template <bool BF>
__device__ __forceinline__ v4f mfma16(u32x4 a, u32x4 b, v4f c) {
  typedef _Float16 h8 __attribute__((ext_vector_type(8)));
  if constexpr (BF) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
}

// x in NP 16-bit parts whose sum is x to 11 NP (f16) or 8 NP (bf16) bits: each part rounds what the parts before it left
template <bool BF, int NP>
__device__ __forceinline__ void split8(float (&x)[8], u32x4 (&w)[NP]) {
#pragma unroll
  for (int p = 0; p < NP; p++)
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const u32 v = pack2<BF>(x[2 * i], x[2 * i + 1]);
      w[p][i] = v;
      if (p + 1 < NP) x[2 * i] -= lo16<BF>(v), x[2 * i + 1] -= hi16<BF>(v);
    }
}

// Eight query values: f32 (as given), or 16 bits widened
template <bool BF, bool F32>
__device__ __forceinline__ void load_q8(const void *q, u64 i, bool vec, float (&x)[8]) {
  if constexpr (F32) load8((const float *)q + i, vec, x);
  else {
    u32x4 w;
    const unsigned short *p = (const unsigned short *)q + i;
    if (vec) w = *(const u32x4 *)p;
    else
#pragma unroll
      for (int k = 0; k < 4; k++) w[k] = (u32)p[2 * k] | (u32)p[2 * k + 1] << 16;
#pragma unroll
    for (int k = 0; k < 4; k++) x[2 * k] = lo16<BF>(w[k]), x[2 * k + 1] = hi16<BF>(w[k]);
  }
}

// Four results of a row to y
template <bool BF, bool F32>
__device__ __forceinline__ void store_y4(void *y, u64 i, v4f v, bool vec) {
  if constexpr (F32) {
    float *d = (float *)y + i;
    if (vec) *(v4f *)d = v;
    else
#pragma unroll
      for (int k = 0; k < 4; k++) d[k] = v[k];
  } else {
    const u32x2 w = {pack2<BF>(v.x, v.y), pack2<BF>(v.z, v.w)};
    unsigned short *d = (unsigned short *)y + i;
    if (vec) *(u32x2 *)d = w;
    else
#pragma unroll
      for (int k = 0; k < 4; k++) d[k] = (unsigned short)(w[k >> 1] >> (16 * (k & 1)));
  }
}

// Are all of a wave's values finite?
__device__ __forceinline__ bool wave_finite(v4f c) {
  const float z = (c.x - c.x) + (c.y - c.y) + (c.z - c.z) + (c.w - c.w); // NaN where one is not
  return __ballot(!(z == 0.0f)) == 0ull;
}

// the 16-bit halves of w (positions p, p + 1, ..) that lie outside [lo, hi), as 0
template <class V>
__device__ __forceinline__ V seen16(V w, u32 p, u32 lo, u32 hi) {
#pragma unroll
  for (u32 i = 0; i < sizeof(V) / 4u; i++) {
    const u32 a = p + 2u * i, b = a + 1u;
    w[i] &= (a >= lo && a < hi ? 0xFFFFu : 0u) | (b >= lo && b < hi ? 0xFFFF0000u : 0u);
  }
  return w;
}

#define DEC_FAN 8u      // partial results joined at once
#define DEC_CMIN 512u   // the shortest chunk, in positions
#define DEC_NT 327680u  // the bytes of a chunk from which its loads are nontemporal

// The sum of v over the lanes up to this one, itself included (in lane 63: over the wave)
__device__ __forceinline__ u32 wave_scan(u32 v) {
  // row_shr 1, 2, 4, 8 inside rows of 16, then the rows' last lanes onto the rows behind (row_bcast 15 and 31)
  v += (u32)__builtin_amdgcn_update_dpp(0, (int)v, 0x111, 0xF, 0xF, false);
  v += (u32)__builtin_amdgcn_update_dpp(0, (int)v, 0x112, 0xF, 0xF, false);
  v += (u32)__builtin_amdgcn_update_dpp(0, (int)v, 0x114, 0xF, 0xF, false);
  v += (u32)__builtin_amdgcn_update_dpp(0, (int)v, 0x118, 0xF, 0xF, false);
  v += (u32)__builtin_amdgcn_update_dpp(0, (int)v, 0x142, 0xA, 0xF, false);
  v += (u32)__builtin_amdgcn_update_dpp(0, (int)v, 0x143, 0xC, 0xF, false);
  return v;
}
__device__ __forceinline__ u32 lane_of(u32 v, u32 lane) { return (u32)__builtin_amdgcn_readlane((int)v, (int)lane); }

// N weights or queries in NP parts, the operands of a step of 32 (N = 8) or 16 (4) positions
template <bool BF, int NP, int N>
__device__ __forceinline__ void split_n(float (&x)[N], u32 (&w)[NP][N / 2]) {
#pragma unroll
  for (int p = 0; p < NP; p++)
#pragma unroll
    for (int i = 0; i < N / 2; i++) {
      const u32 v = pack2<BF>(x[2 * i], x[2 * i + 1]);
      w[p][i] = v;
      if (p + 1 < NP) x[2 * i] -= lo16<BF>(v), x[2 * i + 1] -= hi16<BF>(v);
    }
}

// T rows of G = n_q / n_kv heads of a sequence read the same keys and values. A workgroup takes 16 NC of these T G
// columns (blocks cb of them), one key / value head and one chunk of the sequence's positions; its NW waves take
// the chunk's steps of SP positions in turn, each with a softmax of its own (maximum m, sum l, weighted sum O), joined at
// the end in the LDS.
//
// Reading the cache bounds it: 16 columns cost 4 x 16 x hd flops per 4 hd bytes, a key and a value; at the HBM's 6.3 TB/s that is 1 / 12 of a
// large product's rate (1210 TFLOP/s), in f32's two or three parts 1 / 6 or 1 / 4. So the layout gives every load of a wave whole lines, straight into the matrix units' operands, no LDS between:
//   S^T = K Q^T  (16x16x32: rows are positions, columns are the query rows). SP = 32: row r of tile t (of two) is position
//                8 (r / 4) + 4 t + r % 4 of the step, so that a lane's eight scores are the eight positions 8 g .. 8 g + 7
//                (g = lane / 16) of its column. SP = 16, for heads of 256, whose O and loads in flight fill the registers at half
//                the step: row r is position r, a lane's four scores are 4 g .. 4 g + 3
//   O^T = V^T P^T: those, as 16-bit weights, are the lane's B operand (16x16x32, or 16x16x16) as they stand; the cache keeps a
//                value's eight positions together, which is the A operand.
// In f32, queries and weights go in as sums of 16-bit parts (f16: two, 22 bits; bf16: three, 24), one product each, into the
// same sums; f16 queries are first scaled by a power of two that brings a row's largest value to 2^10 (no overflow, and the second part
// stays a normal number). f16 weights carry 2^8 (their least normal is 2^-14), the sum l the same factor.
// The maximum is raised, and O rescaled, only where a score passes it by 6 (weights stay under 2^14): the join needs a common
// reference, not the largest score.
//
// Chunks: the device divides all sequences' steps by the number of units U that the host wants of a head, so that chunks are
// about equal however different the lengths are; every wave finds its unit by a scan over the lengths. A sequence's chunks
// leave partial results (O, m, l) in the workspace, agent-coherent as split_put's; of every DEC_FAN neighbours the last to arrive
// joins them, in their order, up a tree, so the result does not depend on who was last.
//
// A step that holds positions which not every column sees is multiplied into sums of its own: where these come out finite they are
// added, as weights of 0 are right; if not (0 times an infinity or a NaN that a column must not see), again with what no column sees as
// 0, and if that is not enough token by token with what it does not see as 0.
//
// Measured on MI355X (replayed, buffers in turn; cards differ by 5 %): 60001 positions, 24 / 4 heads of 256, f16, f32 queries (246 MB) 47 to
// 49 us, 5.0 to 5.2 TB/s (bf16, f32 queries 49); 64 sequences of 30 to 16000, 32 / 8 heads of 128, bf16 (699 MB) 135 to 141 us, 5.0 to 5.2 TB/s;
// 8 sequences of 900 to 6000, T = 5, 24 / 4 heads of 256 (104 MB, two blocks of columns, the second from the L2) 34 us, 3.1 TB/s; 421
// positions, 32 / 32 heads of 128 8.3 us, all latency.
// A plain read reaches 6.3 TB/s. Four waves a workgroup, two workgroups a CU and loads not ahead of the queries: 54, 151 and 54 us.
template <int HD, bool BF, bool F32, u32 NC, u32 NW>
__device__ __forceinline__ void dec_body(const amdc_kv_dev &kv, const amdc_attn_args &a) {
  constexpr int NP = F32 ? (BF ? 3 : 2) : 1, KS = HD / 32, DT = HD / 16;
  constexpr u32 SP = HD > 128 || (NC > 1u && HD > 64) ? 16u : 32u, SL = SP / 4u, TT = SP / 16u, R = 16u * NC, NTH = 64u * NW; // positions of a step, scores of a lane, score tiles
  constexpr u32 OS = HD + 4u, QD = HD / 4u; // floats between columns of O in the LDS; quads of a row
  constexpr float BIAS = BF ? 0.0f : 8.0f, RAISE = 6.0f, NINF = -__builtin_inff();
  constexpr u32 NS = NW > 4u && HD * NC > 256 ? 4u : NW, SMQ = NP * HD * 2u * R, SMO = NS * R * OS * 4u, SMB = SMQ > SMO ? SMQ : SMO;
  typedef u32 op __attribute__((ext_vector_type(SL / 2))); // SL 16-bit values
  __shared__ __attribute__((aligned(16))) uint8_t sm[SMB];
  __shared__ float s_cq[R], s_m[NW][R], s_l[NW][R], s_L[R], s_M[R];
  __shared__ u32 s_bad, s_last;
  const u32 tid = threadIdx.x, lane = tid & 63u, wv = (u32)__builtin_amdgcn_readfirstlane((int)(tid >> 6)), n = lane & 15u, g4 = lane >> 4;
  // the blocks of columns of a unit are 8 workgroups apart: on one XCD, whose L2 the second to read finds the cache in
  const u32 cb = blockIdx.x / 8u % a.ncb, x = blockIdx.x / (8u * a.ncb) * 8u + (blockIdx.x & 7u);
  const u32 h = x % kv.n_kv, u = x / kv.n_kv, T = a.T, G = a.G;

  // the unit: sequence b, its chunk ci of nu, of C steps
  auto trust = [&](int L) { return (u32)L - 1u < kv.cap && (u32)L >= T; }; // 1 .. cap, the new rows among them
  auto first = [&](u32 L) { return a.window && L - T + 1u > a.window ? L - T + 1u - a.window : 0u; }; // the first position any row sees
  auto steps = [&](u32 i) {
    const int L = kv.len[i];
    return trust(L) ? cdiv((u32)L, SP) - first((u32)L) / SP : 1u;
  };
  u32 b = 0u, ci = u, nu, slot0 = 0u, C;
  if (kv.n_seq == 1u) {
    const u32 all = steps(0u), c = cdiv(all, a.U);
    C = c < DEC_CMIN / SP ? DEC_CMIN / SP : c;
    nu = cdiv(all, C);
    if (u >= nu) return;
  } else {
    u32 total = 0u;
    for (u32 i = lane; i < kv.n_seq; i += 64u) total += steps(i);
    total = lane_of(wave_scan(total), 63u);
    const u32 c = cdiv(total, a.U);
    C = c < DEC_CMIN / SP ? DEC_CMIN / SP : c;
    // one round of workgroups: the chunks made longer until the units are no more than U
    for (u32 k = 0u; k < 4u && a.fit; k++) {
      u32 all = 0u;
      for (u32 i = lane; i < kv.n_seq; i += 64u) all += cdiv(steps(i), C);
      all = lane_of(wave_scan(all), 63u);
      if (all <= a.U) break;
      C += 1u + (u32)((float)C * (float)(all - a.U) / (float)a.U);
    }
    u32 units = 0u, slots = 0u;
    bool found = false;
    nu = 1u;
    for (u32 i0 = 0u; i0 < kv.n_seq && !found; i0 += 64u) {
      const u32 mine = i0 + lane < kv.n_seq ? cdiv(steps(i0 + lane), C) : 0u;
      const u32 au = wave_scan(mine), as = wave_scan(mine > 1u ? mine : 0u); // units, and partial results (of sequences of several)
      const u64 hit = __ballot(units + au > u);
      if (hit) {
        const u32 f = (u32)__builtin_ctzll(hit);
        b = i0 + f, nu = lane_of(mine, f);
        ci = u - (units + lane_of(au, f) - nu);
        slot0 = slots + lane_of(as, f) - (nu > 1u ? nu : 0u);
        found = true;
      }
      units += lane_of(au, 63u), slots += lane_of(as, 63u);
    }
    if (!found) return;
  }
  nu = (u32)__builtin_amdgcn_readfirstlane((int)nu);

  const u32 r0 = R * cb, nr = T * G - r0 < R ? T * G - r0 : R; // the block's columns
  const u32 nbq = a.n_q * HD / 32u;
  // row r of the block: its query row and head
  auto at = [&](u32 r, u32 &row, u32 &head) {
    const u32 t = (r0 + r) / G;
    row = b * T + t, head = h * G + (r0 + r) - t * G;
  };
  auto put = [&](u32 r, u32 d4, v4f v) {
    u32 row, head;
    at(r, row, head);
    if (a.y) store_y4<BF, F32>(a.y, (u64)row * a.ys + (u64)head * HD + 4u * d4, v, a.vec & 2u);
    if (a.q8) quant_vec4(v, (head * HD + 4u * d4) / 32u, true, a.q8 + (u64)row * a.q8s, nbq);
  };
  const int Ls = __builtin_amdgcn_readfirstlane(kv.len[b]);
  if (!trust(Ls)) { // no part: 0; not to be trusted: NaN
    if (Ls != 0) kv_bad(kv, AMDC_BAD_LEN);
    const float v = Ls != 0 ? __builtin_nanf("") : 0.0f;
    for (u32 i = tid; i < nr * QD; i += NTH) put(i / QD, i % QD, (v4f){v, v, v, v});
    return;
  }
  const u32 L = (u32)Ls;

  // the columns' queries, loaded before the cache (loads complete in order): thread (column, one of 16) holds values
  // 8 c .. 8 c + 7 for c = c0, c0 + 16
  constexpr u32 QE = (16u * R + NTH - 1u) / NTH, QK = HD > 128 ? 2u : 1u;
  float qv[QE][QK][8];
#pragma unroll
  for (u32 e = 0; e < QE; e++) {
    const u32 col = (tid + NTH * e) >> 4, c0 = tid & 15u;
    u32 row, head;
    at(col < nr ? col : nr - 1u, row, head);
#pragma unroll
    for (u32 k = 0; k < QK; k++) {
      const u32 c = c0 + 16u * k;
      load_q8<BF, F32>(a.q, (u64)row * a.qs + (u64)head * HD + 8u * (c < HD / 8u ? c : 0u), a.vec & 1u, qv[e][k]);
    }
  }
  __asm__ volatile("" ::: "memory");

  // the steps of the wave: every NW-th of the chunk's [s0, s1)
  const u32 seen0 = first(L), s0 = seen0 / SP + ci * C, send = cdiv(L, SP), s1 = s0 + C < send ? s0 + C : send;
  const u64 gb = 32ull * HD, hb = gb << (kv.lgp - 4u); // bytes of 16 positions of a head, of a page of a head
  const u32 pmask = (1u << kv.lgp) - 1u;
  const int *table = kv.pages + (u64)b * kv.max_pages;
  u32x4 kr[TT * KS];
  op vr[DT];
  const u32 koff = SP == 32u ? g4 * 256u + (8u * ((n >> 2) & 1u) + (n & 3u)) * 16u : g4 * 256u + n * 16u;
  const u32 voff = SP == 32u ? (g4 & 1u) * (16u * HD) + n * 16u : (g4 >> 1) * (16u * HD) + n * 16u + (g4 & 1u) * 8u;
  int ids = 0; // of the wave's next 64 / TT steps: lane TT i + j holds the page of the j-th 16 positions of step i
  bool bad = false;
  auto get_ids = [&](u32 st) {
    const u32 s = st + NW * (lane / TT), p = SP * s + 16u * (lane % TT);
    // behind the last position that a row sees the last page again, before the first the first: other entries are not looked at
    ids = s < s1 ? table[(p < seen0 ? seen0 : p < L ? p : L - 1u) >> kv.lgp] : 0;
  };
  auto check_ids = [&]() {
    if ((u32)ids >= kv.n_pages) bad = true, ids = 0;
  };
  auto base = [&](u32 st, u32 i, u32 j) {
    const u32 id = lane_of((u32)ids, TT * (i & (64u / TT - 1u)) + j);
    return ((u64)id * kv.n_kv + h) * hb + (((SP * st + 16u * j) & pmask) >> 4) * gb;
  };
  // one round of long chunks: the cache is read once, all of it in the same time, and more than stays in the last-level cache. (The
  // comments in the assembly keep the compiler from making the two branches one, of ordinary loads.)
  const bool nt = a.fit && a.ncb == 1u && C * SP >= DEC_NT / (4u * HD);
  auto load_k = [&](u64 ga, u64 gz) {
    const uint8_t *p = kv.k + (SP == 32u && n & 8u ? gz : ga) + koff;
    auto at = [&](u32 i) { return (const u32x4 *)(p + 64u * (i / KS) + 1024u * (i % KS)); };
    if (nt) {
      __asm__ volatile("; nontemporal");
#pragma unroll
      for (u32 i = 0; i < TT * KS; i++) kr[i] = __builtin_nontemporal_load(at(i));
      __asm__ volatile("; nontemporal");
    } else {
      __asm__ volatile("; cached");
#pragma unroll
      for (u32 i = 0; i < TT * KS; i++) kr[i] = *at(i);
      __asm__ volatile("; cached");
    }
  };
  auto load_v = [&](u64 ga, u64 gz) {
    const uint8_t *p = kv.v + (SP == 32u && g4 & 2u ? gz : ga) + voff;
    if (nt) {
      __asm__ volatile("; nontemporal");
#pragma unroll
      for (int d = 0; d < DT; d++) vr[d] = __builtin_nontemporal_load((const op *)(p + 256 * d));
      __asm__ volatile("; nontemporal");
    } else {
      __asm__ volatile("; cached");
#pragma unroll
      for (int d = 0; d < DT; d++) vr[d] = *(const op *)(p + 256 * d);
      __asm__ volatile("; cached");
    }
  };
  u32 st = s0 + wv;
  u64 ga = 0u, gz = 0u;
  get_ids(st);
  // the queries into the LDS before the cache is asked for (after it, the compiler would wait for both), as the B operand: part p, values 8 c .. 8 c + 7, column
#pragma unroll
  for (u32 e = 0; e < QE; e++) {
    const u32 col = (tid + NTH * e) >> 4, c0 = tid & 15u;
    float big = 0.0f;
#pragma unroll
    for (u32 k = 0; k < QK; k++)
#pragma unroll
      for (int i = 0; i < 8; i++) big = __builtin_fmaxf(big, __builtin_fabsf(qv[e][k][i]));
    float up = 1.0f, down = 1.0f;
    if (F32 && !BF) {
      big = __builtin_fmaxf(big, dpp<0xB1>(big));
      big = __builtin_fmaxf(big, dpp<0x4E>(big));
      big = __builtin_fmaxf(big, dpp<0x141>(big));
      big = __builtin_fmaxf(big, dpp<0x140>(big));
      const u32 ex = __builtin_bit_cast(u32, big) >> 23;
      const u32 k = ex < 11u ? 253u : 264u - ex; // 2^10 / 2^(ex - 127), kept a normal number, as is its inverse
      up = __builtin_bit_cast(float, k << 23), down = __builtin_bit_cast(float, (254u - k) << 23);
    }
    if (col >= R) continue;
    if (c0 == 0u) s_cq[col] = a.c * down;
#pragma unroll
    for (u32 k = 0; k < QK; k++) {
      const u32 c = c0 + 16u * k;
      if (c >= HD / 8u) continue;
      if (F32 && !BF)
#pragma unroll
        for (int i = 0; i < 8; i++) qv[e][k][i] *= up;
      u32 w[NP][4];
      split_n<BF, NP>(qv[e][k], w);
#pragma unroll
      for (int p = 0; p < NP; p++) *(u32x4 *)(sm + ((p * (HD / 8u) + c) * R + col) * 16u) = (u32x4){w[p][0], w[p][1], w[p][2], w[p][3]};
    }
  }
  check_ids();
  if (st < s1) {
    ga = base(st, 0u, 0u), gz = base(st, 0u, TT - 1u);
    load_k(ga, gz), load_v(ga, gz);
  }
  if (tid == 0u) s_bad = 0u;
  v8_barrier(); // not __syncthreads: the first keys and values stay in flight

  // the lane's columns: what they see, and the block's extremes
  const u32 t_a = r0 / G, t_z = (r0 + nr - 1u) / G;
  auto lo_of = [&](u32 t) { const u32 e = L - T + t + 1u; return a.window && e > a.window ? e - a.window : 0u; };
  auto hi_of = [&](u32 t) { return L - T + t + 1u; };
  u32 tc[NC];
  float cq[NC], m[NC], l[NC];
  v4f O[NC][DT];
#pragma unroll
  for (u32 c = 0; c < NC; c++) {
    tc[c] = (r0 + (16u * c + n < nr ? 16u * c + n : nr - 1u)) / G;
    cq[c] = s_cq[16u * c + n], m[c] = NINF, l[c] = 0.0f;
#pragma unroll
    for (int d = 0; d < DT; d++) O[c][d] = (v4f){0.0f, 0.0f, 0.0f, 0.0f};
  }
  const u32 lo_z = lo_of(t_z), hi_a = hi_of(t_a);
  auto mfma_v = [](op v, op p, v4f c) {
    if constexpr (SP == 32u) return mfma16<BF>(v, p, c);
    else if constexpr (BF) return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(s4, v), __builtin_bit_cast(s4, p), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_bit_cast(h4, v), __builtin_bit_cast(h4, p), c, 0, 0, 0);
  };
  for (u32 i = 0u; st < s1; i++, st += NW) {
    v4f S[NC][TT];
#pragma unroll
    for (u32 c = 0; c < NC; c++)
#pragma unroll
      for (u32 t = 0; t < TT; t++) S[c][t] = (v4f){0.0f, 0.0f, 0.0f, 0.0f};
    // heads of 256, or two column tiles: the queries are read from the LDS in every step (kept in registers they would spill others)
#pragma unroll
    for (int s = 0; s < KS; s++) {
      if ((HD > 128 || NC > 1u) && s % 2 == 0) __asm__ volatile("" ::: "memory");
#pragma unroll
      for (u32 c = 0; c < NC; c++)
#pragma unroll
        for (int p = 0; p < NP; p++) {
          const u32x4 qf = *(const u32x4 *)(sm + ((p * (HD / 8u) + 4u * s + g4) * R + 16u * c + n) * 16u);
#pragma unroll
          for (u32 t = 0; t < TT; t++) S[c][t] = mfma16<BF>(kr[t * KS + s], qf, S[c][t]);
        }
    }
    const bool more = st + NW < s1;
    if (more) {
      if ((i & (64u / TT - 1u)) == 64u / TT - 1u) get_ids(st + NW), check_ids();
      ga = base(st + NW, i + 1u, 0u), gz = base(st + NW, i + 1u, TT - 1u);
      load_k(ga, gz);
    }
    const bool edge = SP * st + SP > hi_a || SP * st < lo_z;
    op pw[NC][NP];
#pragma unroll
    for (u32 c = 0; c < NC; c++) {
      float sc[SL], top = NINF;
#pragma unroll
      for (u32 k = 0; k < SL; k++) sc[k] = S[c][k >> 2][k & 3u] * cq[c];
      if (edge) {
        const u32 lo = lo_of(tc[c]), hi = hi_of(tc[c]);
#pragma unroll
        for (u32 k = 0; k < SL; k++) {
          const u32 p = SP * st + SL * g4 + k;
          sc[k] = p >= lo && p < hi ? sc[k] : NINF;
        }
      }
#pragma unroll
      for (u32 k = 0; k < SL; k++) top = __builtin_fmaxf(top, sc[k]);
      if (__ballot(top > m[c] + RAISE)) {
        top = __builtin_fmaxf(top, __shfl_xor(top, 16));
        top = __builtin_fmaxf(top, __shfl_xor(top, 32));
        const float nm = __builtin_fmaxf(m[c], top), f = m[c] == nm ? 1.0f : __builtin_amdgcn_exp2f(m[c] - nm);
#pragma unroll
        for (int d = 0; d < DT; d++) O[c][d] *= f;
        l[c] *= f;
        m[c] = nm;
      }
      const float ref = BIAS - (m[c] == NINF ? 0.0f : m[c]);
#pragma unroll
      for (u32 k = 0; k < SL; k++) sc[k] = __builtin_amdgcn_exp2f(sc[k] + ref);
#pragma unroll
      for (u32 k = 0; k < SL; k += 4u) l[c] += (sc[k] + sc[k + 1u]) + (sc[k + 2u] + sc[k + 3u]); // before a 16-bit type's rounding (pre_body: after it)
      u32 w[NP][SL / 2];
      split_n<BF, NP>(sc, w);
#pragma unroll
      for (int p = 0; p < NP; p++)
#pragma unroll
        for (u32 k = 0; k < SL / 2u; k++) pw[c][p][k] = w[p][k];
    }
    if (!edge) {
#pragma unroll
      for (int d = 0; d < DT; d++)
#pragma unroll
        for (u32 c = 0; c < NC; c++)
#pragma unroll
          for (int p = 0; p < NP; p++) O[c][d] = mfma_v(vr[d], pw[c][p], O[c][d]);
    } else {
#pragma unroll
      for (u32 c = 0; c < NC; c++)
#pragma unroll
        for (int d = 0; d < DT; d++) {
          v4f e = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
          for (int p = 0; p < NP; p++) e = mfma_v(vr[d], pw[c][p], e);
          if (!wave_finite(e)) { // again: without what no column sees (the common case behind the last position), then token by token
            v4f g = {0.0f, 0.0f, 0.0f, 0.0f};
            bool whole = true;
            for (u32 t = t_a;;) {
              e = (v4f){0.0f, 0.0f, 0.0f, 0.0f};
              const op w = seen16(vr[d], SP * st + SL * g4, whole ? lo_of(t_a) : lo_of(t), whole ? hi_of(t_z) : hi_of(t));
#pragma unroll
              for (int p = 0; p < NP; p++) e = mfma_v(w, pw[c][p], e);
              if (whole && wave_finite(e)) {
                g = e;
                break;
              }
              if (!whole) {
                if (tc[c] == t) g = e;
                if (t++ == t_z) break;
              }
              whole = false;
            }
            e = g;
          }
          O[c][d] += e;
        }
    }
    if (more) load_v(ga, gz);
  }
  if (__ballot(bad)) {
    if (lane == 0u) kv_bad(kv, AMDC_BAD_PAGE), s_bad = 1u;
  }
  // the waves' sums brought to one reference and added: NS of them through the LDS (the others' onto the first NS' before)
#pragma unroll
  for (u32 c = 0; c < NC; c++) {
    l[c] += __shfl_xor(l[c], 16);
    l[c] += __shfl_xor(l[c], 32);
    if (g4 == 0u) s_m[wv][16u * c + n] = m[c], s_l[wv][16u * c + n] = l[c];
  }
  __syncthreads(); // and the queries are read, their place is the sums'
  float *so = (float *)sm;
  auto give = [&](u32 to) {
#pragma unroll
    for (u32 c = 0; c < NC; c++)
#pragma unroll
      for (int d = 0; d < DT; d++) *(v4f *)(so + (to * R + 16u * c + n) * OS + 16u * d + 4u * g4) = O[c][d];
  };
#pragma unroll
  for (u32 c = 0; c < NC; c++) {
    float M = s_m[0][16u * c + n];
#pragma unroll
    for (u32 w = 1; w < NW; w++) M = __builtin_fmaxf(M, s_m[w][16u * c + n]);
    const float ref = M == NINF ? 0.0f : M, f = __builtin_amdgcn_exp2f(m[c] - ref);
#pragma unroll
    for (int d = 0; d < DT; d++) O[c][d] *= f;
    if (wv == 0u && g4 == 0u) {
      float sum = 0.0f;
#pragma unroll
      for (u32 w = 0; w < NW; w++) sum += __builtin_amdgcn_exp2f(s_m[w][16u * c + n] - ref) * s_l[w][16u * c + n];
      s_M[16u * c + n] = M, s_L[16u * c + n] = s_bad ? __builtin_nanf("") : sum;
    }
  }
  if (NW > NS) {
    if (wv >= NS) give(wv - NS);
    __syncthreads();
    if (wv < NS)
#pragma unroll
      for (u32 c = 0; c < NC; c++)
#pragma unroll
        for (int d = 0; d < DT; d++) O[c][d] += *(const v4f *)(so + (wv * R + 16u * c + n) * OS + 16u * d + 4u * g4);
  }
  if (wv < NS) give(wv);
  __syncthreads();
  auto mine = [&](u32 i) { // quad i of the workgroup's sums
    const u32 r = i / QD, d4 = i % QD;
    v4f v = *(const v4f *)(so + r * OS + 4u * d4);
#pragma unroll
    for (u32 w = 1; w < NS; w++) v += *(const v4f *)(so + (w * R + r) * OS + 4u * d4);
    return v;
  };
  if (nu == 1u) {
    for (u32 i = tid; i < nr * QD; i += NTH) put(i / QD, i % QD, mine(i) / s_L[i / QD]);
    return;
  }
  // partial results: rmax rows of O, then m and l of R rows
  const u32 rmax = T * G < R ? T * G : R, om = rmax * HD * 4u, sb = om + 8u * R;
  uint8_t *parts = a.ws + AMDC_ATTN_CNT;
  auto slot = [&](u32 k) { return ((u64)(slot0 + k) * kv.n_kv + h) * a.ncb + cb; };
  auto part = [&](u32 k) { return rsrc(parts + slot(k) * sb, sb); };
  {
    const __amdgpu_buffer_rsrc_t d = part(ci);
    for (u32 i = tid; i < nr * QD; i += NTH) __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, mine(i)), d, 16u * i, 0, CPOL_SC1);
    if (tid < nr) {
      __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(u32, s_M[tid]), d, om + 4u * tid, 0, CPOL_SC1);
      __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(u32, s_L[tid]), d, om + 4u * (R + tid), 0, CPOL_SC1);
    }
  }
  u32 k = ci, left = nu, stride = 1u;
  for (u32 level = 0u;; level++) {
    const u32 f0 = k / DEC_FAN * DEC_FAN, cnt = left - f0 < DEC_FAN ? left - f0 : DEC_FAN;
    if (cnt > 1u) {
      __builtin_amdgcn_s_waitcnt(0x0F70); // vmcnt(0): this thread's partial results are stored
      __syncthreads();
      if (tid == 0u) {
        u32 *c = (u32 *)a.ws + slot(f0 * stride + level);
        const bool last = __hip_atomic_fetch_add(c, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) + 1u == cnt;
        if (last) __hip_atomic_store(c, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        s_last = last;
      }
      __syncthreads();
      if (!s_last) return;
      // a thread's first quads of the cnt results, then the weights of every row's results in the LDS (so is free: the
      // results are in the workspace)
      u32x4 v[DEC_FAN];
      auto get = [&](u32 i) {
#pragma unroll
        for (u32 j = 0; j < DEC_FAN; j++) v[j] = __builtin_amdgcn_raw_buffer_load_b128(part((f0 + (j < cnt ? j : 0u)) * stride), 16u * i, 0, CPOL_SC1);
      };
      if (tid < nr * QD) get(tid);
      float *sw = (float *)sm;
      for (u32 e = tid; e < R * DEC_FAN; e += NTH) {
        const u32 r = e % R, j = e / R;
        const uint8_t *d = parts + slot((f0 + (j < cnt ? j : 0u)) * stride) * sb + om + 4u * r;
        const bool in = j < cnt && r < nr;
        sw[e] = in ? __hip_atomic_load((const float *)d, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : NINF;
        sw[R * DEC_FAN + e] = in ? __hip_atomic_load((const float *)(d + 4u * R), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : 0.0f;
      }
      __syncthreads();
      if (tid < R) {
        float M = NINF, sum = 0.0f;
#pragma unroll
        for (u32 j = 0; j < DEC_FAN; j++) M = __builtin_fmaxf(M, sw[R * j + tid]);
#pragma unroll
        for (u32 j = 0; j < DEC_FAN; j++) {
          const float f = __builtin_amdgcn_exp2f(sw[R * j + tid] - (M == NINF ? 0.0f : M));
          sw[R * j + tid] = f, sum += f * sw[R * (DEC_FAN + j) + tid];
        }
        s_M[tid] = M, s_L[tid] = sum;
      }
      __syncthreads();
      const bool final = left <= DEC_FAN;
      const __amdgpu_buffer_rsrc_t to = part(f0 * stride);
      for (u32 i = tid; i < nr * QD; i += NTH) {
        if (i != tid) get(i);
        v4f sum = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (u32 j = 0; j < DEC_FAN; j++)
          if (j < cnt) sum += sw[R * j + i / QD] * __builtin_bit_cast(v4f, v[j]);
        if (final) put(i / QD, i % QD, sum / s_L[i / QD]);
        else __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, sum), to, 16u * i, 0, CPOL_SC1);
      }
      if (final) return;
      if (tid < nr) {
        __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(u32, s_M[tid]), to, om + 4u * tid, 0, CPOL_SC1);
        __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(u32, s_L[tid]), to, om + 4u * (R + tid), 0, CPOL_SC1);
      }
    }
    k /= DEC_FAN, left = cdiv(left, DEC_FAN), stride *= DEC_FAN;
  }
}

#define DEC_KERNEL(HD, KN, TAG, BF, F32, NC) \
  extern "C" __global__ __launch_bounds__(64u * AMDC_DEC_NW, 2) void amdc_attn_dec_h##HD##_##KN##TAG(amdc_kv_dev kv, amdc_attn_args a) { dec_body<HD, BF, F32, NC, AMDC_DEC_NW>(kv, a); }
#define DEC_KERNELS(HD, TAG, NC) \
  DEC_KERNEL(HD, f16, TAG, false, false, NC) DEC_KERNEL(HD, f16_f32, TAG, false, true, NC) DEC_KERNEL(HD, bf16, TAG, true, false, NC) DEC_KERNEL(HD, bf16_f32, TAG, true, true, NC)
DEC_KERNELS(64, , 1u)
DEC_KERNELS(128, , 1u)
DEC_KERNELS(256, , 1u)
DEC_KERNELS(64, _n2, 2u)
DEC_KERNELS(128, _n2, 2u)
#undef DEC_KERNELS
#undef DEC_KERNEL

// ------------------------------------------------------------------ attention of prompts

// c and the two 16-bit values of w
template <bool BF>
__device__ __forceinline__ float sum2(u32 w, float c) {
  typedef _Float16 h2 __attribute__((ext_vector_type(2)));
  if constexpr (BF) return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(b2, w), __builtin_bit_cast(b2, 0x3F803F80u), c, false);
  else return __builtin_amdgcn_fdot2(__builtin_bit_cast(h2, w), __builtin_bit_cast(h2, 0x3C003C00u), c, false);
}

template <bool BF>
__device__ __forceinline__ v16f mfma32(u32x4 a, u32x4 b, v16f c) {
  typedef _Float16 h8 __attribute__((ext_vector_type(8)));
  if constexpr (BF) return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
}

// lds_load16 with a scalar offset too: one lane offset for every piece of a tile
__device__ __forceinline__ void lds_load16s(__amdgpu_buffer_rsrc_t rs, __attribute__((address_space(3))) void *d, u32 voff, u32 soff) {
  const u32 m = __builtin_amdgcn_readfirstlane((u32)(__UINTPTR_TYPE__)d);
  __asm__ volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" ::"s"(m), "v"(voff), "s"(rs), "s"(soff) : "memory");
}

#define PRE_SB(hd) ((AMDC_PRE_BM * (hd) + 2u * AMDC_PRE_BM) * 4u) // bytes of a partial result

// The rows of a unit (a tile of AMDC_PRE_BM rows of a sequence) and the tiles of BN positions [j0, j1) that they see, in ns parts
struct PreUnit {
  SeqRows s;
  u32 b, r0, nr, j0, j1, ns;
};
__device__ __forceinline__ PreUnit pre_unit(const amdc_kv_dev &kv, const amdc_attn_args &a, u32 unit, u32 BN) {
  PreUnit p;
  u32 ti;
  if (a.cu) {
    auto base = [&](u32 i) { const int c = a.cu[i]; return (c < 0 ? 0u : (u32)c * a.G / AMDC_PRE_BM) + i; };
    p.b = find_seq(kv.n_seq, unit, base);
    ti = unit - base(p.b);
  } else {
    const u32 per = cdiv(a.T * a.G, AMDC_PRE_BM);
    p.b = unit / per, ti = unit - p.b * per;
  }
  p.s = seq_rows(kv, a.cu, a.T, p.b);
  p.s.row0 = uniform(p.s.row0), p.s.m = uniform(p.s.m), p.s.len = uniform(p.s.len);
  const u32 R = p.s.m * a.G;
  p.r0 = ti * AMDC_PRE_BM;
  p.nr = p.r0 >= R ? 0u : R - p.r0 < AMDC_PRE_BM ? R - p.r0 : AMDC_PRE_BM;
  if (!p.nr || !p.s.len) return p;
  const u32 m0 = p.s.len - p.s.m, e = m0 + p.r0 / a.G + 1u;
  p.j0 = (a.window && e > a.window ? e - a.window : 0u) / BN, p.j1 = cdiv(m0 + (p.r0 + p.nr - 1u) / a.G + 1u, BN);
  const u32 most = (p.j1 - p.j0) / AMDC_PRE_MINTILES;
  p.ns = most < 1u ? 1u : most < a.U ? most : a.U;
  return p;
}

// The new tokens of a sequence and the G heads that share a key / value head are its rows (token t, head g: t G + g). A workgroup
// takes AMDC_PRE_BM consecutive rows, its waves W = 32 or 16 each, and goes through tiles of BN positions that the LDS holds twice: while the
// waves work on one tile the next is loaded into the other half, straight from the cache (the layout is the one the LDS wants; every
// load moves 1 KB, and every read of an operand, 16 bytes a lane, meets no bank twice).
// The matrix work bounds it (4 hd flops to a row and position), and next to it the exponentials:
//   S^T = K Q^T   (32x32x16; columns are query rows): row r of a group of 32 positions is position
//                 16 (r / 16) + 8 (r / 4 % 2) + 4 (r / 8 % 2) + r % 4, so that the lane's registers 8 s .. 8 s + 7 are the positions
//                 16 s + 8 (lane / 32) .. + 7 of its row; W = 16 is dec_body's arrangement (16x16x32)
//   O^T = V^T P^T: and so, as 16-bit weights, the B operand of step s; a value's eight positions are the A operand.
// A row's maximum and sum are in the two (four) lanes that hold its scores: no reduction over the wave. W = 32 reads each operand
// from the LDS for twice as many rows; W = 16 needs half the registers for O and the queries. Parts in f32, the raised maximum, the
// factor 2^8 and the steps at the edges are dec_body's.
// Rows are dealt from the last tile of the last sequence down: the longest first. Where all rows make fewer workgroups than the CUs
// hold (a short chunk of a long prompt), a tile's positions are split over a.U workgroups; their partial results go through the
// workspace and amdc_attn_join_*, a launch of its own (joined by the last workgroup to arrive, 128 rows of four parts took it 18 us).
// Measured on MI355X (replayed; cards differ by 5 %): 12000 rows of 32 / 8 heads of 128, bf16, 1.11 ms, 1066 TFLOP/s of causal work (a
// large product: 1210), matrix units busy 56 % of the cycles, vector units 44 %, at 1.7 to 1.9 GHz; 11 prompts under a window, heads of
// 64, f16, 71 us, 540 TFLOP/s, matrix units 30 %, vector units 61 %: a tile's scores, softmax and products follow each other in a wave, and
// the two kinds of units run one after the other more than beside each other; a chunk of 256 over 5000, 24 / 4 heads of 256, f32, 77 to 80
// us with its join of 11 (profiled); 77 rows, 32 / 32 heads of 128 12.4 us, latency. 2 x 4096 rows, 32 / 8 heads of 128: 286 bf16, 501 f32 on
// f16, 709 f32 on bf16; 2 x 2048 rows, 24 / 4 heads of 256: 145, 217, 264.
template <int HD, bool BF, bool F32, u32 W, u32 BN>
__device__ __forceinline__ void pre_body(const amdc_kv_dev &kv, const amdc_attn_args &a) {
  typedef typename std::conditional<W == 32u, v16f, v4f>::type acc; // of a matrix instruction: W x W / 64
  constexpr int NP = F32 ? (BF ? 3 : 2) : 1, NA = W == 32u ? 16 : 4, DT = HD / W;
  constexpr u32 TT = W == 32u ? 1u : 2u, KS = HD / (W == 32u ? 16u : 32u), PF = W / 16u; // of 32 positions: score tiles, steps over hd, weight operands
  constexpr u32 NW = AMDC_PRE_BM / W, NTH = 64u * NW, MT = BN / 32u, TB = BN * HD * 2u, QD = HD / 4u;
  // the keys' groups of 16 positions in the LDS: W = 16 reads two at once, 16 banks apart
  constexpr u32 GS = 32u * HD + (W == 16u ? 64u : 0u), KB = BN / 16u * GS;
  constexpr u32 PG = HD / 16u, PW = BN / 16u * PG / NW; // KB of a group of 16 positions (keys, then values), and of a tile for each wave
  constexpr float BIAS = BF ? 0.0f : 8.0f, RAISE = 6.0f, NINF = -__builtin_inff();
  constexpr bool FULL = HD > 128 && NP > 2; // of registers: the queries' last part stays in the LDS
  constexpr int QR = FULL ? NP - 1 : NP;
  __shared__ u32x4 s_q[FULL ? KS : 1][FULL ? NTH : 1]; // step, thread
  __shared__ __attribute__((aligned(16))) uint8_t sm[2][KB + TB]; // half: keys, values
  __shared__ u32 s_bad;
  const u32 tid = threadIdx.x, lane = tid & 63u, wv = (u32)__builtin_amdgcn_readfirstlane((int)(tid >> 6)), n = lane & (W - 1u), gg = lane / W;
  auto zero = []() {
    acc z;
#pragma unroll
    for (int i = 0; i < NA; i++) z[i] = 0.0f;
    return z;
  };
  auto mfma = [](u32x4 x, u32x4 y, acc c) {
    if constexpr (W == 32u) return mfma32<BF>(x, y, c);
    else return mfma16<BF>(x, y, c);
  };
  auto over = [](float v, auto f) { // f over the lanes of a row
    if (W == 16u) v = f(v, __shfl_xor(v, 16));
    return f(v, __shfl_xor(v, 32));
  };
  auto maxf = [](float x, float y) { return __builtin_fmaxf(x, y); };
  auto addf = [](float x, float y) { return x + y; };
  const u32 G = a.G, h = blockIdx.x % kv.n_kv;
  u32 x = blockIdx.x / kv.n_kv;
  const u32 sp = x % a.U, unit = a.ncb - 1u - x / a.U;
  // rows that go past T: no unit need belong to the sequence (one that begins at T has none). The last workgroup's rows are the shortest.
  if (a.cu && blockIdx.x == gridDim.x - 1u && (u32)a.cu[kv.n_seq] > a.T) kv_bad(kv, AMDC_BAD_ROWS);
  const PreUnit pu = pre_unit(kv, a, unit, BN);
  const SeqRows &s = pu.s;
  const u32 r0 = pu.r0, nr = pu.nr, nbq = a.n_q * HD / 32u;
  if (!nr) return;
  auto at = [&](u32 r, u32 &row, u32 &head) { // row r of the workgroup
    const u32 t = (r0 + r) / G;
    row = s.row0 + t, head = h * G + (r0 + r) - t * G;
  };
  auto put = [&](u32 r, u32 d4, v4f v) {
    u32 row, head;
    at(r, row, head);
    if (a.y) store_y4<BF, F32>(a.y, (u64)row * a.ys + (u64)head * HD + 4u * d4, v, a.vec & 2u);
    if (a.q8) quant_vec4(v, (head * HD + 4u * d4) / 32u, true, a.q8 + (u64)row * a.q8s, nbq);
  };
  if (!s.len) { // no part: 0; not to be trusted: NaN
    const float v = s.bad ? __builtin_nanf("") : 0.0f;
    if (sp == 0u)
      for (u32 i = tid; i < nr * QD; i += NTH) put(i / QD, i % QD, (v4f){v, v, v, v});
    return;
  }
  const u32 L = s.len, m0 = L - s.m;
  auto lo_of = [&](u32 t) { const u32 e = m0 + t + 1u; return a.window && e > a.window ? e - a.window : 0u; };
  auto hi_of = [&](u32 t) { return m0 + t + 1u; };

  // the tiles of positions [jb, je) of this workgroup
  const u32 ns = pu.ns;
  if (sp >= ns) return;
  const u32 jb = pu.j0 + amdc_part_at(pu.j1 - pu.j0, sp, ns), je = pu.j0 + amdc_part_at(pu.j1 - pu.j0, sp + 1u, ns);

  // the wave's rows and the lane's
  const u32 w0 = W * wv, wr = nr > w0 ? (nr - w0 < W ? nr - w0 : W) : 0u; // 0: only loads
  const u32 rc = wr ? w0 + (n < wr ? n : wr - 1u) : 0u;
  const u32 tc = (r0 + rc) / G, t_a = (u32)__builtin_amdgcn_readfirstlane((int)((r0 + (wr ? w0 : 0u)) / G)),
            t_z = (u32)__builtin_amdgcn_readfirstlane((int)((r0 + (wr ? w0 + wr - 1u : 0u)) / G));
  const u32 lo = lo_of(tc), hi = hi_of(tc), lo_a = lo_of(t_a), lo_z = lo_of(t_z), hi_a = hi_of(t_a), hi_z = hi_of(t_z);

  // loads: wave wv moves the pieces wv PW .. of a tile, all of one group of positions
  const u32 grp = wv * PW / PG, pc0 = wv * PW % PG;
  constexpr u32 GB = 32u * HD; // bytes of a group: a power of two
  const u32 pmask = (1u << kv.lgp) - 1u;
  const int *table = kv.pages + (u64)pu.b * kv.max_pages;
  u32 at16 = 0u; // where in the pools, in groups, the wave's group of tiles jt .. jt + 63 is (a lane each)
  bool bad = false;
  const u32 seen0 = lo_of(r0 / G) & ~15u;
  auto get_ids = [&](u32 jt) {
    // behind the last tile that one again, behind the sequence's last group of positions that one, before the first that a row sees that
    const u32 j = jt + lane < je ? jt + lane : je - 1u, f = BN * j + 16u * grp, e = (L - 1u) & ~15u, p = f < seen0 ? seen0 : f < e ? f : e;
    u32 id = (u32)table[p >> kv.lgp];
    if (id >= kv.n_pages) bad = true, id = 0u;
    at16 = ((id * kv.n_kv + h) << (kv.lgp - 4u)) + ((p & pmask) >> 4);
  };
  auto issue = [&](u32 j, u32 half) {
    if (((j - jb) & 63u) == 0u) get_ids(j);
    const u64 off = (u64)lane_of(at16, (j - jb) & 63u) * GB;
#pragma unroll
    for (u32 i = 0; i < PW; i++) {
      const u32 c = pc0 + i;
      const bool val = c >= PG / 2u;
      const u32 o = 1024u * (val ? c - PG / 2u : c);
      lds_load16s(rsrc((val ? kv.v : kv.k) + off, GB), (__attribute__((address_space(3))) void *)(sm[half] + (val ? KB + grp * GB : grp * GS) + o), 16u * lane, o);
    }
  };
  if (tid == 0u) s_bad = 0u;
  issue(jb, 0u);

  // the lane's query row: values HD / KS k + 8 gg .. + 7 of step k
  u32x4 qf[QR][KS];
  float cq = __builtin_fabsf(a.c); // a negative scale's sign goes to the queries: the largest product is the largest score
  {
    u32 row, head;
    at(rc, row, head);
    const u64 i0 = (u64)row * a.qs + (u64)head * HD + 8u * gg;
    float up = a.c < 0.0f ? -1.0f : 1.0f, v[KS][8];
#pragma unroll
    for (u32 k = 0; k < KS; k++) load_q8<BF, F32>(a.q, i0 + HD / KS * k, a.vec & 1u, v[k]);
    if (F32 && !BF) {
      float big = 0.0f;
#pragma unroll
      for (u32 k = 0; k < KS; k++)
#pragma unroll
        for (int i = 0; i < 8; i++) big = __builtin_fmaxf(big, __builtin_fabsf(v[k][i]));
      big = over(big, maxf);
      const u32 e = __builtin_bit_cast(u32, big) >> 23, k = e < 11u ? 253u : 264u - e;
      up *= __builtin_bit_cast(float, k << 23), cq *= __builtin_bit_cast(float, (254u - k) << 23);
    }
    cq = cq < 0x1p-149f ? 0x1p-149f : cq; // scale 0: a score of 0 (2^-21 at most), also of -infinity (what is not seen) not NaN; a NaN stays one
#pragma unroll
    for (u32 k = 0; k < KS; k++) {
#pragma unroll
      for (int i = 0; i < 8; i++) v[k][i] *= up;
      u32x4 w[NP];
      split8<BF, NP>(v[k], w);
#pragma unroll
      for (int p = 0; p < QR; p++) qf[p][k] = w[p];
      if (FULL) s_q[k][tid] = w[NP - 1]; // read by this thread alone
    }
  }

  acc O[DT];
#pragma unroll
  for (int d = 0; d < DT; d++) O[d] = zero();
  float m = NINF, l = 0.0f;
  const u32 koff = (W == 32u ? (n >> 4) * GS + (8u * ((n >> 2) & 1u) + 4u * ((n >> 3) & 1u) + (n & 3u)) * 16u
                             : (n >> 3) * GS + (8u * ((n >> 2) & 1u) + (n & 3u)) * 16u) + gg * 256u,
            voff = (gg * HD + n) * 16u;
  // N groups of 32 positions from p0 on, keys at kt and values at vt in the LDS; EDGE: not every row sees all of them
  auto tile = [&](auto edge, auto groups, const uint8_t *kt, const uint8_t *vt, u32 p0) __attribute__((always_inline)) {
    constexpr bool EDGE = decltype(edge)::value;
    constexpr u32 N = decltype(groups)::value, NS = 8u * PF; // scores of a lane in 32 positions: 32 / PF f + 8 gg + 0 .. 7 for f < PF
    float S[N * NS];
    // these products before the other wave's softmax, which then runs beside them (MI355X, us: 2 x 4096 rows of 32 / 8 heads of 128 303,
    // without 308, both products so 307; of heads of 64 173, the softmax raised in their place 179)
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (u32 t = 0; t < N; t++) {
      acc c[TT];
#pragma unroll
      for (u32 u = 0; u < TT; u++) c[u] = zero();
#pragma unroll
      for (u32 k = 0; k < KS; k++) {
        if (FULL && k % 2u == 0u) __asm__ volatile("" ::: "memory"); // few operands at a time: the registers are full
#pragma unroll
        for (u32 u = 0; u < TT; u++) {
          const u32x4 kf = *(const u32x4 *)(kt + t * 2u * GS + 32u * HD / KS * k + 64u * u);
#pragma unroll
          for (int p = 0; p < QR; p++) c[u] = mfma(kf, qf[p][k], c[u]);
          if (FULL) c[u] = mfma(kf, s_q[k][tid], c[u]);
        }
      }
#pragma unroll
      for (u32 i = 0; i < NS; i++) S[NS * t + i] = c[i / NA][i % NA];
    }
    __builtin_amdgcn_s_setprio(0);
    float top = NINF;
#pragma unroll
    for (u32 i = 0; i < N * NS; i++) {
      if (EDGE) {
        const u32 p = p0 + 32u * (i / NS) + 32u / PF * (i % NS / 8u) + 8u * gg + (i & 7u);
        S[i] = p >= lo && p < hi ? S[i] : NINF;
      }
      top = __builtin_fmaxf(top, S[i]);
    }
    if (__ballot(top * cq > m + RAISE)) {
      const float nm = __builtin_fmaxf(m, over(top, maxf) * cq), f = m == nm ? 1.0f : __builtin_amdgcn_exp2f(m - nm);
#pragma unroll
      for (int d = 0; d < DT; d++) O[d] *= f;
      l *= f;
      m = nm;
    }
    const float ref = BIAS - (m == NINF ? 0.0f : m);
    u32x4 pw[NP][PF * N];
#pragma unroll
    for (u32 k = 0; k < PF * N; k++) {
      float v[8];
#pragma unroll
      for (u32 i = 0; i < 8u; i++) v[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(S[8u * k + i], cq, ref));
      if (NP > 1) l += ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
      u32x4 w[NP];
      split8<BF, NP>(v, w);
#pragma unroll
      for (int p = 0; p < NP; p++) pw[p][k] = w[p];
      // 16-bit: the sum of the rounded weights, the ones that the values get, two in an instruction (dec_body, which waits for the HBM, sums
      // them before: either is within the weights' half steps, and the two operators' rows differ by that)
      if (NP == 1)
#pragma unroll
        for (int i = 0; i < 4; i++) l = sum2<BF>(w[0][i], l);
    }
    auto finite = [&](const acc &e) {
      float z = 0.0f;
#pragma unroll
      for (int i = 0; i < NA; i++) z += e[i] - e[i]; // NaN where one is not
      return __ballot(!(z == 0.0f)) == 0ull;
    };
    u32 redo = 0u;
    __asm__ volatile("" : "+v"(l)); // summed here: the compiler would keep the weights for it until after the products
#pragma unroll
    for (int d = 0; d < DT; d++) {
      if (FULL && d % 4 == 0) __asm__ volatile("" ::: "memory");
      acc e = EDGE ? zero() : O[d];
#pragma unroll
      for (u32 k = 0; k < PF * N; k++) {
        const u32x4 vf = *(const u32x4 *)(vt + 64u * HD / PF * k + 16u * W * d);
#pragma unroll
        for (int p = 0; p < NP; p++) e = mfma(vf, pw[p][k], e);
      }
      if (!EDGE) O[d] = e;
      else if (finite(e)) O[d] += e;
      else redo |= 1u << d;
    }
    if (EDGE)
      while (redo) { // the d-th W values again: without what no row sees (the common case behind the last position), then row by row
        const u32 d = (u32)__builtin_ctz(redo);
        redo &= redo - 1u;
        acc g = zero();
        bool whole = true;
        for (u32 t = t_a;;) {
          acc e = zero();
#pragma unroll
          for (u32 k = 0; k < PF * N; k++) {
            const u32x4 vf = seen16(*(const u32x4 *)(vt + 64u * HD / PF * k + 16u * W * d), p0 + 32u / PF * k + 8u * gg, whole ? lo_a : lo_of(t), whole ? hi_z : hi_of(t));
#pragma unroll
            for (int p = 0; p < NP; p++) e = mfma(vf, pw[p][k], e);
          }
          if (whole && finite(e)) {
            g = e;
            break;
          }
          if (!whole) {
            if (tc == t) g = e;
            if (t++ == t_z) break;
          }
          whole = false;
        }
#pragma unroll
        for (int i = 0; i < DT; i++)
          if (d == (u32)i) O[i] += g;
      }
  };
  auto step = [&](u32 j) { // to tile j
    vm_wait(0u);  // it has landed ...
    v8_barrier(); // ... every wave's part, and every wave is done with the other half
    if (j + 1u < je) issue(j + 1u, ((j - jb) & 1u) ^ 1u);
  };
  // every wave goes through all tiles, those that all of its rows see entirely, j0 .. j1 - 1, in a loop of their own (in one loop with the
  // others the compiler copies O to other registers and back in every tile)
  const u32 f0 = wr ? cdiv(lo_z, BN) : je, f1 = wr ? hi_a / BN : je;
  for (u32 j = jb; j < je;) {
    for (; j >= f0 && j < f1 && j < je; j++) {
      step(j);
      const uint8_t *at = sm[(j - jb) & 1u];
      tile(std::false_type(), std::integral_constant<u32, MT>(), at + koff, at + KB + voff, BN * j);
    }
    if (j >= je) break;
    step(j);
    const uint8_t *at = sm[(j - jb) & 1u];
    const u32 p0 = BN * j++;
    if (!wr) continue;
    for (u32 t = 0; t < MT; t++) // an edge, 32 positions at a time
      if (p0 + 32u * t < hi_z && p0 + 32u * t + 32u > lo_a)
        tile(std::true_type(), std::integral_constant<u32, 1u>(), at + koff + t * 2u * GS, at + KB + voff + t * 64u * HD, p0 + 32u * t);
  }
  l = over(l, addf);
  if (__ballot(bad) && lane == 0u) kv_bad(kv, AMDC_BAD_PAGE), s_bad = 1u;
  __syncthreads();
  if (s_bad) l = __builtin_nanf("");

  auto quad = [&](int d, u32 i) { return (v4f){O[d][4 * i], O[d][4 * i + 1], O[d][4 * i + 2], O[d][4 * i + 3]}; }; // values W d + 8 i + 4 gg .. + 3
  if (ns == 1u) {
    u32 row, head, rr = rc;
    __asm__ volatile("" : "+v"(rr)); // where the row is computed again, not kept in registers since the queries
    at(rr, row, head);
    const float inv = 1.0f / l;
#pragma unroll
    for (int d = 0; d < DT; d++) {
      O[d] *= inv;
      if (a.y && n < wr)
#pragma unroll
        for (u32 i = 0; i < NA / 4u; i++) store_y4<BF, F32>(a.y, (u64)row * a.ys + (u64)head * HD + W * d + 8u * i + 4u * gg, quad(d, i), a.vec & 2u);
    }
    if (a.q8)
#pragma unroll
      for (int blk = 0; blk < HD / 32; blk++) { // amdc_quant_q8's d, q and sum of a block, spread over the lanes of the row
        constexpr int BT = 32 / W;
        float big = __builtin_fabsf(O[blk * BT][0]); // not 0: of values that are all NaN, d is NaN
#pragma unroll
        for (int i = 1; i < BT * NA; i++) big = __builtin_fmaxf(big, __builtin_fabsf(O[blk * BT + i / NA][i % NA]));
        const float dd = over(big, maxf) / 127.0f;
        u32 sum = 0u, w[BT * NA / 4];
#pragma unroll
        for (int i = 0; i < BT * NA / 4; i++) {
          int qi[4];
          q8_round4(quad(blk * BT + 4 * i / NA, i % (NA / 4)), dd, qi);
          sum += (u32)qi[0] + (u32)qi[1] + (u32)qi[2] + (u32)qi[3];
          w[i] = (u32)(qi[0] & 255) | (u32)(qi[1] & 255) << 8 | (u32)(qi[2] & 255) << 16 | (u32)qi[3] << 24;
        }
        if (W == 16u) sum += (u32)__shfl_xor((int)sum, 16);
        sum += (u32)__shfl_xor((int)sum, 32);
        if (n < wr) {
          uint8_t *to = a.q8 + (u64)row * a.q8s;
          const u32 at_blk = head * (HD / 32) + blk;
#pragma unroll
          for (u32 i = 0; i < BT * NA / 4; i++) *(u32 *)(to + 32u * at_blk + W * (4u * i / NA) + 8u * (i % (NA / 4)) + 4u * gg) = w[i];
          if (gg == 0u) ((float *)(to + 32u * nbq))[at_blk] = dd, ((u32 *)(to + 36u * nbq))[at_blk] = sum;
        }
      }
    return;
  }
  // a partial result: AMDC_PRE_BM rows of O, then their m and l
  float *part = (float *)(a.ws + AMDC_ATTN_CNT + (((u64)unit * kv.n_kv + h) * a.U + sp) * PRE_SB(HD));
  if (n < wr) {
#pragma unroll
    for (int d = 0; d < DT; d++)
#pragma unroll
      for (u32 i = 0; i < NA / 4u; i++) *(v4f *)(part + (w0 + n) * HD + W * d + 8u * i + 4u * gg) = quad(d, i);
    if (gg == 0u) part[AMDC_PRE_BM * HD + w0 + n] = m, part[AMDC_PRE_BM * (HD + 1u) + w0 + n] = l;
  }
}

// The parts of a split tile joined in the order of their positions: 16 of its rows, JOIN_N parts' loads in flight a thread
#define JOIN_N 8u
template <bool BF, bool F32>
__device__ __forceinline__ void join_body(const amdc_kv_dev &kv, const amdc_attn_args &a, u32 hd, u32 BN) {
  __shared__ float s_w[AMDC_PRE_MAXPARTS][16], s_l[AMDC_PRE_MAXPARTS][16], s_L[16]; // of every part and row: m, then its weight; l
  const u32 tid = threadIdx.x, qd = hd / 4u, nbq = a.n_q * hd / 32u;
  const u32 h = blockIdx.x % kv.n_kv, x = blockIdx.x / kv.n_kv, unit = x / (AMDC_PRE_BM / 16u), f = x % (AMDC_PRE_BM / 16u) * 16u;
  const PreUnit pu = pre_unit(kv, a, unit, BN);
  if (f >= pu.nr || !pu.s.len || pu.ns == 1u) return; // nothing to join: the rows are written
  const u32 nr = pu.nr - f < 16u ? pu.nr - f : 16u, ns = pu.ns, pf = PRE_SB(hd) / 4u; // floats of a partial result
  const float *parts = (const float *)(a.ws + AMDC_ATTN_CNT) + ((u64)unit * kv.n_kv + h) * a.U * pf, *ml = parts + AMDC_PRE_BM * hd + f;
  for (u32 e = tid; e < 16u * ns; e += 256u) {
    const u32 r = e & 15u, k = e >> 4;
    const float *p = ml + (u64)k * pf + (r < nr ? r : 0u);
    s_w[k][r] = p[0], s_l[k][r] = p[AMDC_PRE_BM];
  }
  __syncthreads();
  if (tid < 16u) {
    float M = -__builtin_inff(), sum = 0.0f;
    for (u32 k = 0u; k < ns; k++) M = __builtin_fmaxf(M, s_w[k][tid]);
    const float ref = M == -__builtin_inff() ? 0.0f : M;
    for (u32 k = 0u; k < ns; k++) {
      const float w = __builtin_amdgcn_exp2f(s_w[k][tid] - ref);
      s_w[k][tid] = w, sum += w * s_l[k][tid];
    }
    s_L[tid] = sum;
  }
  __syncthreads();
  v4f v[4]; // quads tid, tid + 256, .. of the 16 rows: at most 4
#pragma unroll
  for (u32 i = 0; i < 4u; i++) v[i] = (v4f){0.0f, 0.0f, 0.0f, 0.0f};
  for (u32 k0 = 0u; k0 < ns; k0 += JOIN_N) {
#pragma unroll
    for (u32 i = 0; i < 4u; i++) {
      const u32 e = tid + 256u * i;
      if (e >= nr * qd) break;
      v4f w[JOIN_N];
#pragma unroll
      for (u32 k = 0; k < JOIN_N; k++) w[k] = *(const v4f *)(parts + (u64)(k0 + k < ns ? k0 + k : k0) * pf + f * hd + 4u * e);
#pragma unroll
      for (u32 k = 0; k < JOIN_N; k++)
        if (k0 + k < ns) v[i] += s_w[k0 + k][e / qd] * w[k];
    }
  }
#pragma unroll
  for (u32 i = 0; i < 4u; i++) {
    const u32 e = tid + 256u * i;
    if (e >= nr * qd) break;
    const u32 r = e / qd, d4 = e - r * qd, t = (pu.r0 + f + r) / a.G, row = pu.s.row0 + t, head = h * a.G + (pu.r0 + f + r) - t * a.G;
    const v4f y = v[i] / s_L[r];
    if (a.y) store_y4<BF, F32>(a.y, (u64)row * a.ys + (u64)head * hd + 4u * d4, y, a.vec & 2u);
    if (a.q8) quant_vec4(y, (head * hd + 4u * d4) / 32u, true, a.q8 + (u64)row * a.q8s, nbq);
  }
}
extern "C" __global__ __launch_bounds__(256) void amdc_attn_join_f32(amdc_kv_dev kv, amdc_attn_args a, u32 hd, u32 bn) { join_body<false, true>(kv, a, hd, bn); }
extern "C" __global__ __launch_bounds__(256) void amdc_attn_join_f16(amdc_kv_dev kv, amdc_attn_args a, u32 hd, u32 bn) { join_body<false, false>(kv, a, hd, bn); }
extern "C" __global__ __launch_bounds__(256) void amdc_attn_join_bf16(amdc_kv_dev kv, amdc_attn_args a, u32 hd, u32 bn) { join_body<true, false>(kv, a, hd, bn); }

// Rows of a wave, positions of a tile, workgroups a CU wanted of the registers (MI355X, us; each pair as measured when it was chosen).
// Heads of 128, 16-bit: two workgroups on tiles of 64 positions; three, on tiles of 32, spill (12000 rows 1084 against 1098, 4096 rows 306
// against 301). Heads of 128, f32 on f16: two on tiles of 32 505 for 2 x 4096 rows, one on tiles of 64 587; bf16's three parts would spill.
// Heads of 256: 32 rows a wave, one wave a SIMD, 144 where 16 rows, two waves, took 110 (256 rows over 5000 positions, 24 / 4 heads, f32; 77 now).
// Heads of 64, 16-bit: three workgroups a CU 76 for 11 prompts under a window, two 81; four spill, as f32's three do.
#define PRE_KERNEL(HD, KN, BF, F32, OCC) \
  extern "C" __global__ __launch_bounds__(64u * AMDC_PRE_BM / AMDC_PRE_W(HD), OCC) void amdc_attn_pre_h##HD##_##KN(amdc_kv_dev kv, amdc_attn_args a) { \
    pre_body<HD, BF, F32, AMDC_PRE_W(HD), AMDC_PRE_BN(HD, BF, F32)>(kv, a); \
  }
PRE_KERNEL(64, f16, false, false, 3)
PRE_KERNEL(64, f16_f32, false, true, 2)
PRE_KERNEL(64, bf16, true, false, 3)
PRE_KERNEL(64, bf16_f32, true, true, 2)
PRE_KERNEL(128, f16, false, false, 2)
PRE_KERNEL(128, f16_f32, false, true, 2)
PRE_KERNEL(128, bf16, true, false, 2)
PRE_KERNEL(128, bf16_f32, true, true, 1)
PRE_KERNEL(256, f16, false, false, 2)
PRE_KERNEL(256, f16_f32, false, true, 2)
PRE_KERNEL(256, bf16, true, false, 2)
PRE_KERNEL(256, bf16_f32, true, true, 2)
#undef PRE_KERNEL
