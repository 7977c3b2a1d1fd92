// amdc_attn.h -- the device code of the paged cache and the attention over it (amdc_kv of amdc_q4.h describes the
// layout); part of amdc_kernels.hip's translation unit.
//
//   amdc_kv_append_{f16,bf16}   rotation, keys and values into the cache, rotated queries

// ------------------------------------------------------------------ helpers

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
    u32 r;
    __asm__("v_cvt_pk_bf16_f32 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
    return r;
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

struct AppendArgs {
  const float *k, *v, *q;
  void *qo;
  const int *cu;
  const float *freq;
  u32 qt, n_q, T, ks, vs, qs, qos, n_rot, rope, lghd, rows, gq, gv, upb, vec;
};

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

// Workgroups 0 .. rows gq - 1: queries and keys, gq of them to a row. The row's n_rot / 2 angles once, into the LDS, then
// eight values a thread: a key's eight are 16 bytes of the cache. Where the pairs are halves apart a thread reads the
// other eight as well (from the L1) instead of trading them.
// The others: values, gv workgroups to a group of eight positions of a sequence, aligned as the cache is (for ragged
// rows, cu[b] / 8 + 2 b is a first group of b's that leaves room for its floor(m / 8) + 2 at most). A thread reads one
// value of up to eight rows and stores them as 16 bytes, or where the group is not full the new ones alone.
template <bool BF>
__device__ __forceinline__ void append_body(const amdc_kv_dev &kv, const AppendArgs &a) {
  __shared__ float s_cos[128], s_sin[128];
  const u32 hd = 1u << a.lghd, tid = threadIdx.x, nrw = a.rows * a.gq;
  const u64 gb = 32ull << a.lghd, lgg = kv.lgp - 4u; // bytes of 16 positions of a head, log2 of such groups in a page
  if (blockIdx.x < nrw) {
    const u32 row = blockIdx.x / a.gq, part = blockIdx.x - row * a.gq;
    const u32 b = a.cu ? find_seq(kv.n_seq, row, [&](u32 i) { const int c = a.cu[i]; return c < 0 ? 0u : (u32)c; }) : row / a.T;
    const SeqRows s = seq_rows(kv, a.cu, a.T, b);
    if (!s.len || row < s.row0 || row - s.row0 >= s.m) return;
    const u32 pos = s.len - s.m + (row - s.row0);
    const int id = kv.pages[(u64)b * kv.max_pages + (pos >> kv.lgp)];
    const bool ok = (u32)id < kv.n_pages;
    if (!ok) kv_bad(kv, AMDC_BAD_PAGE);
    const u32 half = a.n_rot >> 1;
    if (a.rope) {
      if (tid < half) sincos64((double)pos * (double)a.freq[tid], s_sin[tid], s_cos[tid]);
      __syncthreads();
    }
    const u32 nq = a.q ? a.n_q : 0u, nh = nq + kv.n_kv, hpi = 2048u >> a.lghd;
    const u32 slot = pos & ((1u << kv.lgp) - 1u), c = tid & ((hd >> 3) - 1u);
    for (u32 h0 = part * hpi; h0 < nh; h0 += a.gq * hpi) {
      const u32 h = h0 + (tid >> (a.lghd - 3u));
      const bool on = h < nh;
      float x[8];
      if (on) {
        const float *src = h < nq ? a.q + (u64)row * a.qs + (u64)h * hd : a.k + (u64)row * a.ks + (u64)(h - nq) * hd;
        load8(src + 8u * c, a.vec & (h < nq ? 1u : 2u), x);
        if (a.rope == 1u) { // pairs
#pragma unroll
          for (u32 i = 0; i < 8u; i += 2u) {
            const u32 e = 8u * c + i;
            if (e < a.n_rot) {
              const float cs = s_cos[e >> 1], sn = s_sin[e >> 1], u = x[i], w = x[i + 1u];
              x[i] = u * cs - w * sn, x[i + 1u] = u * sn + w * cs;
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
              const float cs = s_cos[f], sn = s_sin[f];
              x[i] = e < half ? x[i] * cs - o[i] * sn : o[i] * sn + x[i] * cs;
            }
          }
        }
      }
      if (a.q == (const float *)a.qo) __syncthreads(); // queries in place: every read of these heads before the first write
      if (!on) continue;
      if (h >= nq) {
        if (!ok) continue;
        const u32x4 w = {pack2<BF>(x[0], x[1]), pack2<BF>(x[2], x[3]), pack2<BF>(x[4], x[5]), pack2<BF>(x[6], x[7])};
        *(u32x4 *)(kv.k + (((((u64)(u32)id * kv.n_kv + (h - nq)) << lgg) + (slot >> 4)) * gb + 256u * c + 16u * (slot & 15u))) = w;
      } else if (a.qt == 0u) {
        float *d = (float *)a.qo + (u64)row * a.qos + (u64)h * hd + 8u * c;
        if (a.vec & 4u) ((v4f *)d)[0] = (v4f){x[0], x[1], x[2], x[3]}, ((v4f *)d)[1] = (v4f){x[4], x[5], x[6], x[7]};
        else
#pragma unroll
          for (int i = 0; i < 8; i++) d[i] = x[i];
      } else {
        const u32x4 w = {pack2<BF>(x[0], x[1]), pack2<BF>(x[2], x[3]), pack2<BF>(x[4], x[5]), pack2<BF>(x[6], x[7])};
        unsigned short *d = (unsigned short *)a.qo + (u64)row * a.qos + (u64)h * hd + 8u * c;
        if (a.vec & 4u) *(u32x4 *)d = w;
        else
#pragma unroll
          for (int i = 0; i < 8; i++) d[i] = (unsigned short)(w[i >> 1] >> (16 * (i & 1)));
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
  for (u32 i = part * 256u + tid; i < n; i += a.gv * 256u) {
    const u32 h = i >> a.lghd, d = i & (hd - 1u);
    float x[8];
#pragma unroll
    for (u32 j = 0; j < 8u; j++) x[j] = j >= j0 && j < j1 ? src[(u64)(j - j0) * a.vs + i] : 0.0f;
    const u32x4 w = {pack2<BF>(x[0], x[1]), pack2<BF>(x[2], x[3]), pack2<BF>(x[4], x[5]), pack2<BF>(x[6], x[7])};
    uint8_t *to = kv.v + (((((u64)(u32)id * kv.n_kv + h) << (lgg + 1u)) + g) * (gb >> 1) + 16u * d);
    if (j1 - j0 == 8u) *(u32x4 *)to = w;
    else
#pragma unroll
      for (u32 j = 0; j < 8u; j++)
        if (j >= j0 && j < j1) ((unsigned short *)to)[j] = (unsigned short)(w[j >> 1] >> (16u * (j & 1u)));
  }
}

#define APPEND_KERNEL(KN, BF) \
  extern "C" __global__ __launch_bounds__(256) void amdc_kv_append_##KN(amdc_kv_dev kv, AppendArgs a) { append_body<BF>(kv, a); }
APPEND_KERNEL(f16, false)
APPEND_KERNEL(bf16, true)
#undef APPEND_KERNEL
