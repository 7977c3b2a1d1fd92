// amdc_gdn.h -- the device code of a linear-attention layer (amdc_slots and amdc_gdn of amdc_q4.h): the short convolution,
// the gated delta rule, and the norms around them; part of amdc_kernels.hip's translation unit.
//
//   amdc_conv_w{2,3,4}_{f32,f16,bf16}   the causal convolution over the channels, with its state
//   amdc_gdn_rec_h{64,128}_{f32,f16,bf16}
//                                       the delta rule, token after token
//   amdc_norm_gate_{f32,f16,bf16}       the heads' norm times the gate, and the Q8 copy
//   amdc_norm_res_{1,2,4,8}             norm, residual, norm, and the Q8 copy

// ------------------------------------------------------------------ helpers

// a value of a row of type TY (AMDC_TYPE_*), and four side by side (vec: aligned to four values)
template <int TY>
__device__ __forceinline__ float ld1(const void *p, u64 i) {
  if constexpr (TY == 0) return ((const float *)p)[i];
  else if constexpr (TY == 1) return h2f(((const unsigned short *)p)[i]);
  else return __builtin_bit_cast(float, (u32)((const unsigned short *)p)[i] << 16);
}
template <int TY>
__device__ __forceinline__ v4f ld4(const void *p, u64 i, bool vec) {
  if (!vec) return (v4f){ld1<TY>(p, i), ld1<TY>(p, i + 1u), ld1<TY>(p, i + 2u), ld1<TY>(p, i + 3u)};
  if constexpr (TY == 0) return *(const v4f *)((const float *)p + i);
  else {
    const u32x2 u = *(const u32x2 *)((const unsigned short *)p + i);
    return (v4f){lo16<TY == 2>(u.x), hi16<TY == 2>(u.x), lo16<TY == 2>(u.y), hi16<TY == 2>(u.y)};
  }
}
// the first n (1 to 4) of them
template <int TY>
__device__ __forceinline__ void st4(void *p, u64 i, v4f v, bool vec, u32 n = 4u) {
  if constexpr (TY == 0) {
    if (vec) *(v4f *)((float *)p + i) = v;
    else
#pragma unroll
      for (u32 e = 0; e < 4u; e++)
        if (e < n) ((float *)p)[i + e] = v[e];
  } else {
    const u32x2 u = {pack2<TY == 2>(v.x, v.y), pack2<TY == 2>(v.z, v.w)};
    if (vec) *(u32x2 *)((unsigned short *)p + i) = u;
    else
#pragma unroll
      for (u32 e = 0; e < 4u; e++)
        if (e < n) ((unsigned short *)p)[i + e] = (unsigned short)(u[e >> 1] >> (16u * (e & 1u)));
  }
}

__device__ __forceinline__ v4f splat(float x) { return (v4f){x, x, x, x}; }
__device__ __forceinline__ v4f fma4(v4f a, v4f b, v4f c) {
  return (v4f){__builtin_fmaf(a.x, b.x, c.x), __builtin_fmaf(a.y, b.y, c.y), __builtin_fmaf(a.z, b.z, c.z), __builtin_fmaf(a.w, b.w, c.w)};
}
__device__ __forceinline__ float nan_() { return __builtin_nanf(""); }

__device__ __forceinline__ void slot_bad(const amdc_slots_dev &sl, u32 why) { __hip_atomic_store(sl.bad, why, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }

// The new rows of sequence b: the first one and their number (0: none, or, after the flag is set, rows outside 0 .. T).
__device__ __forceinline__ u32 slot_rows(const amdc_slots_dev &sl, u32 b, u32 &row0) {
  row0 = b * sl.T;
  if (!sl.cu) return sl.T;
  const int c0 = sl.cu[b], c1 = sl.cu[b + 1u];
  if (c0 < 0 || c1 < c0 || (u32)c1 > sl.T) {
    slot_bad(sl, AMDC_BAD_ROWS);
    return 0u;
  }
  row0 = (u32)c0;
  return (u32)(c1 - c0);
}
// Whether a slot is to be read or written: -1 is none, any other outside the pool is reported (bad).
__device__ __forceinline__ bool slot_ok(const amdc_slots_dev &sl, int s, bool &bad) {
  bad = s < -1 || (s >= 0 && (u32)s >= sl.n_slots);
  if (bad) slot_bad(sl, AMDC_BAD_SLOT);
  return !bad && s >= 0;
}

// 1 / (1 + exp(-v)) with the hardware's exp2 and reciprocal: off by (3 + |v|) 2^-23 of itself; 0 where it is under 2^-126 (v under
// -87.3).
__device__ __forceinline__ float sigmoid_fast(float v) { return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(v * -1.4426950408889634f)); }

// ------------------------------------------------------------------ the short convolution

// Reading and writing bound it. A thread has four channels of up to AMDC_CONV_ROWS rows of a sequence: the window of the last W - 1
// inputs stays in its registers, the next eight rows are in flight while it goes over them, and a row is read again only by the unit
// behind it (W - 1 of 32). The unit of a sequence's first rows reads the state and, after that, writes it: from x where the sequence has rows enough, and
// else from what it has read, so that a slot may be read and written by the same call.
template <u32 W, int TY>
__device__ __forceinline__ void conv_body(const amdc_slots_dev &sl, const amdc_conv_args &a) {
  const u32 ct = blockIdx.x % a.cb, u = blockIdx.x / a.cb, c = 4u * (ct * blockDim.x + threadIdx.x);
  u32 b, first;
  if (sl.cu) {
    const auto base = [&](u32 i) { const int s = sl.cu[i]; return (s < 0 ? 0u : (u32)s) / AMDC_CONV_ROWS + i; };
    b = find_seq(sl.n_seq, u, base), first = base(b);
    if (first > u) return;
  } else b = u / a.upb, first = b * a.upb;
  u32 row0;
  const u32 m = slot_rows(sl, b, row0), t0 = (u - first) * AMDC_CONV_ROWS;
  if (t0 >= m) return;
  const u32 n = c >= a.ch ? 0u : a.ch - c < 4u ? a.ch - c : 4u, t1 = m - t0 < AMDC_CONV_ROWS ? m : t0 + AMDC_CONV_ROWS;
  if (!n) return;
  const bool vec = a.vec & 1u, vecy = a.vec & 2u;
  const auto row = [&](const float *p, u64 i) { // n values of a row
    v4f v = splat(0.0f);
    if (vec) v = *(const v4f *)(p + i);
    else
#pragma unroll
      for (u32 e = 0; e < 4u; e++)
        if (e < n) v[e] = p[i + e];
    return v;
  };
  const float *x = a.x + c + (u64)row0 * a.xs;
  v4f w[W], bias = splat(0.0f), win[W - 1u];
#pragma unroll
  for (u32 e = 0; e < 4u; e++) {
    const u32 ce = c + (e < n ? e : 0u);
#pragma unroll
    for (u32 j = 0; j < W; j++) w[j][e] = a.w[(u64)ce * W + j];
    if (a.bias) bias[e] = a.bias[ce];
  }
  if (t0 == 0u) {
    const int f = sl.from[b];
    bool bad;
    const bool have = slot_ok(sl, f, bad);
#pragma unroll
    for (u32 j = 0; j < W - 1u; j++) win[j] = have ? row(a.state, ((u64)(u32)f * (W - 1u) + j) * a.ch + c) : splat(bad ? nan_() : 0.0f);
    if (!sl.each) {
      const int o = sl.to[b];
      bool worse;
      if (slot_ok(sl, o, worse) && !bad) {
        v4f s[W - 1u]; // all of it, before the first is written
#pragma unroll
        for (u32 j = 0; j < W - 1u; j++) {
          const u32 at = m + j; // of the W - 1 old inputs and the m new ones, those from m on
          v4f old = win[W - 2u];
#pragma unroll
          for (u32 i = 0; i + 1u < W; i++) old = at == i ? win[i] : old;
          s[j] = at < W - 1u ? old : row(x, (u64)(at - (W - 1u)) * a.xs);
        }
#pragma unroll
        for (u32 j = 0; j < W - 1u; j++) st4<0>(a.state, ((u64)(u32)o * (W - 1u) + j) * a.ch + c, s[j], vec, n);
      }
    }
  } else {
#pragma unroll
    for (u32 j = 0; j < W - 1u; j++) win[j] = row(x, (u64)(t0 + j - (W - 1u)) * a.xs);
  }
  const bool keep = sl.each;
  constexpr u32 F = 8u; // rows in flight
  v4f in[F];
#pragma unroll
  for (u32 i = 0; i < F; i++) in[i] = row(x, (u64)(t0 + i < t1 ? t0 + i : t1 - 1u) * a.xs);
  for (u32 t = t0; t < t1; t += F) {
#pragma unroll
    for (u32 i = 0; i < F; i++) {
      if (t + i < t1) {
        const v4f now = in[i];
        in[i] = row(x, (u64)(t + i + F < t1 ? t + i + F : t1 - 1u) * a.xs);
        v4f s = bias;
#pragma unroll
        for (u32 j = 0; j < W - 1u; j++) s = fma4(w[j], win[j], s);
        s = fma4(w[W - 1u], now, s);
#pragma unroll
        for (u32 j = 0; j + 2u < W; j++) win[j] = win[j + 1u];
        win[W - 2u] = now;
        if (a.act)
#pragma unroll
          for (u32 e = 0; e < 4u; e++) s[e] *= sigmoid_fast(s[e]);
        st4<TY>(a.y, (u64)(row0 + t + i) * a.ys + c, s, vecy, n);
        if (keep) {
          const int o = sl.to[row0 + t + i];
          bool bad;
          if (slot_ok(sl, o, bad) && !(sl.from[b] < -1 || (sl.from[b] >= 0 && (u32)sl.from[b] >= sl.n_slots)))
#pragma unroll
            for (u32 j = 0; j < W - 1u; j++) st4<0>(a.state, ((u64)(u32)o * (W - 1u) + j) * a.ch + c, win[j], vec, n);
        }
      }
    }
  }
}

#define CONV(W, N, TY)                                                                                                             \
  extern "C" __global__ __launch_bounds__(256) void amdc_conv_w##W##_##N(const amdc_slots_dev sl, const amdc_conv_args a) { conv_body<W##u, TY>(sl, a); }
#define CONVS(W) CONV(W, f32, 0) CONV(W, f16, 1) CONV(W, bf16, 2)
CONVS(2) CONVS(3) CONVS(4)

// ------------------------------------------------------------------ the gated delta rule, token after token

// log decay (at most 0, NaN kept) and rate of value head h at a row
__device__ __forceinline__ void gdn_gates(const amdc_gdn_args &g, u64 row, u32 h, float &decay, float &rate) {
  const float x = g.a[row * g.as + h] + g.dt[h];
  const float v = g.A[h] * ((x > 0.0f ? x : 0.0f) + log1pf(__builtin_expf(-__builtin_fabsf(x))));
  decay = v > 0.0f ? 0.0f : v;
  rate = 1.0f / (1.0f + __builtin_expf(-g.b[row * g.bs + h]));
}
__device__ __forceinline__ u32 gdn_key_head(const amdc_gdn_args &g, u32 h) { return g.tiled ? h % g.n_k : h / g.G; }
__device__ __forceinline__ float lane_of(float v, u32 l) { return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), (int)l)); }

// The sum of v over the 16 lanes that have the same lane & 3: rotations by 8 and 4 in rows of 16 lanes, then the rows
__device__ __forceinline__ float sum16(float v) {
  v += dpp<0x128>(v);
  v += dpp<0x124>(v);
  auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(u32, v), __builtin_bit_cast(u32, v), false, false);
  u32 x = r[0], y = r[1];
  v = __builtin_bit_cast(float, x) + __builtin_bit_cast(float, y);
  r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(u32, v), __builtin_bit_cast(u32, v), false, false);
  x = r[0], y = r[1];
  return __builtin_bit_cast(float, x) + __builtin_bit_cast(float, y);
}

// The state's columns do not touch each other, so a wave has 16 of a head's (8 KB at dk = 128, contiguous in the pool) and
// goes through the sequence's tokens alone, without the LDS and without a barrier: lane l has the rows 16 i + l / 4 of the columns 4 (l % 4) .. + 3.
// With k and q of norm 1 (their factors rk, rq) and the state as it is before the token's decay e,
//   u = rate (v - e rk k S),  S' = e S + rk k^T u,  y = rq q S' = rq (e q S + rk (q.k) u),
// so that k S, q S, k.k, q.q and k.q go through one reduction a token. Reading and writing the states bounds it for batches; a single
// sequence waits for two dependent loads (its slot, the state).
template <int TY, u32 DK>
__device__ __forceinline__ void gdn_rec_body(const amdc_slots_dev &sl, const amdc_gdn_args &g) {
  constexpr u32 NI = DK / 16u;
  const u32 lane = threadIdx.x & 63u, ng = g.dv >> 4, w = uniform(4u * blockIdx.x + (threadIdx.x >> 6));
  if (w >= sl.n_seq * g.n_v * ng) return;
  const u32 b = w / (g.n_v * ng), hw = w - b * g.n_v * ng, h = hw / ng, c = 16u * (hw - h * ng), hk = gdn_key_head(g, h);
  const u32 r = lane >> 2, c4 = lane & 3u;
  u32 row0;
  const u32 m = uniform(slot_rows(sl, b, row0));
  if (!m) return;
  const int f = sl.from[b];
  bool bad;
  const bool have = slot_ok(sl, f, bad);
  const u64 mat = (u64)DK * g.dv, part = (u64)h * mat + (u64)c * DK + 16u * r + 4u * c4;
  v4f S[NI];
#pragma unroll
  for (u32 i = 0; i < NI; i++) S[i] = have ? *(const v4f *)(g.s + (u64)(u32)f * g.n_v * mat + part + 256u * i) : splat(bad ? nan_() : 0.0f);
  float k[NI], q[NI];
  v4f v;
  const auto load = [&](u32 t) {
    const u64 row = row0 + t;
#pragma unroll
    for (u32 i = 0; i < NI; i++) k[i] = ld1<TY>(g.k, row * g.ks + hk * DK + 16u * i + r), q[i] = ld1<TY>(g.q, row * g.qs + hk * DK + 16u * i + r);
    v = ld4<TY>(g.v, row * g.vs + h * g.dv + c + 4u * c4, g.vec & 1u);
  };
  load(0u);
  float decay = 0.0f, rate = 0.0f;
  for (u32 t = 0; t < m; t++) {
    if (!(t & 63u)) gdn_gates(g, row0 + (t + lane < m ? t + lane : m - 1u), h, decay, rate), decay = __builtin_expf(decay); // those of 64 tokens
    const float e = lane_of(decay, t & 63u), be = lane_of(rate, t & 63u);
    float kk = 0.0f, qq = 0.0f, kq = 0.0f;
    v4f kS = splat(0.0f), qS = splat(0.0f), vt = v;
    float kt[NI];
#pragma unroll
    for (u32 i = 0; i < NI; i++) {
      kt[i] = k[i];
      kk = __builtin_fmaf(k[i], k[i], kk), qq = __builtin_fmaf(q[i], q[i], qq), kq = __builtin_fmaf(k[i], q[i], kq);
      kS = fma4(splat(k[i]), S[i], kS), qS = fma4(splat(q[i]), S[i], qS);
    }
    if (t + 1u < m) load(t + 1u);
    kk = sum16(kk), qq = sum16(qq), kq = sum16(kq);
#pragma unroll
    for (u32 j = 0; j < 4u; j++) kS[j] = sum16(kS[j]), qS[j] = sum16(qS[j]);
    const float rk = 1.0f / __builtin_sqrtf(kk + g.eps), rq = g.scale / __builtin_sqrtf(qq + g.eps);
    v4f u, y;
#pragma unroll
    for (u32 j = 0; j < 4u; j++) {
      u[j] = be * __builtin_fmaf(-(e * rk), kS[j], vt[j]);
      y[j] = rq * __builtin_fmaf(kq * rk, u[j], e * qS[j]);
      u[j] *= rk;
    }
    if (r == 0u) st4<TY>(g.y, (u64)(row0 + t) * g.ys + h * g.dv + c + 4u * c4, y, g.vec & 2u);
#pragma unroll
    for (u32 i = 0; i < NI; i++) S[i] = fma4(splat(kt[i]), u, S[i] * e);
    if (sl.each || t + 1u == m) {
      const int o = sl.to[sl.each ? row0 + t : b];
      bool worse;
      if (slot_ok(sl, o, worse) && !bad)
#pragma unroll
        for (u32 i = 0; i < NI; i++) *(v4f *)(g.s + (u64)(u32)o * g.n_v * mat + part + 256u * i) = S[i];
    }
  }
}

#define GDN_REC(H, N, TY)                                                                                                            \
  extern "C" __global__ __launch_bounds__(256) void amdc_gdn_rec_h##H##_##N(const amdc_slots_dev sl, const amdc_gdn_args g) { gdn_rec_body<TY, H##u>(sl, g); }
#define GDN_RECS(H) GDN_REC(H, f32, 0) GDN_REC(H, f16, 1) GDN_REC(H, bf16, 2)
GDN_RECS(64) GDN_RECS(128)

// ------------------------------------------------------------------ the norms

// y = x s w gate(z), s = 1 / sqrt(sum x^2 / hd + eps) over a head, and its Q8 copy. Reading and writing bound it. Four values a lane, hd / 4 lanes a
// head. Grid (ceil(n / 1024), T).
template <int TY>
__device__ __forceinline__ void norm_gate_body(const amdc_norm_args &a) {
  const u32 i0 = 4u * (blockIdx.x * NT + threadIdx.x), n = a.n;
  const bool on = i0 < n; // whole heads, and whole blocks of 32, at once
  const u32 i = on ? i0 : n - 4u;
  const v4f x = ld4<TY>((const uint8_t *)a.x + (u64)blockIdx.y * a.xs, i, a.vec & 1u), z = ld4<0>((const uint8_t *)a.z + (u64)blockIdx.y * a.zs, i, a.vec & 2u);
  const v4f w = ld4<0>(a.w, i & (a.hd - 1u), a.vec & 4u);
  const float ss = seg_sum((x.x * x.x + x.y * x.y) + (x.z * x.z + x.w * x.w), a.hd >> 2);
  const float s = 1.0f / __builtin_sqrtf(ss / (float)a.hd + a.eps);
  v4f y;
#pragma unroll
  for (u32 j = 0; j < 4u; j++) {
    const float g = sigmoid_fast(z[j]);
    y[j] = x[j] * s * w[j] * (a.gate ? g : z[j] * g);
  }
  if (on && a.y) st4<0>((uint8_t *)a.y + (u64)blockIdx.y * a.ys, i, y, a.vec & 8u);
  if (a.q) quant_vec4(y, i >> 5, on, a.q + (u64)blockIdx.y * a.qs, n >> 5);
}
extern "C" __global__ __launch_bounds__(256) void amdc_norm_gate_f32(const amdc_norm_args a) { norm_gate_body<0>(a); }
extern "C" __global__ __launch_bounds__(256) void amdc_norm_gate_f16(const amdc_norm_args a) { norm_gate_body<1>(a); }
extern "C" __global__ __launch_bounds__(256) void amdc_norm_gate_bf16(const amdc_norm_args a) { norm_gate_body<2>(a); }

// 1 / sqrt(mean square + eps) of a row that the workgroup's threads have NV fours each of
template <u32 NV>
__device__ __forceinline__ float row_scale(const v4f (&x)[NV], float rn, float eps, float *part) {
  float ss = 0.0f;
#pragma unroll
  for (u32 j = 0; j < NV; j++) ss += (x[j].x * x[j].x + x[j].y * x[j].y) + (x[j].z * x[j].z + x[j].w * x[j].w);
  ss = seg_sum(ss, 64u);
  const u32 nw = blockDim.x >> 6;
  if (nw > 1u) {
    if ((threadIdx.x & 63u) == 0u) part[threadIdx.x >> 6] = ss;
    __syncthreads();
    ss = seg_sum((threadIdx.x & 15u) < nw ? part[threadIdx.x & 15u] : 0.0f, 16u);
  }
  return 1.0f / __builtin_sqrtf(ss * rn + eps);
}

// h = res + scale (x s1 w1, or x itself), y = h s2 w2 and its Q8 copy: a row to a workgroup, which keeps it in its registers between the two
// norms. h may be res: a thread reads and writes the same places. Grid (1, T).
template <u32 NV>
__device__ __forceinline__ void norm_res_body(const amdc_norm_args &a) {
  __shared__ float part[2][16];
  const u32 n = a.n, step = 4u * blockDim.x;
  const float rn = 1.0f / (float)n;
  const uint8_t *px = (const uint8_t *)a.x + (u64)blockIdx.y * a.xs, *pr = (const uint8_t *)a.z + (u64)blockIdx.y * a.zs;
  v4f x[NV], h[NV];
#pragma unroll
  for (u32 j = 0; j < NV; j++) {
    const u32 i = 4u * threadIdx.x + j * step;
    x[j] = i < n ? ld4<0>(px, i, a.vec & 1u) : splat(0.0f), h[j] = i < n ? ld4<0>(pr, i, a.vec & 2u) : splat(0.0f);
  }
  const float s1 = a.w ? row_scale<NV>(x, rn, a.eps, part[0]) : 1.0f;
#pragma unroll
  for (u32 j = 0; j < NV; j++) {
    const u32 i = 4u * threadIdx.x + j * step;
    if (i < n) {
      if (a.w) x[j] = x[j] * s1 * ld4<0>(a.w, i, a.vec & 4u);
      h[j] = fma4(splat(a.scale), x[j], h[j]);
      st4<0>((uint8_t *)a.h + (u64)blockIdx.y * a.hs, i, h[j], a.vec & 16u);
    }
  }
  const float s2 = row_scale<NV>(h, rn, a.eps, part[1]);
#pragma unroll
  for (u32 j = 0; j < NV; j++) {
    const u32 i = 4u * threadIdx.x + j * step;
    const bool on = i < n;
    const v4f y = h[j] * s2 * ld4<0>(a.w2, on ? i : 0u, a.vec & 32u);
    if (on && a.y) st4<0>((uint8_t *)a.y + (u64)blockIdx.y * a.ys, i, y, a.vec & 8u);
    if (a.q) quant_vec4(y, (on ? i : 0u) >> 5, on, a.q + (u64)blockIdx.y * a.qs, n >> 5);
  }
}
#define NORM_RES(NV, LIM)                                                                                                              \
  extern "C" __global__ __launch_bounds__(LIM) void amdc_norm_res_##NV(const amdc_norm_args a) { norm_res_body<NV##u>(a); }
NORM_RES(1, 1024) NORM_RES(2, 1024) NORM_RES(4, 1024) NORM_RES(8, 1024)
