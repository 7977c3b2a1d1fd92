// amdc_gdn.h -- the device code of a linear-attention layer (amdc_slots and amdc_gdn of amdc_q4.h): the short convolution,
// the gated delta rule, and the norms around them; part of amdc_kernels.hip's translation unit.
//
//   amdc_conv_w{2,3,4}_{f32,f16,bf16}[_odd]
//                                       the causal convolution over the channels, with its state
//   amdc_gdn_rec_h{64,128}_{f32,f16,bf16}
//                                       the delta rule, token after token
//   amdc_gdn_prep_h{64,128}_{f32,f16,bf16}, amdc_gdn_scan_h{64,128}_{f32,f16,bf16,f16_odd,bf16_odd}
//                                       the delta rule in chunks of 64 tokens: what does not depend on the state, then the states
//   amdc_norm_gate_{f32,f16,bf16}       the heads' norm times the gate, and the Q8 copy
//   amdc_norm_res_{1,2,4,8}             norm, residual, norm, and the Q8 copy

// ------------------------------------------------------------------ helpers

// A value of a row of type TY (AMDC_TYPE_*), and four side by side, aligned to one: the memory takes them at any
// address, and a branch on the alignment would keep the loads behind it from being in flight together.
typedef float f4_any __attribute__((ext_vector_type(4), aligned(4)));
typedef unsigned short u4_any __attribute__((ext_vector_type(4), aligned(2)));
template <int TY>
__device__ __forceinline__ float ld1(const void *p, u64 i) {
  if constexpr (TY == 0) return ((const float *)p)[i];
  else if constexpr (TY == 1) return h2f(((const unsigned short *)p)[i]);
  else return __builtin_bit_cast(float, (u32)((const unsigned short *)p)[i] << 16);
}
template <int TY>
__device__ __forceinline__ v4f ld4(const void *p, u64 i) {
  if constexpr (TY == 0) {
    const f4_any v = *(const f4_any *)((const float *)p + i);
    return (v4f){v.x, v.y, v.z, v.w};
  } else {
    const u4_any u = *(const u4_any *)((const unsigned short *)p + i);
    return TY == 1 ? (v4f){h2f(u.x), h2f(u.y), h2f(u.z), h2f(u.w)}
                   : (v4f){__builtin_bit_cast(float, (u32)u.x << 16), __builtin_bit_cast(float, (u32)u.y << 16), __builtin_bit_cast(float, (u32)u.z << 16),
                           __builtin_bit_cast(float, (u32)u.w << 16)};
  }
}
template <int TY>
__device__ __forceinline__ void st4(void *p, u64 i, v4f v) {
  if constexpr (TY == 0) *(f4_any *)((float *)p + i) = (f4_any){v.x, v.y, v.z, v.w};
  else {
    const u32 a = pack2<TY == 2>(v.x, v.y), b = pack2<TY == 2>(v.z, v.w);
    *(u4_any *)((unsigned short *)p + i) = (u4_any){(unsigned short)a, (unsigned short)(a >> 16), (unsigned short)b, (unsigned short)(b >> 16)};
  }
}
// C (4 or 1) of them: the others are 0
template <int TY, u32 C>
__device__ __forceinline__ v4f ldc(const void *p, u64 i) {
  if constexpr (C == 4u) return ld4<TY>(p, i);
  else return (v4f){ld1<TY>(p, i), 0.0f, 0.0f, 0.0f};
}
template <int TY, u32 C>
__device__ __forceinline__ void stc(void *p, u64 i, v4f v) {
  if constexpr (C == 4u) st4<TY>(p, i, v);
  else if constexpr (TY == 0) ((float *)p)[i] = v.x;
  else ((unsigned short *)p)[i] = (unsigned short)pack2<TY == 2>(v.x, 0.0f);
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
// Sequence i's rows, for the report alone: where cu decreases, the searches below may come upon no row of a sequence that is at fault. `part`: 0
// for one workgroup of each i.
__device__ __forceinline__ void check_rows(const amdc_slots_dev &sl, u32 i, u32 part) {
  u32 row0;
  if (part == 0u && i < sl.n_seq) slot_rows(sl, i, row0);
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

// Reading and writing bound it. A thread has four channels (one, where their number is no multiple of four: _odd) of a unit of up to
// AMDC_CONV_ROWS rows of a sequence, which are all in flight at once, with the W - 1 inputs before them. The unit of a sequence's first
// rows reads the state and, after that, writes it: the window behind its rows, or from x where the sequence has more, so that a
// slot may be read and written by the same call; with `each` one unit has all rows of a sequence, eight after eight, for the same
// reason. Workgroups of one wave. 8192 channels, 9 prompts of 1100 tokens, into bf16: units of 8 rows 85 us (5.7 TB/s), of 4 90 us, of 32 with 8
// rows in flight 105 us; 256 threads 87 us; units that follow each other on one XCD 87 us (the rows that two units read come from
// the last-level cache). One token of 10240 channels: 2.8 us.
template <u32 W, int TY, u32 C>
__device__ __forceinline__ void conv_body(const amdc_slots_dev &sl, const amdc_conv_args &a) {
  const u32 ct = blockIdx.x % a.cb, u = blockIdx.x / a.cb, c = C * (ct * blockDim.x + threadIdx.x);
  u32 b, first;
  if (sl.cu) {
    check_rows(sl, u, ct); // a unit for each sequence at least
    const auto base = [&](u32 i) { const int s = sl.cu[i]; return (s < 0 ? 0u : (u32)s) / AMDC_CONV_ROWS + i; };
    b = find_seq(sl.n_seq, u, base), first = base(b);
    if (first > u) return;
  } else b = u / a.upb, first = b * a.upb;
  u32 row0;
  const u32 m = slot_rows(sl, b, row0), t0 = (u - first) * AMDC_CONV_ROWS;
  if (t0 >= m) return;
  const bool keep = sl.each;
  const u32 t1 = keep || m - t0 < AMDC_CONV_ROWS ? m : t0 + AMDC_CONV_ROWS;
  if (c >= a.ch) return;
  const auto row = [](const float *p, u64 i) { return ldc<0, C>(p, i); };
  const float *x = a.x + c + (u64)row0 * a.xs;
  const bool first_rows = t0 == 0u;
  v4f w[W], bias = splat(0.0f), win[W - 1u], in[AMDC_CONV_ROWS];
  const auto rows = [&](u32 t) {
#pragma unroll
    for (u32 i = 0; i < AMDC_CONV_ROWS; i++) in[i] = row(x, (u64)(t + i < t1 ? t + i : t1 - 1u) * a.xs);
  };
  const int f = sl.from[b], o = sl.to[keep ? row0 : b]; // no branch around them: all these loads are in flight together
  rows(t0);
#pragma unroll
  for (u32 j = 0; j < W; j++) w[j] = splat(0.0f);
#pragma unroll
  for (u32 e = 0; e < C; e++)
#pragma unroll
    for (u32 j = 0; j < W; j++) w[j][e] = a.w[(u64)(c + e) * W + j];
  if (a.bias) bias = row(a.bias, c);
  bool bad;
  const bool have = slot_ok(sl, f, bad);
  if (bad) bias = splat(nan_()); // all rows, also those that see nothing of the state
  if (first_rows) {
#pragma unroll
    for (u32 j = 0; j < W - 1u; j++) win[j] = splat(0.0f);
    if (have)
#pragma unroll
      for (u32 j = 0; j < W - 1u; j++) win[j] = row(a.state, ((u64)(u32)f * (W - 1u) + j) * a.ch + c);
  } else {
#pragma unroll
    for (u32 j = 0; j < W - 1u; j++) win[j] = row(x, (u64)(t0 + j - (W - 1u)) * a.xs);
  }
  const auto put_state = [&](int slot) { // the window
    bool worse;
    if (slot_ok(sl, slot, worse) && !bad)
#pragma unroll
      for (u32 j = 0; j < W - 1u; j++) stc<0, C>(a.state, ((u64)(u32)slot * (W - 1u) + j) * a.ch + c, win[j]);
  };
  for (u32 t = t0;;) {
#pragma unroll
    for (u32 i = 0; i < AMDC_CONV_ROWS; i++) {
      if (t + i >= t1) break;
      v4f s = bias;
#pragma unroll
      for (u32 j = 0; j < W - 1u; j++) s = fma4(w[j], win[j], s);
      s = fma4(w[W - 1u], in[i], s);
#pragma unroll
      for (u32 j = 0; j + 2u < W; j++) win[j] = win[j + 1u];
      win[W - 2u] = in[i];
      if (a.act)
#pragma unroll
        for (u32 e = 0; e < C; e++) s[e] *= sigmoid_fast(s[e]);
      stc<TY, C>(a.y, (u64)(row0 + t + i) * a.ys + c, s);
      if (keep) put_state(sl.to[row0 + t + i]);
    }
    t += AMDC_CONV_ROWS;
    if (t >= t1) break;
    rows(t);
  }
  if (!first_rows || keep) return;
  if (t1 < m) // the last rows are other units'
#pragma unroll
    for (u32 j = 0; j < W - 1u; j++) win[j] = row(x, (u64)(m + j - (W - 1u)) * a.xs);
  put_state(o);
}

#define CONV(W, N, TY, C)                                                                                                          \
  extern "C" __global__ __launch_bounds__(64) void amdc_conv_w##W##_##N(const amdc_slots_dev sl, const amdc_conv_args a) { conv_body<W##u, TY, C##u>(sl, a); }
#define CONVS(W) CONV(W, f32, 0, 4) CONV(W, f16, 1, 4) CONV(W, bf16, 2, 4) CONV(W, f32_odd, 0, 1) CONV(W, f16_odd, 1, 1) CONV(W, bf16_odd, 2, 1)
CONVS(2) CONVS(3) CONVS(4)

// ------------------------------------------------------------------ the gated delta rule, token after token

// What the gates of value head h at a row are made of; its log decay (at most 0, NaN kept) and rate
struct GdnGates {
  float a, b, A, dt;
  __device__ __forceinline__ GdnGates(const amdc_gdn_args &g, u64 row, u32 h) : a(g.a[row * g.as + h]), b(g.b[row * g.bs + h]), A(g.A[h]), dt(g.dt[h]) {}
  __device__ __forceinline__ void get(float &decay, float &rate) const {
    const float x = a + dt, v = A * ((x > 0.0f ? x : 0.0f) + log1pf(__builtin_expf(-__builtin_fabsf(x))));
    decay = v > 0.0f ? 0.0f : v;
    rate = 1.0f / (1.0f + __builtin_expf(-b));
  }
};
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
// so that k S, q S, k.k, q.q and k.q go through one reduction a token. Reading and writing the states bounds it for batches: 96
// sequences of 32 heads of 128 x 128, 405 MB, in 80 us (5.0 TB/s, a copy's rate here); 8 of 48 heads and 5 tokens, a state kept after each,
// 154 MB in 33 us. A single sequence waits for two dependent loads (its slot, the state): 4.3 us, and 0.8 a token more, which a wave's
// instructions take. Rows and gates are loaded ahead of the state, which waits for its slot: behind it, 84, 35 and 4.6 us.
template <int TY, u32 DK>
__device__ __forceinline__ void gdn_rec_body(const amdc_slots_dev &sl, const amdc_gdn_args &g, u32 most) {
  constexpr u32 NI = DK / 16u;
  const u32 lane = threadIdx.x & 63u, ng = g.dv >> 4, w = uniform(4u * blockIdx.x + (threadIdx.x >> 6));
  if (w >= sl.n_seq * g.n_v * ng) return;
  const u32 b = w / (g.n_v * ng), hw = w - b * g.n_v * ng, h = hw / ng, c = 16u * (hw - h * ng), hk = gdn_key_head(g, h);
  const u32 r = lane >> 2, c4 = lane & 3u;
  u32 row0;
  const u32 m = uniform(slot_rows(sl, b, row0));
  if (!m || m > most) return;
  const int f = sl.from[b];
  const GdnGates gates(g, row0 + (lane < m ? lane : m - 1u), h); // a token to a lane: all of them are loaded beside the state
  float k[NI], q[NI];
  v4f v;
  const auto load = [&](u32 t) {
    const u64 row = row0 + t;
#pragma unroll
    for (u32 i = 0; i < NI; i++) k[i] = ld1<TY>(g.k, row * g.ks + hk * DK + 16u * i + r), q[i] = ld1<TY>(g.q, row * g.qs + hk * DK + 16u * i + r);
    v = ld4<TY>(g.v, row * g.vs + h * g.dv + c + 4u * c4);
  };
  load(0u);
  bool bad;
  const bool have = slot_ok(sl, f, bad);
  const u64 mat = (u64)DK * g.dv, part = (u64)h * mat + (u64)c * DK + 16u * r + 4u * c4;
  v4f S[NI];
#pragma unroll
  for (u32 i = 0; i < NI; i++) S[i] = splat(bad ? nan_() : 0.0f);
  if (have)
#pragma unroll
    for (u32 i = 0; i < NI; i++) S[i] = *(const v4f *)(g.s + (u64)(u32)f * g.n_v * mat + part + 256u * i);
  float decay, rate;
  gates.get(decay, rate);
  decay = __builtin_expf(decay);
  for (u32 t = 0; t < m; t++) {
    const float e = lane_of(decay, t), be = lane_of(rate, t);
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
    if (r == 0u) st4<TY>(g.y, (u64)(row0 + t) * g.ys + h * g.dv + c + 4u * c4, y);
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
  extern "C" __global__ __launch_bounds__(256) void amdc_gdn_rec_h##H##_##N(const amdc_slots_dev sl, const amdc_gdn_args g) { gdn_rec_body<TY, H##u>(sl, g, AMDC_LIN_MAX_T); }
#define GDN_RECS(H) GDN_REC(H, f32, 0) GDN_REC(H, f16, 1) GDN_REC(H, bf16, 2)
GDN_RECS(64) GDN_RECS(128)

// ------------------------------------------------------------------ the gated delta rule in chunks of 64 tokens
//
// Inside a chunk, with G_i the sum of the log decays up to token i, the updates u_i = beta_i (v_i - k_i S_(i-1)) solve
//   (I + L) U = R,  L_ij = beta_i e^(G_i - G_j) k_i.k_j (j < i),  R_i = beta_i (v_i - e^(G_i) k_i S)
// for the state S before the chunk, and then
//   y_i = e^(G_i) q_i S + sum_(j <= i) e^(G_i - G_j) q_i.k_j u_j,   S <- e^(G_63) S + sum_j e^(G_63 - G_j) k_j^T u_j.
// Two launches: amdc_gdn_prep computes what does not depend on the state, for all chunks at once: M = (I + L)^-1 and the weights
// A_ij = e^(G_i - G_j) q_i.k_j for each value head, and the normed keys and queries as operands; amdc_gdn_scan takes the chunks of a sequence
// one after the other, 32 columns of a head's state to a workgroup. Of packed prompts the sequences of up to AMDC_LIN_MAX_T rows (decode steps
// beside prompts) go token after token, in workgroups of amdc_gdn_prep's launch ahead of its own: 96 of one token, 48 heads of 128, in 152 us,
// as chunks 522; 32 of 5 tokens 80 and 171, of 16 162 and 168. A prompt of 12000 tokens, 16 heads of keys and 48 of values of 128: 0.58 ms,
// 0.14 of it amdc_gdn_prep's, which writes 0.51 GB of operands (4.4 TB/s with what it reads); token after token it takes 11.1 ms. Prompts go
// through the workspace in parts of AMDC_GDN_WS bytes (a launch of the scan begins and ends with all its workgroups): 12000, 24000 and 48000 tokens in parts of
// 64 MB 0.68, 1.35, 2.70 ms, 128 MB 0.63, 1.25, 2.50, 256 MB 0.61, 1.21, 2.43, 512 MB 0.58, 1.15, 2.32, 1 GB 0.58, 1.13, 2.28; 4 of 6000 1.34, 1.23, 1.20, 1.22,
// 1.06 (192 workgroups a sequence on 256 CUs: two sequences in a part are two rounds, four in one are three).
//
// Exponents are of differences that are at most 0, and those are taken in 64 bits: after a strong decay the sums are large and
// their differences small. |M_ij|, |A_ij| <= 1: (I - beta k^T k) shrinks whatever it multiplies, for beta <= 1 and |k| <= 1.
//
// All products are on the f16 matrix units with both operands in two parts, x = hi + lo with 11 bits each, and three products, hi hi +
// hi lo + lo hi, which keeps 22 bits and so f32's accuracy (the errors against 64 bits are those of the recurrence in f32). What f16's
// range needs: M is at most 1 (its parts end at 2^-25, f32's accuracy of the 1s on its diagonal), keys, queries and A are and are multiplied by 2^8;
// columns of S, R and U by a power of two each, from a bound of the column's values. For S += K^T U both sides have 2^4.
//
// The operands' k index is permuted so that the results of one product, four rows of a tile in a lane, are the next product's operand in
// the same lane: place (g, e) of 32, lane group g, element e, is k = 16 (e / 4) + 4 g + e % 4.

typedef _Float16 h4 __attribute__((ext_vector_type(4)));
#define GDN_C 64u        // tokens of a chunk
#define GDN_UP 256.0f    // what operands of size up to 1 are multiplied by
#define GDN_UT 16.0f     // and those of the product that adds to S, on either side: S is in the square of this
#define GDN_P 68u        // words of a row of 64 in the LDS: four lane groups, four rows apart, are 16 banks apart

__device__ __forceinline__ h8 join8(h4 a, h4 b) { return (h8){a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]}; }
// four values in two parts each
__device__ __forceinline__ void split4(v4f x, h4 &hi, h4 &lo) {
  hi = __builtin_convertvector(x, h4);
#pragma unroll
  for (u32 e = 0; e < 4u; e++) lo[e] = (_Float16)__builtin_fmaf((float)hi[e], -1.0f, x[e]);
}
__device__ __forceinline__ v4f mfma_f16(h8 a, h8 b, v4f c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
// (a[0] + a[1]) (b[0] + b[1]) without the product of the low parts
__device__ __forceinline__ v4f mfma3(const h8 (&a)[2], const h8 (&b)[2], v4f c) { return mfma_f16(a[0], b[0], mfma_f16(a[0], b[1], mfma_f16(a[1], b[0], c))); }
// the wave's own LDS accesses stay in order
__device__ __forceinline__ void wave_order() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}
// The power of two that brings values of up to m under 2^7, and its inverse. Both are normal: of values under 2^-112 fewer bits are kept.
__device__ __forceinline__ void pow2_of(float m, float &up, float &down) {
  const u32 e = __builtin_bit_cast(u32, m) >> 23 & 255u;
  const u32 f = 260u - e < 246u ? 260u - e : 246u;
  up = __builtin_bit_cast(float, f << 23), down = __builtin_bit_cast(float, (254u - f) << 23);
}
__device__ __forceinline__ float max4(v4f x) { return __builtin_fmaxf(__builtin_fmaxf(__builtin_fabsf(x.x), __builtin_fabsf(x.y)), __builtin_fmaxf(__builtin_fabsf(x.z), __builtin_fabsf(x.w))); }
// The largest of the four lanes that are 16 apart, of values that are not negative: their bits are in their order, NaN the largest
__device__ __forceinline__ float max_groups(float v) {
  u32 u = __builtin_bit_cast(u32, v);
  auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  u = r[0] > r[1] ? r[0] : r[1];
  r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  u = r[0] > r[1] ? r[0] : r[1];
  return __builtin_bit_cast(float, u);
}

// Where chunk slot s (of all sequences', in their order) lies: with cu, sequence b's chunks are the slots cu[b] / 64 + b on, which leaves room for
// each one's last, partial chunk.
__device__ __forceinline__ u32 gdn_base(const amdc_slots_dev &sl, u32 nc, u32 b) {
  if (!sl.cu) return b * nc;
  const int c = sl.cu[b];
  return (c < 0 ? 0u : (u32)c) / GDN_C + b;
}
__device__ __forceinline__ u32 gdn_seq(const amdc_slots_dev &sl, u32 nc, u32 s) {
  return sl.cu ? find_seq(sl.n_seq, s, [&](u32 i) { return gdn_base(sl, nc, i); }) : s / nc;
}

// What amdc_gdn_scan has to know of packed sequences, 64 to a wave (block k) of amdc_gdn_prep's launch: of those with chunks in this launch, from the one
// of its first slot on, the number, first row, rows (0: no chunk here) and first slot; of each 64 of them in the order of their chunks here, the
// most first, so that of these those which take longest begin first. Without it each of the scan's
// workgroups searches for its sequence: 90 sequences of up to 150 tokens, 32 heads of 128, 262 us, 294 without; 40 of up to 900, 16 heads of 64, 78 and 92.
// A single sequence needs none (77 tokens: 22.0 us, 23.7 with it).
__device__ __forceinline__ void gdn_table(const amdc_slots_dev &sl, const amdc_gdn_args &g, u32 k) {
  const u32 lane = threadIdx.x, seqs = g.groups / g.n_k, n = seqs - 64u * k < 64u ? seqs - 64u * k : 64u;
  if (lane >= 64u) return;
  const u32 b = gdn_seq(sl, g.nc, g.s0) + 64u * k + lane, end = g.s0 + g.ns;
  u32 row0 = 0u, m = 0u, base = 0u, len = 0u;
  if (lane < n && b < sl.n_seq) {
    m = slot_rows(sl, b, row0), base = gdn_base(sl, g.nc, b);
    const u32 to = base + (m + GDN_C - 1u) / GDN_C, x = base > g.s0 ? base : g.s0, y = to < end ? to : end;
    len = m > g.few && y > x ? y - x : 0u;
  }
  u32 rank = 0u;
  for (u32 j = 0; j < n; j++) {
    const u32 other = (u32)__builtin_amdgcn_readlane((int)len, (int)j);
    rank += other > len || (other == len && j < lane);
  }
  if (lane < n) g.table[64u * k + rank] = (amdc_gdn_seq){b, row0, len ? m : 0u, base};
}

// The workspace: a chunk slot holds for every key head its keys, queries and transposed keys as operands (fragments of 1 KB: 16
// rows, 32 of k, the lanes' 16 bytes in order; two parts each), then for every value head M and A (the 6 fragments that are not all above the
// diagonal, in parts) and for each token the factors beta, 2^-8 beta e^G, e^G, 2^-4 e^(G_63 - G).
__device__ __forceinline__ u32 gdn_tri(u32 i, u32 s) { return i < 2u ? i : 2u * (i - 1u) + s; }

template <int TY, u32 DK>
__device__ __forceinline__ void gdn_prep_body(const amdc_slots_dev &sl, const amdc_gdn_args &g) {
  constexpr u32 KS = DK / 32u, SCR = 4u * 4u * 336u * 4u;
  constexpr u32 FA = 64u * DK * 4u > SCR ? 64u * DK * 4u : SCR, FB = 2u * 64u * GDN_P * 4u > DK * GDN_P * 4u ? 2u * 64u * GDN_P * 4u : DK * GDN_P * 4u;
  __shared__ __align__(16) uint8_t s_a[FA]; // the keys' fragments; then each wave's blocks
  __shared__ __align__(16) uint8_t s_b[FB]; // the keys, transposed, two parts in a word; then k.k and q.k
  __shared__ double s_G[4][64];
  __shared__ float s_beta[4][64];
  const u32 tid = threadIdx.x, lane = tid & 63u, w = uniform(tid >> 6), n = lane & 15u, gr = lane >> 4;
  const u32 wg = blockIdx.x - g.rec - g.tabs, at = wg / g.n_k, hk = wg - at * g.n_k, slot = g.s0 + at;
  if (sl.cu && !g.few) check_rows(sl, slot, hk); // else the waves that go token after token have
  const u32 b = gdn_seq(sl, g.nc, slot);
  if (b >= sl.n_seq) return;
  u32 row0;
  const u32 m = uniform(slot_rows(sl, b, row0)), c = slot - uniform(gdn_base(sl, g.nc, b));
  if (m <= g.few || c >= (m + GDN_C - 1u) / GDN_C) return;
  const u32 first = row0 + c * GDN_C, mc = m - c * GDN_C < GDN_C ? m - c * GDN_C : GDN_C;
  uint8_t *ws = g.ws + (u64)at * g.sb, *wk = ws + (u64)hk * (3u * 64u * DK * 4u);

  // the gates of a value head, a token to a lane: the sums of its log decays into the LDS, the tokens' factors into the workspace
  const auto head = [&](u32 v) { return g.tiled ? hk + v * g.n_k : hk * g.G + v; };
  const auto raw_gates = [&](u32 v) { return GdnGates(g, first + (lane < mc ? lane : mc - 1u), head(v < g.G ? v : 0u)); };
  const auto gates = [&](u32 v, const GdnGates &raw) {
    const u32 h = head(v);
    float decay, beta;
    raw.get(decay, beta);
    // e^-10000 is 0: an infinite decay makes no NaN of a difference
    decay = lane < mc ? decay < -1e4f ? -1e4f : decay : 0.0f, beta = lane < mc ? beta : 0.0f;
    double G = (double)decay;
#pragma unroll
    for (u32 o = 1; o < 64u; o <<= 1) {
      const double up = __shfl_up(G, o);
      G += lane >= o ? up : 0.0;
    }
    s_G[w][lane] = G, s_beta[w][lane] = beta;
    const float since = __builtin_expf((float)G), until = __builtin_expf((float)(__shfl(G, 63) - G));
    float *cf = (float *)(ws + (u64)g.n_k * (3u * 64u * DK * 4u) + (u64)h * AMDC_GDN_VB + 24576u);
    cf[lane] = beta, cf[64u + lane] = beta * since * (1.0f / GDN_UP), cf[128u + lane] = since, cf[192u + lane] = until * (GDN_UT / GDN_UP);
  };
  // keys and queries: wave w the rows 16 w .. + 15, as operands of the products along dk
  h8 kf[KS][2], qf[KS][2];
  {
    const GdnGates raw = raw_gates(w); // asked for ahead of the others, and used while they are on their way
    const u32 r = 16u * w + n;
    const bool on = r < mc;
    const u64 row = first + (on ? r : mc - 1u);
    v4f k[KS][2], q[KS][2];
#pragma unroll
    for (u32 s = 0; s < KS; s++)
#pragma unroll
      for (u32 p = 0; p < 2u; p++) {
        k[s][p] = ld4<TY>(g.k, row * g.ks + hk * DK + 32u * s + 16u * p + 4u * gr);
        q[s][p] = ld4<TY>(g.q, row * g.qs + hk * DK + 32u * s + 16u * p + 4u * gr);
      }
    if (w < g.G) gates(w, raw);
    v4f kk = splat(0.0f), qq = splat(0.0f);
#pragma unroll
    for (u32 s = 0; s < KS; s++)
#pragma unroll
      for (u32 p = 0; p < 2u; p++) kk = fma4(k[s][p], k[s][p], kk), qq = fma4(q[s][p], q[s][p], qq);
    float sk = (kk.x + kk.y) + (kk.z + kk.w), sq = (qq.x + qq.y) + (qq.z + qq.w);
    sk += __shfl_xor(sk, 16), sq += __shfl_xor(sq, 16);
    sk += __shfl_xor(sk, 32), sq += __shfl_xor(sq, 32);
    const float rk = on ? GDN_UP / __builtin_sqrtf(sk + g.eps) : 0.0f, rq = on ? GDN_UP / __builtin_sqrtf(sq + g.eps) : 0.0f;
    u32 *kt = (u32 *)s_b;
#pragma unroll
    for (u32 s = 0; s < KS; s++) {
      h4 hi[2], lo[2], qh[2], ql[2];
#pragma unroll
      for (u32 p = 0; p < 2u; p++) {
        split4(k[s][p] * rk, hi[p], lo[p]);
        split4(q[s][p] * rq, qh[p], ql[p]);
#pragma unroll
        for (u32 e = 0; e < 4u; e++) {
          const _Float16 x = hi[p][e], y = lo[p][e];
          kt[(32u * s + 16u * p + 4u * gr + e) * GDN_P + r] = (u32)__builtin_bit_cast(unsigned short, x) | (u32)__builtin_bit_cast(unsigned short, y) << 16;
        }
      }
      kf[s][0] = join8(hi[0], hi[1]), kf[s][1] = join8(lo[0], lo[1]);
      qf[s][0] = join8(qh[0], qh[1]), qf[s][1] = join8(ql[0], ql[1]);
#pragma unroll
      for (u32 p = 0; p < 2u; p++) {
        const u32 f = 1024u * ((w * KS + s) * 2u + p) + 16u * lane;
        *(h8 *)(s_a + f) = kf[s][p];
        *(h8 *)(wk + f) = kf[s][p];
        *(h8 *)(wk + 64u * DK * 4u + f) = qf[s][p];
      }
    }
  }
  __syncthreads();
  // the transposed keys
#pragma unroll
  for (u32 i = 0; i < DK / 64u; i++) {
    const u32 M = w + 4u * i;
#pragma unroll
    for (u32 s = 0; s < 2u; s++) {
      const u32 *kt = (const u32 *)s_b + (16u * M + n) * GDN_P + 32u * s + 4u * gr;
      const u32x4 x = *(const u32x4 *)kt, y = *(const u32x4 *)(kt + 16u);
      const u32x4 hi = {__builtin_amdgcn_perm(x.y, x.x, 0x05040100u), __builtin_amdgcn_perm(x.w, x.z, 0x05040100u), __builtin_amdgcn_perm(y.y, y.x, 0x05040100u),
                        __builtin_amdgcn_perm(y.w, y.z, 0x05040100u)};
      const u32x4 lo = {__builtin_amdgcn_perm(x.y, x.x, 0x07060302u), __builtin_amdgcn_perm(x.w, x.z, 0x07060302u), __builtin_amdgcn_perm(y.y, y.x, 0x07060302u),
                        __builtin_amdgcn_perm(y.w, y.z, 0x07060302u)};
      const u32 f = 2u * 64u * DK * 4u + 1024u * ((M * 2u + s) * 2u) + 16u * lane;
      *(h8 *)(wk + f) = __builtin_bit_cast(h8, hi) * (_Float16)(GDN_UT / GDN_UP);
      *(h8 *)(wk + f + 1024u) = __builtin_bit_cast(h8, lo) * (_Float16)(GDN_UT / GDN_UP);
    }
  }
  // k.k and q.k, the tiles up to the diagonal: a fragment of keys is either operand
  v4f kk[4], qk[4];
#pragma unroll
  for (u32 j = 0; j < 4u; j++) {
    kk[j] = qk[j] = splat(0.0f);
    if (j <= w)
#pragma unroll
      for (u32 s = 0; s < KS; s++) {
        const h8 bf[2] = {*(const h8 *)(s_a + 1024u * ((j * KS + s) * 2u) + 16u * lane), *(const h8 *)(s_a + 1024u * ((j * KS + s) * 2u + 1u) + 16u * lane)};
        kk[j] = mfma3(kf[s], bf, kk[j]), qk[j] = mfma3(qf[s], bf, qk[j]);
      }
  }
  __syncthreads();
  float *KK = (float *)s_b, *QK = KK + 64u * GDN_P;
#pragma unroll
  for (u32 j = 0; j < 4u; j++)
    if (j <= w)
#pragma unroll
      for (u32 e = 0; e < 4u; e++) {
        const u32 f = (16u * w + 4u * gr + e) * GDN_P + 16u * j + n;
        KK[f] = kk[j][e] * (1.0f / (GDN_UP * GDN_UP)), QK[f] = qk[j][e] * (1.0f / GDN_UP); // q.k stays multiplied by 2^8
      }
  __syncthreads();
  // a value head to a wave
  float *blk = (float *)(s_a + w * (SCR / 4u));
  for (u32 v = w; v < g.G; v += 4u) {
    const u32 h = head(v);
    uint8_t *wv = ws + (u64)g.n_k * (3u * 64u * DK * 4u) + (u64)h * AMDC_GDN_VB;
    if (v >= 4u) gates(v, raw_gates(v));
    wave_order();
    // L by blocks of 16 x 16, row n, columns 4 gr .. of a block in a lane; A's fragments on the way
    v4f L[10];
#pragma unroll
    for (u32 i = 0; i < 4u; i++) {
      const u32 r = 16u * i + n;
      const double Gr = s_G[w][r];
      const float be = s_beta[w][r];
      h4 hi[4], lo[4];
#pragma unroll
      for (u32 j = 0; j < 4u; j++) {
        if (j > i) {
          hi[j] = lo[j] = (h4){0, 0, 0, 0};
          continue;
        }
        const u32 cl = 16u * j + 4u * gr;
        const v4f x = *(const v4f *)(KK + r * GDN_P + cl), y = *(const v4f *)(QK + r * GDN_P + cl);
        v4f l, a;
#pragma unroll
        for (u32 e = 0; e < 4u; e++) {
          const float d = __builtin_amdgcn_exp2f((float)(Gr - s_G[w][cl + e]) * 1.4426950408889634f);
          l[e] = cl + e < r ? be * (x[e] * d) : 0.0f;
          a[e] = cl + e <= r ? y[e] * d : 0.0f;
        }
        L[i * (i + 1u) / 2u + j] = l;
        split4(a, hi[j], lo[j]);
      }
#pragma unroll
      for (u32 s = 0; s < (i < 2u ? 1u : 2u); s++) {
        uint8_t *f = wv + 12288u + 2048u * gdn_tri(i, s) + 16u * lane;
        *(h8 *)f = join8(hi[2u * s], hi[2u * s + 1u]);
        *(h8 *)(f + 1024u) = join8(lo[2u * s], lo[2u * s + 1u]);
      }
      // the diagonal block, for its inverse
      *(v4f *)(blk + 336u * i + 20u * n + 4u * gr) = L[i * (i + 1u) / 2u + i];
    }
    wave_order();
    // the inverses of the four diagonal blocks: block gr, column n in a lane
    {
      float t[16];
      const float *lb = blk + 336u * gr;
#pragma unroll
      for (u32 r = 0; r < 16u; r++) {
        float s = r == n ? 1.0f : 0.0f;
#pragma unroll
        for (u32 j0 = 0; j0 < r; j0 += 4u) {
          const v4f x = *(const v4f *)(lb + 20u * r + j0);
#pragma unroll
          for (u32 e = 0; e < 4u; e++)
            if (j0 + e < r) s = __builtin_fmaf(-x[e], t[j0 + e], s);
        }
        t[r] = s;
      }
      wave_order();
#pragma unroll
      for (u32 r = 0; r < 16u; r++) blk[336u * gr + 20u * r + n] = t[r];
    }
    wave_order();
    v4f M[10], dg[4]; // M by blocks as L; the diagonal ones also column n, rows 4 gr .. in a lane, as results and right operands have them
#pragma unroll
    for (u32 i = 0; i < 4u; i++) {
      M[i * (i + 1u) / 2u + i] = *(const v4f *)(blk + 336u * i + 20u * n + 4u * gr);
#pragma unroll
      for (u32 e = 0; e < 4u; e++) dg[i][e] = blk[336u * i + 20u * (4u * gr + e) + n];
    }
    wave_order();
    // M_ij = -M_ii sum_m L_im M_mj, f32 matrix units
#pragma unroll
    for (u32 j = 0; j < 3u; j++) {
      v4f col[4];
      col[j] = dg[j];
#pragma unroll
      for (u32 i = j + 1u; i < 4u; i++) {
        v4f x = splat(0.0f), y = splat(0.0f);
#pragma unroll
        for (u32 k = j; k < i; k++)
#pragma unroll
          for (u32 e = 0; e < 4u; e++) x = __builtin_amdgcn_mfma_f32_16x16x4f32(L[i * (i + 1u) / 2u + k][e], col[k][e], x, 0, 0, 0);
#pragma unroll
        for (u32 e = 0; e < 4u; e++) y = __builtin_amdgcn_mfma_f32_16x16x4f32(M[i * (i + 1u) / 2u + i][e], x[e], y, 0, 0, 0);
        col[i] = -y;
#pragma unroll
        for (u32 e = 0; e < 4u; e++) blk[336u * i + 20u * (4u * gr + e) + n] = col[i][e];
      }
      wave_order();
#pragma unroll
      for (u32 i = j + 1u; i < 4u; i++) M[i * (i + 1u) / 2u + j] = *(const v4f *)(blk + 336u * i + 20u * n + 4u * gr);
      wave_order();
    }
#pragma unroll
    for (u32 i = 0; i < 4u; i++) {
      h4 hi[4], lo[4];
#pragma unroll
      for (u32 j = 0; j < 4u; j++)
        if (j <= i) split4(M[i * (i + 1u) / 2u + j], hi[j], lo[j]);
        else hi[j] = lo[j] = (h4){0, 0, 0, 0};
#pragma unroll
      for (u32 s = 0; s < (i < 2u ? 1u : 2u); s++) {
        uint8_t *f = wv + 2048u * gdn_tri(i, s) + 16u * lane;
        *(h8 *)f = join8(hi[2u * s], hi[2u * s + 1u]);
        *(h8 *)(f + 1024u) = join8(lo[2u * s], lo[2u * s + 1u]);
      }
    }
  }
}

// The chunks of a sequence one after the other: a workgroup has 32 columns of a head's state (in its registers, as results of the
// products), and for each chunk three products that wait for each other:
//   R = beta v - beta e^G (K S), and Q S on the way;   U = M R;   y = e^G (Q S) + A U and S = e^(G_63) S + K^T (e^(G_63 - G) U).
// Eight waves, in two roles, two to a SIMD: a wave alone has every wait to itself. Waves 0 to 3 have 16 tokens' rows each: they make R, then U, and y while the
// others bring S on. Waves 4 to 7 have 32 rows of S (dk = 64: 16), and of Q S what 16 tokens need, which they make beside U. Keys, queries, M and A are read
// once a workgroup, straight into registers; S, R, U and Q S go through the LDS.
// A column's R, U and its next S are under 12 max |S| + 65 max |beta v| of the chunk (a token adds at most beta |v| to the column's norm, and the rest of
// its step shrinks it): the power of two of this bound brings them into f16's range, and as they share it U needs no scaling. max |S| is not waited for:
// what it was a chunk before bounds it, by the same rule. S is kept as the products with K^T give it: they add to it.
// A chunk takes 2.3 to 2.5 us, waits of many kinds: matrix units 27 % busy, vector units 36 %, the LDS 34 %; without its products it
// would take 92 % of that, without its reads of the workspace 93 %. 16 columns a workgroup would read the workspace twice as
// often, 64 leave half of the CUs idle.
// PAIR: two values side by side in v and y are aligned to both (32-bit ones need not be).
template <int TY, u32 DK, bool PAIR>
__device__ __forceinline__ void gdn_scan_body(const amdc_slots_dev &sl, const amdc_gdn_args &g) {
  constexpr u32 KS = DK / 32u, RT = DK / 64u, ES = TY ? 2u : 4u; // RT: row tiles of S that a wave has
  __shared__ __align__(16) uint8_t s_S[KS * 4096u], s_R[8192], s_U[8192], s_W[8192], s_Q[8192];
  __shared__ __align__(16) float s_smax[2][4][32], s_vmax[2][4][32], s_cf[4][4][64];
  const u32 tid = threadIdx.x, lane = tid & 63u, wave = uniform(tid >> 6), w = wave & 3u, n = lane & 15u, gr = lane >> 4;
  const u32 nb = (g.dv + 31u) / 32u, per = g.G * nb;
  // the workgroups of a key head are on one XCD (workgroups go round the 8 of them), where the group count allows it: 12000 tokens 578 us, as they
  // come 666; 77 tokens 22.3 and 24.2
  u32 gi, in;
  if (g.groups >= 8u) {
    const u32 x = blockIdx.x & 7u, y = blockIdx.x >> 3;
    gi = (y / per) * 8u + x, in = y % per;
  } else gi = blockIdx.x / per, in = blockIdx.x % per;
  if (gi >= g.groups) return;
  const u32 i = gi / g.n_k, hk = gi % g.n_k, vh = in / nb, cb = in - vh * nb;
  u32 b, row0, m, base;
  if (g.packed) {
    const amdc_gdn_seq e = g.table[i];
    b = uniform(e.b), row0 = uniform(e.row0), m = uniform(e.m), base = uniform(e.base);
  } else { // all of one length, or a single one
    b = sl.cu ? 0u : g.s0 / g.nc + i;
    if (b >= sl.n_seq) return;
    m = uniform(slot_rows(sl, b, row0)), row0 = uniform(row0), base = uniform(gdn_base(sl, g.nc, b));
    if (m <= g.few) return;
  }
  const u32 all = (m + GDN_C - 1u) / GDN_C, end = g.s0 + g.ns;
  if (!m || base >= end || base + all <= g.s0) return;
  const u32 h = g.tiled ? hk + vh * g.n_k : hk * g.G + vh;
  const u32 c0 = base < g.s0 ? g.s0 - base : 0u, c1 = base + all < end ? all : end - base;
  const u32 col = 32u * cb + 2u * n; // the lane's columns: this one in the products' first column tile, the next in the second
  const u64 mat = (u64)DK * g.dv;

  // the state: from the slot, or where the call's launches left off
  const bool chain = wave < 4u;
  bool bad = false;
  v4f S[2][RT];
  const auto s_at = [&](u32 t, u32 p, u32 e) { return ((u64)((col + t) >> 4) * DK + 16u * (RT * w + p) + 4u * gr + e) * 16u + (col + t & 15u); };
  if (!chain) {
    const int f = sl.from[b];
    const bool have = slot_ok(sl, f, bad) && c0 == 0u;
    const float *src = have ? g.s + ((u64)(u32)f * g.n_v + h) * mat : g.carry_in + (u64)h * mat;
    const bool on = col < g.dv && (have || c0);
#pragma unroll
    for (u32 t = 0; t < 2u; t++)
#pragma unroll
      for (u32 p = 0; p < RT; p++)
#pragma unroll
        for (u32 e = 0; e < 4u; e++) S[t][p][e] = on ? src[s_at(t, p, e)] : bad && !c0 ? nan_() : 0.0f;
  }
  const auto put_smax = [&](u32 c, const float(&by)[2]) {
#pragma unroll
    for (u32 t = 0; t < 2u; t++) s_smax[c & 1u][w][16u * t + n] = by[t] * max_groups(RT == 2u ? __builtin_fmaxf(max4(S[t][0]), max4(S[t][RT - 1u])) : max4(S[t][0]));
  };
  const auto put_S = [&]() { // S as a right operand
#pragma unroll
    for (u32 t = 0; t < 2u; t++) {
      h4 hi[RT], lo[RT];
#pragma unroll
      for (u32 p = 0; p < RT; p++) split4(S[t][p], hi[p], lo[p]);
      if constexpr (RT == 2u) {
        uint8_t *f = s_S + 1024u * ((w * 2u + t) * 2u) + 16u * lane;
        *(h8 *)f = join8(hi[0], hi[1]);
        *(h8 *)(f + 1024u) = join8(lo[0], lo[1]);
      } else {
        uint8_t *f = s_S + 1024u * (((w >> 1) * 2u + t) * 2u) + 16u * lane + 8u * (w & 1u);
        *(h4 *)f = hi[0];
        *(h4 *)(f + 1024u) = lo[0];
      }
    }
  };
  const auto put = [&](uint8_t *to, u32 t, v4f x) { // 16 rows of a right operand of 64
    h4 hi, lo;
    split4(x, hi, lo);
    uint8_t *f = to + 1024u * (((w >> 1) * 2u + t) * 2u) + 16u * lane + 8u * (w & 1u);
    *(h4 *)f = hi;
    *(h4 *)(f + 1024u) = lo;
  };
  const auto get = [&](const uint8_t *from, u32 s, u32 t, h8 (&x)[2]) {
    const uint8_t *f = from + 1024u * ((s * 2u + t) * 2u) + 16u * lane;
    x[0] = *(const h8 *)f, x[1] = *(const h8 *)(f + 1024u);
  };
  // Loads go where they hold up no wave that others wait for: 128 KB a chunk come at 64 bytes a cycle, and a wave whose loads find the queue
  // full waits. That is behind U for the first four waves, and ahead of U for the others.
  h8 kq[KS][2], tf[RT][2][2], mf[2][2], af[2][2]; // keys or queries; K^T; M; A
  v4f raw[2], val[2];                   // the values; beta times them
  float factor = 0.0f;
  // a chunk's slot of the workspace (under 2^31 bytes), where key head and value head begin in it, and the lane's 16 bytes of a fragment. A line
  // of 128 bytes is asked for by one load of the workgroup: a second one while it is on its way would stop the cache until it is there.
  const auto chunk_ws = [&](u32 c) { return rsrc(g.ws + (u64)(base + (c < c1 ? c : c1 - 1u) - g.s0) * g.sb, (u32)g.sb); };
  const u32 ok = hk * (3u * 64u * DK * 4u), ov = g.n_k * (3u * 64u * DK * 4u) + h * AMDC_GDN_VB;
  const auto frag = [&](__amdgpu_buffer_rsrc_t r, u32 at) { return __builtin_bit_cast(h8, __builtin_amdgcn_raw_buffer_load_b128(r, 16u * lane, at, 0)); };
  // the tokens' factors, 64 of each of four kinds: a wave's load each, in the LDS from the chunk before to the one behind
  const auto load_factor = [&](u32 c) { factor = __builtin_bit_cast(float, (u32)__builtin_amdgcn_raw_buffer_load_b32(chunk_ws(c), 4u * lane, ov + 24576u + 256u * w, 0)); };
  const auto put_factor = [&](u32 c) { s_cf[c & 3u][w][lane] = factor; };
  const auto four = [&](u32 c, u32 i) { return *(const v4f *)&s_cf[c & 3u][i][16u * w + 4u * gr]; };
  // rows and columns that are not there are beyond the end of these buffers: loads give 0, stores nothing
  const auto rows_of = [&](const void *p, u32 c, u32 stride) {
    const u32 left = c < c1 ? m - c * GDN_C : 0u;
    return rsrc((const uint8_t *)p + (u64)(row0 + c * GDN_C) * stride * ES, (left < GDN_C ? left : GDN_C) * stride * ES);
  };
  u32 voff[4], yoff[4];
#pragma unroll
  for (u32 e = 0; e < 4u; e++) {
    const u32 r = 16u * w + 4u * gr + e;
    voff[e] = col < g.dv ? (r * g.vs + h * g.dv + col) * ES : 0xC0000000u, yoff[e] = col < g.dv ? (r * g.ys + h * g.dv + col) * ES : 0xC0000000u;
  }
  const auto load_val = [&](u32 c) {
    const __amdgpu_buffer_rsrc_t r = rows_of(g.v, c, g.vs);
#pragma unroll
    for (u32 e = 0; e < 4u; e++) {
      u32 x, y = 0u;
      if constexpr (TY == 0) {
        const u32x2 p = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(r, voff[e], 0, 0));
        x = p.x, y = p.y;
      } else if constexpr (PAIR) x = (u32)__builtin_amdgcn_raw_buffer_load_b32(r, voff[e], 0, 0); // both halves
      else x = (u32)__builtin_amdgcn_raw_buffer_load_b16(r, voff[e], 0, 0), y = (u32)__builtin_amdgcn_raw_buffer_load_b16(r, voff[e] + 2u, 0, 0);
      raw[0][e] = __builtin_bit_cast(float, x), raw[1][e] = __builtin_bit_cast(float, y);
    }
  };
  const auto load_kq = [&](u32 c, u32 q, u32 s) { // the part along 32 of dk
    const __amdgpu_buffer_rsrc_t r = chunk_ws(c);
#pragma unroll
    for (u32 i = 0; i < 2u; i++) kq[s][i] = frag(r, ok + q * (64u * DK * 4u) + 1024u * ((KS * w + s) * 2u + i));
  };
  const auto put_vmax = [&](u32 c) {
    const v4f beta = four(c, 0u);
#pragma unroll
    for (u32 e = 0; e < 4u; e++) {
      const float x = raw[0][e], y = raw[1][e];
      const u32 u = __builtin_bit_cast(u32, x), v = __builtin_bit_cast(u32, y), z = PAIR ? u >> 16 : v;
      val[0][e] = beta[e] * (TY == 0 ? x : TY == 2 ? __builtin_bit_cast(float, u << 16) : h2f(u));
      val[1][e] = beta[e] * (TY == 0 ? y : TY == 2 ? __builtin_bit_cast(float, z << 16) : h2f(z));
    }
#pragma unroll
    for (u32 t = 0; t < 2u; t++) {
      s_vmax[c & 1u][w][16u * t + n] = max_groups(max4(val[t]));
    }
  };
  // A line from the memory takes as long as half a chunk. So each of the workgroups that share a key head (per of them) or a value head (nb)
  // asks for its part of a chunk two ahead, a line to a lane, which brings it into the L2: where that is an eighth of what it loads at most (12000 tokens,
  // 48 heads of 128 on 16: 262 -> 242 us a launch; heads of 64, two to a key head, a third of it: 82 -> 95, so not there).
  constexpr u32 LK = 3u * 64u * DK * 4u / 128u, LV = AMDC_GDN_VB / 128u;
  const u32 lines_k = (LK + per - 1u) / per, lines_v = (LV + nb - 1u) / nb;
  u32 ahead = 0u, line = 0xC0000000u; // where the lane's line is in a slot
  if (8u * (lines_k + lines_v) <= LK + LV) {
    const u32 i = 64u * w + lane;
    if (i < lines_k && in * lines_k + i < LK) line = ok + 128u * (in * lines_k + i);
    else if (i >= lines_k && i < lines_k + lines_v && cb * lines_v + i - lines_k < LV) line = ov + 128u * (cb * lines_v + i - lines_k);
  }
  const auto prefetch = [&](u32 c) { ahead = (u32)__builtin_amdgcn_raw_buffer_load_b32(chunk_ws(c), line, 0, 0); };
  const u32 upper = w < 2u ? 0xC0000000u : 16u * lane; // the fragments above the diagonal are not there: beyond the end, 0
  const auto load_ma = [&](u32 c, u32 a, h8(&x)[2][2]) { // M or A
    const __amdgpu_buffer_rsrc_t r = chunk_ws(c);
#pragma unroll
    for (u32 i = 0; i < 2u; i++) {
      const u32 at = ov + 12288u * a + 2048u * gdn_tri(w, 0u) + 1024u * i;
      x[0][i] = frag(r, at);
      x[1][i] = __builtin_bit_cast(h8, __builtin_amdgcn_raw_buffer_load_b128(r, upper, at + 2048u, 0));
    }
  };
  const auto load_t = [&](u32 c, u32 k) { // part k of KS
    const __amdgpu_buffer_rsrc_t r = chunk_ws(c);
#pragma unroll
    for (u32 j = 0; j < 2u; j++) {
      const u32 i = RT == 2u ? k & 1u : 0u, s = RT == 2u ? k >> 1 : k;
      tf[i][s][j] = frag(r, ok + 2u * 64u * DK * 4u + 1024u * (((RT * w + i) * 2u + s) * 2u + j));
    }
  };
  struct Tops { // of a column: what the waves say of |S| a chunk ago and of |beta v|, and that chunk's whole decay
    float s[2][4], v[2][4], whole;
  };
  const auto get_tops = [&](u32 c, Tops &x) {
#pragma unroll
    for (u32 t = 0; t < 2u; t++)
#pragma unroll
      for (u32 i = 0; i < 4u; i++) x.s[t][i] = s_smax[(c - 1u) & 1u][i][16u * t + n], x.v[t][i] = s_vmax[c & 1u][i][16u * t + n];
    x.whole = s_cf[(c - 1u) & 3u][2][63];
  };
  const auto top = [](const float(&x)[4]) { return __builtin_fmaxf(__builtin_fmaxf(x[0], x[1]), __builtin_fmaxf(x[2], x[3])); };
  // 16 rows by the columns of both tiles: three products for each 32 of k
  const auto times_S = [&](v4f(&o)[2], auto between) {
    h8 r[KS][2][2];
#pragma unroll
    for (u32 s = 0; s < 2u; s++) get(s_S, s, 0u, r[s][0]), get(s_S, s, 1u, r[s][1]);
    o[0] = o[1] = splat(0.0f);
#pragma unroll
    for (u32 s = 0; s < KS; s++) {
      if (s + 2u < KS) get(s_S, s + 2u, 0u, r[s + 2u][0]), get(s_S, s + 2u, 1u, r[s + 2u][1]);
#pragma unroll
      for (u32 i = 0; i < 3u; i++)
#pragma unroll
        for (u32 t = 0; t < 2u; t++) o[t] = mfma_f16(kq[s][i == 0u], r[s][t][i == 1u], o[t]);
      between(s);
      if (s + 1u < KS) __builtin_amdgcn_sched_barrier(0); // not all of S's operands at once: the registers
    }
  };
  const auto times_64 = [&](const h8(&f)[2][2], const uint8_t *from, v4f(&o)[2]) {
    h8 r[2][2][2];
    o[0] = o[1] = splat(0.0f);
#pragma unroll
    for (u32 s = 0; s < 2u; s++)
      if (s == 0u || w >= 2u) get(from, s, 0u, r[s][0]), get(from, s, 1u, r[s][1]);
#pragma unroll
    for (u32 s = 0; s < 2u; s++)
      if (s == 0u || w >= 2u)
#pragma unroll
        for (u32 i = 0; i < 3u; i++)
#pragma unroll
          for (u32 t = 0; t < 2u; t++) o[t] = mfma_f16(f[s][i == 0u], r[s][t][i == 1u], o[t]);
  };
  // bounds of |S| and |beta v|; the factor of R, U and the next S, and the inverses of S's and of that
  float most[2], vmost[2], up[2], down_S[2], down[2];
  const auto factors = [&](u32 c, const Tops &x) {
#pragma unroll
    for (u32 t = 0; t < 2u; t++) {
      if (c != c0) most[t] = __builtin_fmaf(12.0f * x.whole, top(x.s[t]), 65.0f * vmost[t]);
      vmost[t] = top(x.v[t]);
      pow2_of(__builtin_fmaf(12.0f, most[t], 65.0f * vmost[t]), up[t], down[t]);
    }
  };
  if (chain) {
    load_factor(c0), put_factor(c0), load_factor(c0 + 1u), put_factor(c0 + 1u);
#pragma unroll
    for (u32 s = 0; s < KS; s++) load_kq(c0, 0u, s);
    load_ma(c0, 0u, mf), load_ma(c0, 1u, af), load_val(c0);
  } else {
    const float one[2] = {1.0f, 1.0f};
    put_smax(c0 + 1u, one);
  }
  __syncthreads();
#pragma unroll
  for (u32 t = 0; t < 2u; t++) {
    float x[4];
#pragma unroll
    for (u32 i = 0; i < 4u; i++) x[i] = s_smax[(c0 + 1u) & 1u][i][16u * t + n];
    most[t] = top(x), vmost[t] = 0.0f;
    pow2_of(most[t], up[t], down_S[t]);
  }
  if (chain) {
    put_vmax(c0), load_val(c0 + 1u), load_factor(c0 + 2u);
    for (u32 c = c0; c < c1; c++) {
      __syncthreads(); // S is there
      Tops tops;
      get_tops(c, tops);
      const v4f bs = four(c, 1u);
      v4f P[2];
      times_S(P, [](u32) {});
      factors(c, tops);
#pragma unroll
      for (u32 t = 0; t < 2u; t++) put(s_R, t, fma4(-bs, P[t] * (down_S[t] * (1.0f / GDN_UP)), val[t]) * (up[t] * GDN_UP));
      __syncthreads(); // R is there
      v4f U[2];
      times_64(mf, s_R, U);
      const v4f until = four(c, 3u);
#pragma unroll
      for (u32 t = 0; t < 2u; t++) {
        put(s_W, t, U[t] * until);
        load_kq(c + 1u, 0u, t); // a load takes its time: between the others
        put(s_U, t, U[t]);
      }
      put_factor(c + 2u);
      __syncthreads(); // U and Q S are there
#pragma unroll
      for (u32 s = 2; s < KS; s++) load_kq(c + 1u, 0u, s);
      load_ma(c + 1u, 0u, mf), load_factor(c + 3u);
      put_vmax(c + 1u);
      asm volatile("" ::"v"(ahead));
      load_val(c + 2u), prefetch(c + 2u);
      v4f y[2];
      times_64(af, s_U, y);
      load_ma(c + 1u, 1u, af);
      const __amdgpu_buffer_rsrc_t ry = rows_of(g.y, c, g.ys);
      const float sc = g.scale * (1.0f / GDN_UP / GDN_UP);
      const v4f since = four(c, 2u);
#pragma unroll
      for (u32 t = 0; t < 2u; t++) {
        const v4f q = *(const v4f *)(s_Q + 2048u * w + 1024u * t + 16u * lane);
        y[t] = fma4(splat(down[t] * sc), y[t], since * (down_S[t] * sc) * q);
        down_S[t] = down[t];
      }
#pragma unroll
      for (u32 e = 0; e < 4u; e++) {
        const float o = y[0][e], z = y[1][e];
        const u32 u = __builtin_bit_cast(u32, o), v = __builtin_bit_cast(u32, z);
        if constexpr (TY == 0) __builtin_amdgcn_raw_buffer_store_b64((u32x2){u, v}, ry, yoff[e], 0, 0);
        else {
          const u32 x = pack2<TY == 2>(o, z);
          if constexpr (PAIR) __builtin_amdgcn_raw_buffer_store_b32(x, ry, yoff[e], 0, 0);
          else __builtin_amdgcn_raw_buffer_store_b16((unsigned short)x, ry, yoff[e], 0, 0), __builtin_amdgcn_raw_buffer_store_b16((unsigned short)(x >> 16), ry, yoff[e] + 2u, 0, 0);
        }
      }
    }
    return;
  }
#pragma unroll
  for (u32 t = 0; t < 2u; t++)
#pragma unroll
    for (u32 p = 0; p < RT; p++) S[t][p] *= up[t] * GDN_UP;
  put_S();
  for (u32 c = c0; c < c1; c++) {
    __syncthreads(); // S is there
#pragma unroll
    for (u32 s = 0; s < KS; s++) load_kq(c, 1u, s);
    const float by[2] = {down_S[0] * (1.0f / GDN_UP), down_S[1] * (1.0f / GDN_UP)};
    put_smax(c, by);
    Tops tops;
    get_tops(c, tops);
    factors(c, tops);
    const float whole = s_cf[c & 3u][2][63];
#pragma unroll
    for (u32 t = 0; t < 2u; t++) {
#pragma unroll
      for (u32 p = 0; p < RT; p++) S[t][p] = S[t][p] * down_S[t] * whole * up[t];
      down_S[t] = down[t];
    }
    __syncthreads(); // R is there
    v4f Q[2];
    times_S(Q, [&](u32 s) { load_t(c, s); });
#pragma unroll
    for (u32 t = 0; t < 2u; t++) *(v4f *)(s_Q + 2048u * w + 1024u * t + 16u * lane) = Q[t];
    __syncthreads(); // U and Q S are there
    h8 z[2][2][2];
#pragma unroll
    for (u32 s = 0; s < 2u; s++)
#pragma unroll
      for (u32 t = 0; t < 2u; t++) get(s_W, s, t, z[s][t]);
#pragma unroll
    for (u32 s = 0; s < 2u; s++)
#pragma unroll
      for (u32 i = 0; i < 3u; i++)
#pragma unroll
        for (u32 t = 0; t < 2u; t++)
#pragma unroll
          for (u32 p = 0; p < RT; p++) S[t][p] = mfma_f16(tf[p][s][i == 0u], z[s][t][i == 1u], S[t][p]);
    put_S();
  }
  // the state: into its slot, or for the launch that goes on
  float *dst = g.carry_out + (u64)h * mat;
  bool write = true;
  if (c1 == all) {
    const int o = sl.to[b];
    bool worse;
    const bool start_ok = sl.from[b] >= -1 && sl.from[b] < (int)sl.n_slots;
    write = slot_ok(sl, o, worse) && start_ok;
    dst = g.s + ((u64)(u32)(o < 0 ? 0 : o) * g.n_v + h) * mat;
  }
  if (!write || col >= g.dv) return;
#pragma unroll
  for (u32 t = 0; t < 2u; t++)
#pragma unroll
    for (u32 p = 0; p < RT; p++)
#pragma unroll
      for (u32 e = 0; e < 4u; e++) dst[s_at(t, p, e)] = S[t][p][e] * (down[t] * (1.0f / GDN_UP));
}

#define GDN_PREP(H, N, TY)                                                                                                             \
  extern "C" __global__ __launch_bounds__(256) void amdc_gdn_prep_h##H##_##N(const amdc_slots_dev sl, const amdc_gdn_args g) { \
    if (blockIdx.x < g.rec) gdn_rec_body<TY, H##u>(sl, g, g.few);                                                                       \
    else if (blockIdx.x < g.rec + g.tabs) gdn_table(sl, g, blockIdx.x - g.rec);                                                         \
    else gdn_prep_body<TY, H##u>(sl, g);                                                                                               \
  }
#define GDN_SCAN(H, N, TY, PAIR)                                                                                                       \
  extern "C" __global__ __launch_bounds__(512) void amdc_gdn_scan_h##H##_##N(const amdc_slots_dev sl, const amdc_gdn_args g) { gdn_scan_body<TY, H##u, PAIR>(sl, g); }
#define GDN_PRES(H)                                                                                                                    \
  GDN_PREP(H, f32, 0) GDN_PREP(H, f16, 1) GDN_PREP(H, bf16, 2)                                                                         \
  GDN_SCAN(H, f32, 0, true) GDN_SCAN(H, f16, 1, true) GDN_SCAN(H, bf16, 2, true) GDN_SCAN(H, f16_odd, 1, false) GDN_SCAN(H, bf16_odd, 2, false)
GDN_PRES(64) GDN_PRES(128)

// ------------------------------------------------------------------ the norms

// y = x s w gate(z), s = 1 / sqrt(sum x^2 / hd + eps) over a head, and its Q8 copy. Reading and writing bound it. Four values a lane, hd / 4 lanes a
// head. Grid (ceil(n / 1024), T). 4097 rows of 32 heads of 128 from bf16: 168 MB in 31 us (5.4 TB/s); one row of 48 heads 2.4 us. With the Q8 copy
// alone, as the next matrix takes it: 122 MB in 27.6 us (4.4 TB/s; from f32 155 MB in 29.6, 5.2 TB/s), one row 2.5 us.
template <int TY>
__device__ __forceinline__ void norm_gate_body(const amdc_norm_args &a) {
  const u32 i0 = 4u * (blockIdx.x * NT + threadIdx.x), n = a.n;
  const bool on = i0 < n; // whole heads, and whole blocks of 32, at once
  const u32 i = on ? i0 : n - 4u;
  const v4f x = ld4<TY>((const uint8_t *)a.x + (u64)blockIdx.y * a.xs, i), z = ld4<0>((const uint8_t *)a.z + (u64)blockIdx.y * a.zs, i);
  const v4f w = ld4<0>(a.w, i & (a.hd - 1u));
  const float ss = seg_sum((x.x * x.x + x.y * x.y) + (x.z * x.z + x.w * x.w), a.hd >> 2);
  const float s = 1.0f / __builtin_sqrtf(ss / (float)a.hd + a.eps);
  v4f y;
#pragma unroll
  for (u32 j = 0; j < 4u; j++) {
    const float g = sigmoid_fast(z[j]);
    y[j] = x[j] * s * w[j] * (a.gate ? g : z[j] * g);
  }
  if (on && a.y) st4<0>((uint8_t *)a.y + (u64)blockIdx.y * a.ys, i, y);
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
// norms. h may be res: a thread reads and writes the same places. Grid (1, T). Reading and writing bound it: 3001 rows of 4096, 197 MB, in 40 us
// (4.9 TB/s, a copy's rate); one row of 5120 3.4 us. With the Q8 copy alone, as the next matrix takes it: 163 MB in 37 us (4.4 TB/s), one row
// 4.5 us. 256 threads of more values each: 45 and 4.8 us, to y (1024 rows of 4096, which the caches hold, 12.3 against 12.6).
template <u32 NV>
__device__ __forceinline__ void norm_res_body(const amdc_norm_args &a) {
  __shared__ float part[2][16];
  const u32 n = a.n, step = 4u * blockDim.x;
  const float rn = 1.0f / (float)n;
  const uint8_t *px = (const uint8_t *)a.x + (u64)blockIdx.y * a.xs, *pr = (const uint8_t *)a.z + (u64)blockIdx.y * a.zs;
  constexpr bool EARLY = NV <= 2u; // the weights beside the rows; more do not fit the registers
  v4f x[NV], h[NV], w1[EARLY ? NV : 1u], w2[EARLY ? NV : 1u];
#pragma unroll
  for (u32 j = 0; j < NV; j++) {
    const u32 i = 4u * threadIdx.x + j * step, k = i < n ? i : n - 4u;
    x[j] = ld4<0>(px, k), h[j] = ld4<0>(pr, k);
    if (i >= n) x[j] = h[j] = splat(0.0f);
    if constexpr (EARLY) w1[j] = a.w ? ld4<0>(a.w, k) : splat(1.0f), w2[j] = ld4<0>(a.w2, k);
  }
  const float s1 = a.w ? row_scale<NV>(x, rn, a.eps, part[0]) : 1.0f;
#pragma unroll
  for (u32 j = 0; j < NV; j++) {
    const u32 i = 4u * threadIdx.x + j * step;
    if (i < n) {
      if (a.w) x[j] = x[j] * s1 * (EARLY ? w1[EARLY ? j : 0u] : ld4<0>(a.w, i));
      h[j] = fma4(splat(a.scale), x[j], h[j]);
      st4<0>((uint8_t *)a.h + (u64)blockIdx.y * a.hs, i, h[j]);
    }
  }
  const float s2 = row_scale<NV>(h, rn, a.eps, part[1]);
#pragma unroll
  for (u32 j = 0; j < NV; j++) {
    const u32 i = 4u * threadIdx.x + j * step;
    const bool on = i < n;
    const v4f y = h[j] * s2 * (EARLY ? w2[EARLY ? j : 0u] : ld4<0>(a.w2, on ? i : 0u));
    if (on && a.y) st4<0>((uint8_t *)a.y + (u64)blockIdx.y * a.ys, i, y);
    if (a.q) quant_vec4(y, (on ? i : 0u) >> 5, on, a.q + (u64)blockIdx.y * a.qs, n >> 5);
  }
}
#define NORM_RES(NV, LIM)                                                                                                              \
  extern "C" __global__ __launch_bounds__(LIM) void amdc_norm_res_##NV(const amdc_norm_args a) { norm_res_body<NV##u>(a); }
NORM_RES(1, 1024) NORM_RES(2, 1024) NORM_RES(4, 1024) NORM_RES(8, 1024)
