// Selective state space scan over (batch, length, channels), forward:
//   dt = softplus(delta + bias),  h[n] = exp(dt A[n]) h[n] + dt u B[n],
//   out = (sum_n h[n] C[n] + D u) * silu(z)
//
// A step maps h to a h + b, and such maps compose: (a2, b2) after (a1, b1) is
// (a2 a1, a2 b1 + b2). So the steps of one channel are split over G lanes, 8
// consecutive steps each: a lane composes its 8 maps, the G lanes scan the
// compositions by shuffles (log2 G rounds), and each lane, now knowing the
// state in front of its steps, walks them again for the outputs, with the
// same a and b still in registers. A range's factor is the product of its
// steps' while none of them can be above 1. Where A > 0, or dt < 0 for want of
// the softplus, that product can pass the largest float32 in front of a state
// that is 0 or small; there a block takes exp(A sum dt), applied as its square
// root, twice (8 x 2048 x 2048 without softplus: 391 us against 367 with the
// products; a second form of the whole kernel for dt >= 0 there took 380). Each exponential is computed once, which
// matters because they bound the kernel: N per value on the special-function
// unit (16 a clock and SM) against about 6 N FP32 operations (128 a clock).
// Splitting the axis over blocks instead would need the exponentials twice.
// A block holds 128 / G channels and walks the sequence in pieces of 8 G
// steps. The next piece's rows come by asynchronous copies while a piece is
// computed (global rows run over channels, a lane needs its channel's steps,
// so they pass through shared memory); B and C, shared by the block's
// channels, are converted to float32 once per piece. States go in fours: 4
// chains in flight, 16-byte reads of B and C, and the two-wide FP32
// instructions over pairs of states.
// Measured, 16 states, bf16: 8 x 2048 x 2048 in 390 us, 1.4e12 exponentials a
// second (38 % of the special-function unit, issue slots 55 %, shared memory
// 63 %; HBM would take 41 us); 1 x 8192 x 2048 in 318 us. What is
// left is latency at 13 warps an SM: steps are a chain within a channel.
// Giving each thread a share of a channel's states over all steps instead (no
// compositions, 30 % fewer instructions) took 350 us at 8 x 2048 x 2048, but
// 756 at 1 x 8192 x 2048, where too few warps are left.
#include <algorithm>

#include "scan.cuh"

namespace ferrum {
namespace seq {
namespace {

constexpr int kLaneSteps = 8;

// G lanes share a channel's steps, S warps its states.
template <class T, int G, int S, int NP>
struct FwdCfg {
  static constexpr int THREADS = S == 1 ? 128 : 256;
  static constexpr int CH = THREADS / S / G;      // channels per block
  static constexpr int CK = kLaneSteps * G;       // steps per piece
  static constexpr int ROUNDS = G == 4 ? 2 : (G == 8 ? 3 : 4);   // log2 G
  static constexpr int XS = Piece<T, CH>::size(CK), RS = Piece<T, NP>::size(CK);
  static constexpr int FS = Piece<float, NP>::size(CK);
  static constexpr int YS = CH * (CK + 4);        // a float32 (channel, step) tile
  static constexpr size_t BYTES =
      sizeof(T) * (size_t)(6 * XS + 2 * RS) +
      sizeof(float) * (size_t)(2 * FS + 2 * CH * NP + (S == 1 ? 0 : (S + 1) * YS));
};

// The square roots of two states' factors over steps whose dt add up to 2 w.
// Clamped below the exponent range's end: a factor that large overflows any
// state but 0. A NaN stays.
__device__ __forceinline__ f2 root_factor(float w, float Ax, float Ay) {
  const float2 e = unpack(exponents(pack(w, w), pack(Ax, Ay)));
  return pack(ex2(min_nan(e.x, 127.f)), ex2(min_nan(e.y, 127.f)));
}

template <class T, int G, int S, int NP>
__global__ void __launch_bounds__(FwdCfg<T, G, S, NP>::THREADS, 512 / FwdCfg<T, G, S, NP>::THREADS)
scan_fwd_kernel(ScanIn<T> in, Rows<T> out, float* fin, float* __restrict__ saved, ScanSizes s,
                int64_t col_blocks, int unit, int bc_unit, int out_unit, bool save_vec) {
  using C = FwdCfg<T, G, S, NP>;
  constexpr int CH = C::CH, CK = C::CK, kThreads = C::THREADS, ROUNDS = C::ROUNDS;
  using X = Piece<T, CH>;
  using F = Piece<float, NP>;
  extern __shared__ float4 smem4[];
  float* sB = (float*)smem4;
  float* sC = sB + C::FS;
  float* sA = sC + C::FS;              // A log2 e
  float* sH = sA + CH * NP;            // the state in front of the piece
  float* sDt = sH + CH * NP;           // S > 1: dt, then the warps' parts of y
  float* sY = sDt + (S == 1 ? 0 : C::YS);
  T* raw = (T*)(sY + (S == 1 ? 0 : S * C::YS));   // 2 x (u, delta, z), then B, C as they come
  T* rawB = raw + 6 * C::XS;
  T* rawC = rawB + C::RS;

  int64_t q = blockIdx.x;
  const int64_t cb = q % col_blocks;
  q /= col_blocks;
  const int64_t grp = q % s.groups, b = q / s.groups;
  const int64_t d0 = grp * s.per_group + cb * CH;
  const int nch = (int)(s.per_group - cb * CH < CH ? s.per_group - cb * CH : CH);
  const int64_t len = scan_length(in.lengths, b, s.length);
  const int tid = threadIdx.x, g = tid % G, sg = tid / (CH * G);   // sg: this warp's states
  const int c = tid / G % CH, row = c * (CK + 4) + g * 8;
  const bool live = c < nch;

  auto fetch = [&](int64_t t0, int buf) {
    const int rows = (int)(len - t0 < CK ? len - t0 : CK);
    T* x = raw + buf * 3 * C::XS;
    copy_piece<T, CK, CH, kThreads>(x, in.u.at(b, t0) + d0, (int)in.u.st, rows, nch, unit, tid);
    copy_piece<T, CK, CH, kThreads>(x + C::XS, in.delta.at(b, t0) + d0, (int)in.delta.st, rows,
                                    nch, unit, tid);
    if (in.z)
      copy_piece<T, CK, CH, kThreads>(x + 2 * C::XS, in.z.at(b, t0) + d0, (int)in.z.st, rows, nch,
                                      unit, tid);
    copy_piece<T, CK, NP, kThreads>(rawB, in.B.at(b, t0) + grp * in.B_group, (int)in.B.st, rows,
                                    s.states, bc_unit, tid);
    copy_piece<T, CK, NP, kThreads>(rawC, in.C.at(b, t0) + grp * in.C_group, (int)in.C.st, rows,
                                    s.states, bc_unit, tid);
  };
  auto put = [&](int64_t t0, int buf) {
    store_piece<T, CK, CH, kThreads>(out.at(b, t0) + d0, raw + buf * 3 * C::XS, (int)out.st,
                                     (int)(s.length - t0 < CK ? s.length - t0 : CK), nch, out_unit,
                                     tid);
  };
  if (len > 0) fetch(0, 0);

  bool above = !s.softplus;
  for (int i = tid; i < CH * NP; i += kThreads) {
    const int cc = i / NP, n = i % NP;
    const bool ok = cc < nch && n < s.states;
    const int64_t o = (d0 + cc) * s.states + n;
    sA[i] = ok ? scaled_rate(in.A[o]) : 0.f;
    above = above || sA[i] > 0.f;
    sH[i] = (ok && in.initial) ? in.initial[b * s.channels * s.states + o] : 0.f;
  }
  const float bias = (in.bias && live) ? in.bias[d0 + c] : 0.f;
  const float skip = (in.D && live) ? in.D[d0 + c] : 0.f;

  int buf = 0;
  auto walk = [&](auto flag) {
    constexpr bool ABOVE = decltype(flag)::value;   // some factor may be above 1
    for (int64_t t0 = 0; t0 < len; t0 += CK, buf ^= 1) {
      cp_async_wait();
      __syncthreads();
      if (t0 > 0) put(t0 - CK, buf ^ 1);
      widen_piece<T, CK, NP, kThreads>(sB, rawB, tid);
      widen_piece<T, CK, NP, kThreads>(sC, rawC, tid);

      T* mine = raw + buf * 3 * C::XS + X::at(g * 8, c);
      const int64_t left = len - t0 - g * 8;          // valid steps from this lane's first on
      const int steps = left < 0 ? 0 : (left > 8 ? 8 : (int)left);
      float dt[8], du[8];
      f2 y[8];
      constexpr int PART = 8 / S;                     // steps whose dt and output are this warp's
#pragma unroll
      for (int k = 0; k < PART; ++k) {
        const int i = S == 1 ? k : sg * PART + k;
        float v = to_f(mine[C::XS + i * CH]) + bias;
        if (!ABOVE || s.softplus) v = softplus_f(v);
        v = i < steps ? v : 0.f;                      // past the end: a = 1, b = 0
        if constexpr (S == 1)
          dt[k] = v;
        else
          sDt[row + i] = v;
      }
      __syncthreads();
      if (t0 + CK < len) fetch(t0 + CK, buf ^ 1);
      if constexpr (S > 1)
#pragma unroll
        for (int i = 0; i < 8; ++i) dt[i] = sDt[row + i];
#pragma unroll
      for (int i = 0; i < 8; ++i) du[i] = dt[i] * to_f(mine[i * CH]), y[i] = 0;
      float hw[ROUNDS];                               // half the sums of dt over 1, 2, 4.. lanes
      if constexpr (ABOVE) {
        hw[0] = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) hw[0] = fmaf(0.5f, dt[i], hw[0]);
#pragma unroll
        for (int r = 1; r < ROUNDS; ++r)
          hw[r] = hw[r - 1] + __shfl_up_sync(0xffffffffu, hw[r - 1], 1 << (r - 1), G);
      }
      const int64_t ts = t0 + g * 8;
      float* so = nullptr;
      if (saved != nullptr && ts % kSaveSteps == 0 && live && ts < s.length)
        so = saved + ((b * s.saves + ts / kSaveSteps) * s.channels + d0 + c) * s.states;
#pragma unroll 1
      for (int n = sg * (NP / S); n < (sg + 1) * (NP / S); n += 4) {
        const float4 A4 = *(const float4*)(sA + c * NP + n);
        const f2 Ax = pack(A4.x, A4.x), Ay = pack(A4.y, A4.y), Az = pack(A4.z, A4.z),
                 Aw = pack(A4.w, A4.w);
        const float* pb = sB + F::at(g * 8, n);
        const float* pc = sC + F::at(g * 8, n);
        f2 a0[8], a1[8], b0[8], b1[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float4 B4 = *(const float4*)(pb + i * NP);
          b0[i] = pack(du[i] * B4.x, du[i] * B4.y);
          b1[i] = pack(du[i] * B4.z, du[i] * B4.w);
          if (i % 2 == 0) {     // exponents of two steps at a time: A's halves stay put
            const f2 w = pack(dt[i], dt[i + 1]);
            const float2 p = unpack(exponents(w, Ax)), q = unpack(exponents(w, Ay));
            const float2 r = unpack(exponents(w, Az)), v = unpack(exponents(w, Aw));
            a0[i] = pack(ex2(p.x), ex2(q.x)), a0[i + 1] = pack(ex2(p.y), ex2(q.y));
            a1[i] = pack(ex2(r.x), ex2(v.x)), a1[i + 1] = pack(ex2(r.y), ex2(v.y));
          }
        }
        float4* carry = (float4*)(sH + c * NP + n);
        const float4 h4 = *carry;
        f2 h0 = pack(h4.x, h4.y), h1 = pack(h4.z, h4.w), H0 = b0[0], H1 = b1[0];
        f2 P0 = a0[0], P1 = a1[0];
#pragma unroll
        for (int i = 1; i < 8; ++i) {
          H0 = fma2(a0[i], H0, b0[i]), H1 = fma2(a1[i], H1, b1[i]);
          if constexpr (!ABOVE) P0 = mul2(a0[i], P0), P1 = mul2(a1[i], P1);
        }
        // the range's map at the state h
        auto after = [&](f2 P, f2 h, f2 H) { return fma2(P, ABOVE ? mul2(P, h) : h, H); };
#pragma unroll
        for (int r = 0; r < ROUNDS; ++r) {
          const int o = 1 << r;
          if constexpr (ABOVE)
            P0 = root_factor(hw[r], A4.x, A4.y), P1 = root_factor(hw[r], A4.z, A4.w);
          if (r == 0 && g == 0) H0 = after(P0, h0, H0), H1 = after(P1, h1, H1);
          const f2 u0 = __shfl_up_sync(0xffffffffu, H0, o, G);
          const f2 u1 = __shfl_up_sync(0xffffffffu, H1, o, G);
          if (g >= o) H0 = after(P0, u0, H0), H1 = after(P1, u1, H1);
          if (!ABOVE && 2 * o < G) {
            const f2 v0 = __shfl_up_sync(0xffffffffu, P0, o, G);
            const f2 v1 = __shfl_up_sync(0xffffffffu, P1, o, G);
            if (g >= o) P0 = mul2(P0, v0), P1 = mul2(P1, v1);
          }
        }
        // the state in front of this lane's steps; lane 0 gets the piece's last
        const f2 u0 = __shfl_sync(0xffffffffu, H0, (g + G - 1) % G, G);
        const f2 u1 = __shfl_sync(0xffffffffu, H1, (g + G - 1) % G, G);
        if (g == 0) {
          const float2 p = unpack(u0), r = unpack(u1);
          *carry = make_float4(p.x, p.y, r.x, r.y);
        } else {
          h0 = u0, h1 = u1;
        }
        if (so != nullptr) {
          const float2 p = unpack(h0), r = unpack(h1);
          if (!ABOVE && save_vec) {     // (vectors there too spill: 1 x 8191 x 2048 327 us against 316)
            *(float4*)(so + n) = make_float4(p.x, p.y, r.x, r.y);
          } else {
            if (n + 0 < s.states) so[n + 0] = p.x;
            if (n + 1 < s.states) so[n + 1] = p.y;
            if (n + 2 < s.states) so[n + 2] = r.x;
            if (n + 3 < s.states) so[n + 3] = r.y;
          }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float4 C4 = *(const float4*)(pc + i * NP);
          h0 = fma2(a0[i], h0, b0[i]);
          h1 = fma2(a1[i], h1, b1[i]);
          y[i] = fma2(h0, pack(C4.x, C4.y), y[i]);
          y[i] = fma2(h1, pack(C4.z, C4.w), y[i]);
        }
      }
      float sum[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float2 p = unpack(y[i]);
        sum[i] = p.x + p.y;
      }
      if constexpr (S > 1) {
        float4* w = (float4*)(sY + sg * C::YS + row);
        w[0] = make_float4(sum[0], sum[1], sum[2], sum[3]);
        w[1] = make_float4(sum[4], sum[5], sum[6], sum[7]);
        __syncthreads();
      }
#pragma unroll
      for (int k = 0; k < PART; ++k) {
        const int i = S == 1 ? k : sg * PART + k;
        float v = S == 1 ? sum[k] : 0.f;
        if constexpr (S > 1)
#pragma unroll
          for (int r = 0; r < S; ++r) v += sY[r * C::YS + row + i];
        v = fmaf(skip, to_f(mine[i * CH]), v);
        if (in.z) {
          const float z = to_f(mine[2 * C::XS + i * CH]);
          v *= z * sigmoid_f(z);
        }
        mine[i * CH] = from_f<T>(i < steps ? v : 0.f);   // in u's place
      }
    }
  };
  if (__syncthreads_or(above))
    walk(std::true_type());
  else
    walk(std::false_type());
  if (len > 0) {
    __syncthreads();
    put((len - 1) / CK * CK, buf ^ 1);
  }
  // steps past the sequence's last piece
  if (tid % CH < nch)
    for (int64_t t = (len + CK - 1) / CK * CK + tid / CH; t < s.length; t += kThreads / CH)
      out.at(b, t)[d0 + tid % CH] = from_f<T>(0.f);
  if (fin != nullptr) {
    __syncthreads();
    for (int i = tid; i < CH * NP; i += kThreads) {
      const int cc = i / NP, n = i % NP;
      if (cc < nch && n < s.states)
        fin[(b * s.channels + d0 + cc) * s.states + n] = sH[i];
    }
  }
}

// One step: every value of the state is read and written once, which is all
// the traffic that counts. L lanes share a channel, 4 states each (16-byte
// accesses), and add up the output by shuffles. A thread takes its channel in
// BT sequences, with all their loads issued first. The lanes share out the
// sequences' softplus and gate (lane k of a channel those of sequence k), and
// addresses advance by whole strides: with every lane doing both for itself
// the instructions bound the kernel (256 x 4096 x 16: 47 us against 29 for a
// copy of the state).
template <class T, int L, int BT>
__global__ void __launch_bounds__(128)
scan_step_kernel(ScanIn<T> in, Rows<T> out, float* fin, ScanSizes s, bool vec, bool bc_vec,
                 int64_t col_blocks) {
  const int64_t d0 = blockIdx.x % col_blocks * (128 / L) + threadIdx.x / L;
  const int64_t b0 = blockIdx.x / col_blocks * BT;
  const int lane = threadIdx.x % L, n0 = lane * 4, own = lane % BT;
  const bool live = d0 < s.channels;
  const int64_t d = live ? d0 : 0, g = d / s.per_group;
  const int count = s.batch - b0 < BT ? (int)(s.batch - b0) : BT;
  const int64_t bo = b0 + (own < count ? own : 0);         // this lane's sequence

  float h[BT][4], a[4], Bv[BT][4], Cv[BT][4];
  const int64_t step = s.channels * s.states, so = (b0 * s.channels + d) * s.states + n0;
  const float* ph = in.initial + so;
  const T* pb = in.B.at(b0, 0) + g * in.B_group + n0;
  const T* pc = in.C.at(b0, 0) + g * in.C_group + n0;
#pragma unroll
  for (int k = 0; k < BT; ++k) {
    if (k < count) {
      if (vec) {
        load_vec<float, 4>(ph, h[k]);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) h[k][e] = n0 + e < s.states ? ph[e] : 0.f;
      }
      if (bc_vec) {
        load_vec<T, 4>(pb, Bv[k]);
        load_vec<T, 4>(pc, Cv[k]);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          Bv[k][e] = n0 + e < s.states ? to_f(pb[e]) : 0.f;
          Cv[k][e] = n0 + e < s.states ? to_f(pc[e]) : 0.f;
        }
      }
    }
    ph += step, pb += in.B.sb, pc += in.C.sb;
  }
  const float x = to_f(in.u.at(bo, 0)[d]);
  float dt = to_f(in.delta.at(bo, 0)[d]) + (in.bias ? in.bias[d] : 0.f);
  const float z = in.z ? to_f(in.z.at(bo, 0)[d]) : 0.f;
  const float* pa = in.A + d * s.states + n0;
  if (vec) {
    load_vec<float, 4>(pa, a);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) a[e] = n0 + e < s.states ? pa[e] : 0.f;
  }
  const float skip = in.D ? in.D[d] : 0.f;
#pragma unroll
  for (int e = 0; e < 4; ++e) a[e] = scaled_rate(a[e]);
  if (s.softplus) dt = softplus_f(dt);
  const float dx = dt * x;
  float* pf = fin + so;
  float mine = 0.f;
#pragma unroll
  for (int k = 0; k < BT; ++k) {
    if (k < count) {                       // the same for the whole block
      const float dtk = BT == 1 ? dt : __shfl_sync(0xffffffffu, dt, k, L);
      const float dxk = BT == 1 ? dx : __shfl_sync(0xffffffffu, dx, k, L);
      float y = 0.f;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        h[k][e] = fmaf(ex2(fmaf(dtk, a[e], kExponentShift)), h[k][e], dxk * Bv[k][e]);
        y = fmaf(h[k][e], Cv[k][e], y);
      }
#pragma unroll
      for (int o = L / 2; o > 0; o >>= 1) y += __shfl_xor_sync(0xffffffffu, y, o, L);
      if (own == k) mine = y;
      if (live) {
        if (vec) {
          store_vec<float, 4>(pf, h[k]);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (n0 + e < s.states) pf[e] = h[k][e];
        }
      }
    }
    pf += step;
  }
  if (live && lane < count) {
    float y = fmaf(skip, x, mine);
    if (in.z) y *= z * sigmoid_f(z);
    out.at(bo, 0)[d] = from_f<T>(y);
  }
}

template <class T, int G, int S, int NP>
ferrum_status run_fwd(const ferrum_scan_args* a, const ScanSizes& s, cudaStream_t stream,
                      const char* what) {
  using C = FwdCfg<T, G, S, NP>;
  static std::atomic<uint64_t> done{0};
  const int64_t col_blocks = ceil_div(s.per_group, C::CH);
  const int64_t blocks = s.batch * s.groups * col_blocks;
  if (blocks > 0x7fffffff) return invalid(what, "too many blocks for one launch");
  cudaError_t e = launch_detail::ensure_smem(scan_fwd_kernel<T, G, S, NP>, C::BYTES, done);
  if (e != cudaSuccess) return cuda_error(e, what);
  const bool one_group = s.groups == 1;
  int unit = std::min(copy_unit<T>(a->u), copy_unit<T>(a->delta, one_group ? 0 : s.per_group));
  if (a->z.ptr) unit = std::min(unit, copy_unit<T>(a->z));
  const int bc_unit = std::min(copy_unit<T>(a->B, a->B_group_stride),
                               copy_unit<T>(a->C, a->C_group_stride));
  launch_detail::clear_stale_error();
  scan_fwd_kernel<T, G, S, NP><<<(unsigned)blocks, C::THREADS, C::BYTES, stream>>>(
      scan_in<T>(a), rows_of<T>(a->out), a->final_state, a->saved_states, s, col_blocks, unit,
      bc_unit, copy_unit<T>(a->out, one_group ? 0 : s.per_group),
      s.states == NP && aligned(a->saved_states, 16));
  return launched(what);
}

int log_states(int states) {   // log2 of the padded number of states, at least 2
  int l = 2;
  while ((1 << l) < states) ++l;
  return l;
}

ferrum_status scan_fwd(ferrum_device* dev, const ferrum_scan_args* a, cudaStream_t stream,
                       const char* what) {
  if (a->batch == 0 || a->channels == 0) return FERRUM_OK;
  const ScanSizes s = scan_sizes(a);
  DeviceGuard guard(dev->ordinal);
  if (guard.status() != cudaSuccess) return cuda_error(guard.status(), "cudaSetDevice");
  // Lanes per channel: few keep the shuffles short. Where a batch has too few
  // channels to fill the GPU that way, a channel gets more lanes, then several
  // warps that share its states. Measured (us, bf16, lanes x warps; the choice
  // marked):
  //                             4 x 1   8 x 1   16 x 1   16 x 2   16 x 4
  //   8 x 2048 x 2048, 16       390*    380     431      549      744
  //   4 x 4096 x 2048, 16       515     422*    437      568      741
  //   2 x 8192 x 2048, 16       851     568     484*     625      758
  //   1 x 8192 x 2048, 16       850     482     338      318*     431
  //   1 x 4096 x 512, 16        427     246     144      120       78*
  //   13 x 777 x 1000, 16, f32  140*    152     184      212      252
  //   8 x 2048 x 2048, 8        266*    258     285      352
  //   2 x 8192 x 2048, 8        613     390     317*     396
  //   1 x 8192 x 2048, 8        613     334     226      204*
  //   2 x 8192 x 2048, 32      1348     935*   1135      936     1196
  //   1 x 8192 x 2048, 32      1348     764     580      475*     671
  //   8 x 2048 x 2048, 64      1153*   1335    3035     1956     2565
  //   2 x 8192 x 2048, 64      2342    1678*   3399     2199     2538
  //   1 x 8192 x 2048, 64      2341    1380    1714     1111*    1450
  // (16 x 1 loses above 16 states: pieces of 128 steps of B and C leave room for
  // three blocks an SM with 32 states, for one with 64.)
  const int64_t rows = s.batch * s.channels;
  const int level = rows >= 12288 || s.length <= 32  ? 0
                    : rows >= 6000 || s.length <= 64 ? 1
                    : rows >= 3000                   ? (s.states > 16 ? 1 : 2)
                    : rows >= 1000                   ? 3 : 4;
  return with_dtype(a->dtype, [&](auto tag) {
    using T = decltype(tag);
    return with_states(s.states, [&](auto np) -> ferrum_status {
      constexpr int NP = decltype(np)::value;
      if (level == 0) return run_fwd<T, 4, 1, NP>(a, s, stream, what);
      if (level == 1) return run_fwd<T, 8, 1, NP>(a, s, stream, what);
      if constexpr (NP <= 16)
        if (level == 2) return run_fwd<T, 16, 1, NP>(a, s, stream, what);
      if (level == 3 || NP == 8) return run_fwd<T, 16, 2, NP>(a, s, stream, what);
      if constexpr (NP > 8) return run_fwd<T, 16, 4, NP>(a, s, stream, what);
      return FERRUM_OK;
    });
  });
}

ferrum_status scan_step(ferrum_device* dev, const ferrum_scan_args* a, cudaStream_t stream,
                        const char* what) {
  if (a->batch == 0 || a->channels == 0) return FERRUM_OK;
  const ScanSizes s = scan_sizes(a);
  const int lanes = 1 << (log_states(s.states) - 2);
  const bool vec = s.states == 4 * lanes && aligned(a->A, 16) && aligned(a->initial_state, 16) &&
                   aligned(a->final_state, 16);
  DeviceGuard guard(dev->ordinal);
  if (guard.status() != cudaSuccess) return cuda_error(guard.status(), "cudaSetDevice");
  return with_dtype(a->dtype, [&](auto tag) {
    using T = decltype(tag);
    auto quad = [&](const ferrum_rows& r, int64_t group) {   // 4 values of a row at once
      const int64_t e = sizeof(T);
      return aligned(r.ptr, 4 * e) && r.batch_stride % 4 == 0 && group % 4 == 0;
    };
    const bool bc_vec = s.states == 4 * lanes && quad(a->B, a->B_group_stride) &&
                        quad(a->C, a->C_group_stride);
    auto go = [&](auto l, auto bt) -> ferrum_status {
      constexpr int L = decltype(l)::value, BT = decltype(bt)::value;
      const int64_t col_blocks = ceil_div(s.channels, 128 / L);
      const int64_t blocks = col_blocks * ceil_div(s.batch, BT);
      if (blocks > 0x7fffffff) return invalid(what, "too many blocks for one launch");
      launch_detail::clear_stale_error();
      scan_step_kernel<T, L, BT><<<(unsigned)blocks, 128, 0, stream>>>(
          scan_in<T>(a), rows_of<T>(a->out), a->final_state, s, vec, bc_vec, col_blocks);
      return launched(what);
    };
    auto lane = [&](auto l) -> ferrum_status {
      // sequences a thread: up to 4 where that still leaves two full waves of blocks
      constexpr int L = decltype(l)::value, BT = L < 4 ? L : 4;
      if (ceil_div(s.channels, 128 / L) * (s.batch / BT) >= 148 * 16)
        return go(l, std::integral_constant<int, BT>());
      return go(l, std::integral_constant<int, 1>());
    };
    switch (lanes) {
      case 1: return lane(std::integral_constant<int, 1>());
      case 2: return lane(std::integral_constant<int, 2>());
      case 4: return lane(std::integral_constant<int, 4>());
      case 8: return lane(std::integral_constant<int, 8>());
      default: return lane(std::integral_constant<int, 16>());
    }
  });
}

}  // namespace

ferrum_status check_scan(const ferrum_device* dev, const ferrum_scan_args* a, const char* what,
                         bool bwd) {
  if (ferrum_status s = check_args(dev, a, what)) return s;
  if (a->states < 1 || a->states > FERRUM_SCAN_MAX_STATES)
    return invalid(what, "states must be in [1, 64], got " + std::to_string(a->states));
  if (a->groups < 1 || a->channels % a->groups != 0)
    return invalid(what, "groups must divide channels (" + std::to_string(a->groups) + ", " +
                             std::to_string(a->channels) + ")");
  if (a->length > (size_t)kMaxElems ||      // (and length + 1 would wrap around)
      bounded_product({a->batch, a->length + 1, a->channels, a->states}) < 0)
    return invalid(what, "batch * length * channels * states is too large");
  for (const ferrum_rows* r : {&a->u, &a->delta, &a->z, &a->out, &a->B, &a->C, &a->dout, &a->du,
                               &a->ddelta, &a->dz})
    if (r->row_stride > 0x7fffffff || r->row_stride < -0x7fffffff)
      return invalid(what, "row strides must fit 32 bits");
  const size_t e = dtype_size(a->dtype);
  const bool none = a->batch == 0 || a->channels == 0, empty = none || a->length == 0;
  if (ferrum_status s = check_ptr(a->A, 4, none, what, "A")) return s;
  if (ferrum_status s = check_ptr(a->D, 4, true, what, "D")) return s;
  if (ferrum_status s = check_ptr(a->delta_bias, 4, true, what, "delta_bias")) return s;
  if (ferrum_status s = check_ptr(a->lengths, 4, true, what, "lengths")) return s;
  if (ferrum_status s = check_ptr(a->initial_state, 4, true, what, "initial_state")) return s;
  if (ferrum_status s = check_ptr(a->u.ptr, e, empty, what, "u")) return s;
  if (ferrum_status s = check_ptr(a->delta.ptr, e, empty, what, "delta")) return s;
  if (ferrum_status s = check_ptr(a->B.ptr, e, empty, what, "B")) return s;
  if (ferrum_status s = check_ptr(a->C.ptr, e, empty, what, "C")) return s;
  if (ferrum_status s = check_ptr(a->z.ptr, e, true, what, "z")) return s;
  if (!bwd) {
    if (ferrum_status s = check_ptr(a->out.ptr, e, empty, what, "out")) return s;
    if (ferrum_status s = check_ptr(a->final_state, 4, true, what, "final_state")) return s;
    return check_ptr(a->saved_states, 4, true, what, "saved_states");
  }
  if (ferrum_status s = check_ptr(a->saved_states, 4, empty, what, "saved_states")) return s;
  if (ferrum_status s = check_ptr(a->dout.ptr, e, empty, what, "dout")) return s;
  if (ferrum_status s = check_ptr(a->du.ptr, e, empty, what, "du")) return s;
  if (ferrum_status s = check_ptr(a->ddelta.ptr, e, empty, what, "ddelta")) return s;
  if (ferrum_status s = check_ptr(a->dz.ptr, e, empty || a->z.ptr == nullptr, what, "dz")) return s;
  if (ferrum_status s = check_ptr(a->dB, e, empty, what, "dB")) return s;
  if (ferrum_status s = check_ptr(a->dC, e, empty, what, "dC")) return s;
  if (ferrum_status s = check_ptr(a->dA, 4, a->channels == 0, what, "dA")) return s;
  if (ferrum_status s = check_ptr(a->dD, 4, true, what, "dD")) return s;
  if (ferrum_status s = check_ptr(a->ddelta_bias, 4, true, what, "ddelta_bias")) return s;
  if (ferrum_status s = check_ptr(a->dfinal_state, 4, true, what, "dfinal_state")) return s;
  return check_ptr(a->dinitial_state, 4, true, what, "dinitial_state");
}

}  // namespace seq
}  // namespace ferrum

using namespace ferrum;
using namespace ferrum::seq;

extern "C" {

ferrum_status ferrum_selective_scan(ferrum_device* dev, const ferrum_scan_args* a, void* stream) {
  const char* what = "selective_scan";
  return guarded(what, [&]() -> ferrum_status {
    if (ferrum_status s = check_scan(dev, a, what, false)) return s;
    return scan_fwd(dev, a, (cudaStream_t)stream, what);
  });
}

ferrum_status ferrum_selective_scan_step(ferrum_device* dev, const ferrum_scan_args* a,
                                         void* stream) {
  const char* what = "selective_scan_step";
  return guarded(what, [&]() -> ferrum_status {
    if (ferrum_status s = check_scan(dev, a, what, false)) return s;
    if (a->length != 1) return invalid(what, "length must be 1, got " + std::to_string(a->length));
    if (a->batch > 0 && a->channels > 0 &&
        (a->initial_state == nullptr || a->final_state == nullptr))
      return invalid(what, "initial_state and final_state are required");
    if (a->lengths != nullptr) return invalid(what, "lengths does not apply to one step");
    return scan_step(dev, a, (cudaStream_t)stream, what);
  });
}

}  // extern "C"
