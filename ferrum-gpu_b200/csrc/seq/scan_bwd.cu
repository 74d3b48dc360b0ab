// Gradient of the selective scan. With h the states, a_t = exp(dt_t A) and
// gh_t the gradient of h_t:
//   gh_t = C_t dy_t + a_{t+1} gh_{t+1}
//   dC_t = sum_d dy_t h_t,           dB_t = sum_d gh_t dt_t u_t
//   du_t = D dy_t + dt_t sum_n gh_t B_t
//   ddt_t = sum_n gh_t (A a_t h_{t-1} + u_t B_t),   dA = sum_t gh_t dt_t a_t h_{t-1}
// A block holds 64 channels: a thread owns two adjacent ones (the FP32
// instructions work on such pairs) and NS of the N states, the S = N / NS warps
// share the states. It walks the saved 16-step pieces from the last to the
// first, in blocks of RB steps. Per block a thread recomputes its states from
// the saved one, keeping them and the exponentials in registers, then walks
// the block backwards. Sums over states go from the warps through shared
// memory; sums over channels (dB, dC) likewise, 16 values of 32 lanes at a
// time (a transposed read costs a third of a reduction by shuffles), and from
// block to block through a workspace, all in fixed order.
// Measured, 8 x 2048 x 2048, 16 states, bf16: 1.15 ms (HBM would take 90 us, the
// special-function unit about 200). Shared memory bandwidth (75 %: tiles, and
// the sums over states and channels) and short-scoreboard waits at 14 warps
// an SM bound it; issue slots are 46 % used. Few sequences leave SMs idle: the
// blocks of one (32 at 2048 channels) walk its steps in a chain, so that
// 1 x 2048 x 2048 takes 0.78 ms, 1 x 8192 x 2048 3.04 and 1 x 4096 x 512 1.50. Four states a thread with the
// sums over states by shuffles inside a warp halves the shared memory
// traffic but leaves 7 warps an SM at that size: 1.35 ms (0.99 against 1.07 at
// 64 x 256 x 2048, 6.7 against 3.7 with 64 states).
#include <algorithm>

#include "scan.cuh"

namespace ferrum {
namespace seq {
namespace {

constexpr int CK = kSaveSteps;   // steps per piece
constexpr int CHN = 64;          // channels per block
constexpr float kLn2 = 0.6931471805599453f;

template <class T, int NP>
struct BwdCfg {
  static constexpr int NS = NP == 64 ? 4 : 2;     // states per thread
  static constexpr int S = NP / NS;               // warps
  static constexpr int RB = NP == 64 ? 4 : 8;     // steps per register block
  static constexpr int NB = CK / RB;
  static constexpr int THREADS = 32 * S;
  static constexpr int FLUSH = 8 / NS;            // steps whose dB, dC make 16 values
  static constexpr int XS = Piece<T, CHN>::size(CK), RS = Piece<T, NP>::size(CK);
  static constexpr int ES = CK * CHN;             // a float32 (step, channel) tile
  static constexpr int DUP = CK * NP * 2;         // B or C, each value twice
  static constexpr int RED = 16 * 36;             // a warp's 16 values of 32 lanes
  static constexpr int SLAB = RB * CHN;           // a warp's part of a sum over states
  // States in front of the later blocks. With two blocks a thread keeps them
  // in its own part of the y sums, which it writes only after reading them
  // back: 4 KB less lets two blocks share an SM.
  static constexpr int CKS = NB > 2 ? (NB - 1) * CHN * NP : 0;
  static constexpr int FLOATS =
      6 * ES + 2 * DUP + CHN * NP + CKS + S * RED + 3 * S * SLAB + CK * 2 * NP;
  static constexpr size_t BYTES = sizeof(float) * (size_t)FLOATS + sizeof(T) * (4 * XS + 2 * RS);
};

template <class T>
struct ScanGrad {
  Rows<T> dout, du, ddelta, dz;
  const float *dfin, *saved;
  float* dinit;
  float *partBC, *partA;  // (blocks, batch, groups, length, 2, N) and (batch, channels, N + 2)
};

__device__ __forceinline__ f2 add2(f2 a, f2 b) {
  f2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// A piece's B or C in float32, each value twice in a row.
template <class T, int NP, int THREADS>
__device__ __forceinline__ void widen_twice(float* dst, const T* src, int tid) {
  for (int i = tid; i < CK * NP; i += THREADS) {
    const float v = to_f(src[Piece<T, NP>::at(i / NP, i % NP)]);
    *(float2*)(dst + 2 * i) = make_float2(v, v);
  }
}

template <class T>
__device__ __forceinline__ void store_pair(T* p, float2 v, int n, bool vec) {
  if constexpr (sizeof(T) == 2) {
    if (vec && n == 2) {
      *(uint32_t*)p = pack_pair<T>(v.x, v.y);
      return;
    }
  }
  if (n > 0) p[0] = from_f<T>(v.x);
  if (n > 1) p[1] = from_f<T>(v.y);
}

template <class T, int NP>
__global__ void __launch_bounds__(BwdCfg<T, NP>::THREADS, 512 / BwdCfg<T, NP>::THREADS)
scan_bwd_kernel(ScanIn<T> in, ScanGrad<T> gr, ScanSizes s, int64_t group_blocks, int unit,
                int bc_unit, bool state_vec, bool out_vec) {
  using C = BwdCfg<T, NP>;
  constexpr int NS = C::NS, S = C::S, RB = C::RB, NB = C::NB, THREADS = C::THREADS;
  using X = Piece<T, CHN>;
  extern __shared__ float4 smem4[];
  float* sDt = (float*)smem4;
  float* sDu = sDt + C::ES;        // dt * u
  float* sDy = sDu + C::ES;        // gradient of y
  float* sX = sDy + C::ES;         // u
  float* sSl = sX + C::ES;         // d dt / d delta
  float* sZg = sSl + C::ES;        // dout * silu'(z)
  float* sB = sZg + C::ES;
  float* sC = sB + C::DUP;
  float* sH0 = sC + C::DUP;        // the piece's saved states
  float* sCk = sH0 + CHN * NP;
  float* sRed = sCk + C::CKS;
  float* sY = sRed + S * C::RED;   // the warps' parts of y, sum g B and sum gah A
  float* sG = sY + S * C::SLAB;
  float* sT = sG + S * C::SLAB;
  float* sBC = sT + S * C::SLAB;   // (step, B / C, state) sums over the channels
  T* raw = (T*)(sBC + CK * 2 * NP);   // u, delta, z, dout, then B and C as they come
  T* rawB = raw + 4 * C::XS;
  T* rawC = rawB + C::RS;

  int64_t q = blockIdx.x;
  const int64_t blk = q % group_blocks;
  q /= group_blocks;
  const int64_t grp = q % s.groups, b = q / s.groups;
  const int64_t d0 = grp * s.per_group + blk * CHN;
  const int nch = (int)(s.per_group - blk * CHN < CHN ? s.per_group - blk * CHN : CHN);
  const int64_t len = scan_length(in.lengths, b, s.length);
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5, n0 = w * NS;
  const int c = 2 * lane;                         // this thread's first channel
  const int nc = nch - c < 0 ? 0 : (nch - c > 2 ? 2 : nch - c);
  const int64_t pieces = (len + CK - 1) / CK;

  auto fetch = [&](int64_t p) {
    const int64_t t0 = p * CK;
    const int rows = (int)(len - t0 < CK ? len - t0 : CK);
    copy_piece<T, CK, CHN, THREADS>(raw, in.u.at(b, t0) + d0, (int)in.u.st, rows, nch, unit, tid);
    copy_piece<T, CK, CHN, THREADS>(raw + C::XS, in.delta.at(b, t0) + d0, (int)in.delta.st, rows,
                                    nch, unit, tid);
    if (in.z)
      copy_piece<T, CK, CHN, THREADS>(raw + 2 * C::XS, in.z.at(b, t0) + d0, (int)in.z.st, rows,
                                      nch, unit, tid);
    copy_piece<T, CK, CHN, THREADS>(raw + 3 * C::XS, gr.dout.at(b, t0) + d0, (int)gr.dout.st, rows,
                                    nch, unit, tid);
    copy_piece<T, CK, NP, THREADS>(rawB, in.B.at(b, t0) + grp * in.B_group, (int)in.B.st, rows,
                                   s.states, bc_unit, tid);
    copy_piece<T, CK, NP, THREADS>(rawC, in.C.at(b, t0) + grp * in.C_group, (int)in.C.st, rows,
                                   s.states, bc_unit, tid);
  };
  auto fetch_state = [&](int64_t p) {
    const float* h0 = gr.saved + ((b * s.saves + p) * s.channels + d0) * s.states;
    if (state_vec) {
      for (int i = tid; i < CHN * NP / 4; i += THREADS)
        cp_async<16>(sH0 + 4 * i, i * 4 < nch * NP ? h0 + 4 * i : h0, i * 4 < nch * NP ? 16 : 0);
    } else {
      for (int i = tid; i < CHN * NP; i += THREADS) {
        const int cc = i / NP, n = i % NP;
        sH0[i] = cc < nch && n < s.states ? h0[cc * s.states + n] : 0.f;
      }
    }
  };
  if (pieces > 0) fetch(pieces - 1), fetch_state(pieces - 1);

  f2 A[NS], r[NS], dA[NS];         // A log2 e; gradient of the state behind; sum
#pragma unroll
  for (int k = 0; k < NS; ++k) {
    float a[2], g[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const bool ok = e < nc && n0 + k < s.states;
      const int64_t o = (d0 + c + e) * s.states + n0 + k;
      a[e] = ok ? scaled_rate(in.A[o]) : 0.f;
      g[e] = ok && gr.dfin ? gr.dfin[b * s.channels * s.states + o] : 0.f;
    }
    A[k] = pack(a[0], a[1]), r[k] = pack(g[0], g[1]), dA[k] = 0;
  }
  float2 bias = make_float2(0.f, 0.f), skip = bias, dD = bias, dbias = bias;
  if (in.bias && nc > 0) bias.x = in.bias[d0 + c];
  if (in.bias && nc > 1) bias.y = in.bias[d0 + c + 1];
  if (in.D && nc > 0) skip.x = in.D[d0 + c];
  if (in.D && nc > 1) skip.y = in.D[d0 + c + 1];

  for (int64_t p = pieces - 1; p >= 0; --p) {
    const int64_t t0 = p * CK;
    const int rows = (int)(len - t0 < CK ? len - t0 : CK);
    cp_async_wait();
    __syncthreads();
    widen_twice<T, NP, THREADS>(sB, rawB, tid);
    widen_twice<T, NP, THREADS>(sC, rawC, tid);
    for (int t = w; t < CK; t += S) {
      float vdt[2], vx[2], vdy[2], vsl[2], vzg[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const bool ok = t < rows && e < nc;
        const int o = X::at(t, c) + e;
        const float v = to_f(raw[C::XS + o]) + (e ? bias.y : bias.x);
        vx[e] = to_f(raw[o]);
        vdy[e] = to_f(raw[3 * C::XS + o]);
        float dt = v, slope = 1.f;
        if (s.softplus) dt = softplus_f(v, slope);
        vdt[e] = ok ? dt : 0.f;
        vsl[e] = ok ? slope : 0.f;
        vzg[e] = 0.f;
        if (in.z) {
          const float z = to_f(raw[2 * C::XS + o]), sg = sigmoid_f(z);
          vzg[e] = vdy[e] * sg * (1.f + z * (1.f - sg));
          vdy[e] *= z * sg;
        }
      }
      const int o = t * CHN + c;
      *(float2*)(sDt + o) = make_float2(vdt[0], vdt[1]);
      *(float2*)(sDu + o) = make_float2(vdt[0] * vx[0], vdt[1] * vx[1]);
      *(float2*)(sDy + o) = make_float2(vdy[0], vdy[1]);
      *(float2*)(sX + o) = make_float2(vx[0], vx[1]);
      *(float2*)(sSl + o) = make_float2(vsl[0], vsl[1]);
      *(float2*)(sZg + o) = make_float2(vzg[0], vzg[1]);
    }
    f2 h0[NS];
#pragma unroll
    for (int k = 0; k < NS; ++k)
      h0[k] = pack(sH0[c * NP + n0 + k], sH0[(c + 1) * NP + n0 + k]);
    // this thread's slots for the states in front of block 1 and up
    f2* ck = NB > 2 ? (f2*)sCk + tid : (f2*)(sY + w * C::SLAB + c);
    constexpr int CKSTEP = NB > 2 ? THREADS : CHN / 2;
    __syncthreads();
    if (p > 0) fetch(p - 1), fetch_state(p - 1);

    // the states in front of the later blocks
    {
      f2 h[NS];
#pragma unroll
      for (int k = 0; k < NS; ++k) h[k] = h0[k];
#pragma unroll 4
      for (int t = 0; t < (NB - 1) * RB; ++t) {
        const f2 dt = *(const f2*)(sDt + t * CHN + c), du = *(const f2*)(sDu + t * CHN + c);
#pragma unroll
        for (int k = 0; k < NS; ++k) {
          const float2 e = unpack(exponents(dt, A[k]));
          h[k] = fma2(pack(ex2(e.x), ex2(e.y)), h[k],
                      mul2(du, *(const f2*)(sB + (t * NP + n0 + k) * 2)));
        }
        if ((t + 1) % RB == 0)
#pragma unroll
          for (int k = 0; k < NS; ++k) ck[(((t + 1) / RB - 1) * NS + k) * CKSTEP] = h[k];
      }
    }
#pragma unroll 1
    for (int j = NB - 1; j >= 0; --j) {
      const int tb = j * RB;
      f2 a[RB][NS], h[RB + 1][NS];
#pragma unroll
      for (int k = 0; k < NS; ++k)
        h[0][k] = j == 0 ? h0[k] : ck[((j - 1) * NS + k) * CKSTEP];
#pragma unroll
      for (int i = 0; i < RB; ++i) {
        const int t = tb + i;
        const f2 dt = *(const f2*)(sDt + t * CHN + c), du = *(const f2*)(sDu + t * CHN + c);
        f2 y = 0;
#pragma unroll
        for (int k = 0; k < NS; ++k) {
          const float2 e = unpack(exponents(dt, A[k]));
          a[i][k] = pack(ex2(e.x), ex2(e.y));
          h[i + 1][k] = fma2(a[i][k], h[i][k], mul2(du, *(const f2*)(sB + (t * NP + n0 + k) * 2)));
          y = fma2(h[i + 1][k], *(const f2*)(sC + (t * NP + n0 + k) * 2), y);
        }
        *(f2*)(sY + w * C::SLAB + i * CHN + c) = y;
      }
      float* red = sRed + w * C::RED;
#pragma unroll
      for (int i = RB - 1; i >= 0; --i) {
        const int t = tb + i;
        const f2 dt = *(const f2*)(sDt + t * CHN + c), du = *(const f2*)(sDu + t * CHN + c);
        const f2 dy = *(const f2*)(sDy + t * CHN + c);
        f2 gB = 0, dd = 0;
#pragma unroll
        for (int k = 0; k < NS; ++k) {
          const f2 g = fma2(*(const f2*)(sC + (t * NP + n0 + k) * 2), dy, r[k]);
          const float2 vB = unpack(mul2(du, g)), vC = unpack(mul2(dy, h[i + 1][k]));
          const int v = (i % C::FLUSH * NS + k) * 2;
          red[v * 36 + lane] = vB.x + vB.y;
          red[(v + 1) * 36 + lane] = vC.x + vC.y;
          gB = fma2(g, *(const f2*)(sB + (t * NP + n0 + k) * 2), gB);
          r[k] = mul2(a[i][k], g);
          const f2 gah = mul2(r[k], h[i][k]);
          dd = fma2(gah, A[k], dd);
          dA[k] = fma2(gah, dt, dA[k]);
        }
        *(f2*)(sG + w * C::SLAB + i * CHN + c) = gB;
        *(f2*)(sT + w * C::SLAB + i * CHN + c) = dd;
        if (i % C::FLUSH == 0) {      // two lanes add up one value of the 32 lanes
          __syncwarp();
          const int v = lane >> 1;
          const ulonglong2* m = (const ulonglong2*)(red + v * 36 + (lane & 1) * 16);
          f2 s0 = 0, s1 = 0;
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const ulonglong2 u = m[x];
            s0 = add2(s0, u.x), s1 = add2(s1, u.y);
          }
          const float2 u = unpack(add2(s0, s1));
          float sum = u.x + u.y;
          sum += __shfl_xor_sync(0xffffffffu, sum, 1);
          if ((lane & 1) == 0)
            sBC[((t + v / (2 * NS)) * 2 + v % 2) * NP + n0 + v / 2 % NS] = sum;
          __syncwarp();
        }
      }
      __syncthreads();
      for (int i = w; i < RB; i += S) {
        const int t = tb + i, o = t * CHN + c, po = i * CHN + c;
        f2 y = 0, gB = 0, dd = 0;
#pragma unroll
        for (int x = 0; x < S; ++x) {
          y = add2(y, *(const f2*)(sY + x * C::SLAB + po));
          gB = add2(gB, *(const f2*)(sG + x * C::SLAB + po));
          dd = add2(dd, *(const f2*)(sT + x * C::SLAB + po));
        }
        float2 vy = unpack(y);
        const float2 vg = unpack(gB), vd = unpack(dd);
        const float2 x = *(const float2*)(sX + o), dt = *(const float2*)(sDt + o);
        const float2 dy = *(const float2*)(sDy + o), sl = *(const float2*)(sSl + o);
        const float2 zg = *(const float2*)(sZg + o);
        float2 dd2 = make_float2(fmaf(vg.x, x.x, vd.x * kLn2) * sl.x,
                                 fmaf(vg.y, x.y, vd.y * kLn2) * sl.y);
        float2 du2 = make_float2(fmaf(vg.x, dt.x, skip.x * dy.x), fmaf(vg.y, dt.y, skip.y * dy.y));
        if (t >= rows)      // behind the sequence, whatever the states and their gradients hold
          dd2 = du2 = vy = make_float2(0.f, 0.f);
        dD.x = fmaf(dy.x, x.x, dD.x), dD.y = fmaf(dy.y, x.y, dD.y);
        dbias.x += dd2.x, dbias.y += dd2.y;
        const int64_t tt = t0 + t;
        if (tt < s.length) {
          store_pair(gr.du.at(b, tt) + d0 + c, du2, nc, out_vec);
          store_pair(gr.ddelta.at(b, tt) + d0 + c, dd2, nc, out_vec);
          if (in.z)
            store_pair(gr.dz.at(b, tt) + d0 + c,
                       make_float2(zg.x * fmaf(skip.x, x.x, vy.x), zg.y * fmaf(skip.y, x.y, vy.y)),
                       nc, out_vec);
        }
      }
      __syncthreads();
    }
    // the piece's dB, dC sums over this block's channels
    for (int i = tid; i < CK * 2 * NP; i += THREADS) {
      const int t = i / (2 * NP), k = i / NP % 2, n = i % NP;
      if (t < rows && n < s.states)
        gr.partBC[((((blk * s.batch + b) * s.groups + grp) * s.length + t0 + t) * 2 + k) * s.states +
                  n] = sBC[i];
    }
  }
  // steps past the sequence's last piece
  for (int64_t t = pieces * CK + w; t < s.length; t += S) {
    const float2 zero = make_float2(0.f, 0.f);
    store_pair(gr.du.at(b, t) + d0 + c, zero, nc, out_vec);
    store_pair(gr.ddelta.at(b, t) + d0 + c, zero, nc, out_vec);
    if (in.z) store_pair(gr.dz.at(b, t) + d0 + c, zero, nc, out_vec);
  }
  __syncthreads();
  float* sum = sY;                                 // (warps, 2, channels)
  *(float2*)(sum + (w * 2 + 0) * CHN + c) = dD;
  *(float2*)(sum + (w * 2 + 1) * CHN + c) = dbias;
  __syncthreads();
  float* pa = gr.partA + (b * s.channels + d0) * (s.states + 2);
  for (int i = tid; i < 2 * nch; i += THREADS) {
    const int k = i / nch, cc = i % nch;
    float v = 0.f;
    for (int x = 0; x < S; ++x) v += sum[(x * 2 + k) * CHN + cc];
    pa[cc * (s.states + 2) + s.states + k] = v;
  }
#pragma unroll
  for (int k = 0; k < NS; ++k) {
    const float2 va = unpack(dA[k]), vr = unpack(r[k]);
#pragma unroll
    for (int e = 0; e < 2; ++e)
      if (e < nc && n0 + k < s.states) {
        pa[(c + e) * (s.states + 2) + n0 + k] = e ? va.y : va.x;
        if (gr.dinit)
          gr.dinit[(b * s.channels + d0 + c + e) * s.states + n0 + k] = e ? vr.y : vr.x;
      }
  }
}

// dB and dC (batch, length, groups, N) from the blocks' sums, in block order.
template <class T>
__global__ void sum_bc_kernel(const float* __restrict__ part, T* dB, T* dC,
                              const int32_t* __restrict__ lengths, ScanSizes s, int64_t blocks) {
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  const int64_t per = s.batch * s.groups * s.length * 2 * s.states;
  if (i >= per) return;
  const int n = (int)(i % s.states);
  const bool isC = (i / s.states) % 2;
  int64_t q = i / (2 * s.states);
  const int64_t t = q % s.length;
  q /= s.length;
  const int64_t g = q % s.groups, b = q / s.groups;
  float v = 0.f;
  if (t < scan_length(lengths, b, s.length))
    for (int64_t k = 0; k < blocks; ++k) v += part[k * per + i];
  (isC ? dC : dB)[((b * s.length + t) * s.groups + g) * s.states + n] = from_f<T>(v);
}

// dA, dD and the bias gradient: sums over the batch, in order.
__global__ void sum_params_kernel(const float* __restrict__ part, float* dA, float* dD,
                                  float* dbias, ScanSizes s) {
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  const int64_t w = s.states + 2, per = s.channels * w;
  if (i >= per) return;
  float v = 0.f;
  for (int64_t b = 0; b < s.batch; ++b) v += part[b * per + i];
  const int64_t d = i / w;
  const int n = (int)(i % w);
  if (n < s.states)
    dA[d * s.states + n] = v;
  else if (n == s.states) {
    if (dD) dD[d] = v;
  } else if (dbias) {
    dbias[d] = v;
  }
}

}  // namespace
}  // namespace seq
}  // namespace ferrum

using namespace ferrum;
using namespace ferrum::seq;

extern "C" ferrum_status ferrum_selective_scan_bwd(ferrum_device* dev, const ferrum_scan_args* a,
                                                   void* stream) {
  const char* what = "selective_scan_bwd";
  return guarded(what, [&]() -> ferrum_status {
    if (ferrum_status s = check_scan(dev, a, what, true)) return s;
    if (a->channels == 0) return FERRUM_OK;
    cudaStream_t st = (cudaStream_t)stream;
    const ScanSizes s = scan_sizes(a);
    const int64_t group_blocks = ceil_div(s.per_group, CHN);
    const int64_t blocks = s.batch * s.groups * group_blocks;
    const int64_t bc = s.batch * s.groups * s.length * 2 * s.states;
    const int64_t pa = s.channels * (s.states + 2);
    if (blocks > 0x7fffffff || ceil_div(bc, 256) > 0x7fffffff)
      return invalid(what, "too many blocks for one launch");
    DeviceGuard guard(dev->ordinal);
    if (guard.status() != cudaSuccess) return cuda_error(guard.status(), "cudaSetDevice");
    PoolBuffer wbc(dev, (size_t)(group_blocks * bc) * 4 + 4, st);
    PoolBuffer wa(dev, (size_t)(s.batch * pa) * 4 + 4, st);
    if (wbc.status() != cudaSuccess) return cuda_error(wbc.status(), "workspace");
    if (wa.status() != cudaSuccess) return cuda_error(wa.status(), "workspace");
    return with_dtype(a->dtype, [&](auto tag) -> ferrum_status {
      using T = decltype(tag);
      ScanGrad<T> gr{rows_of<T>(a->dout), rows_of<T>(a->du), rows_of<T>(a->ddelta),
                     rows_of<T>(a->dz), a->dfinal_state, a->saved_states, a->dinitial_state,
                     wbc.as<float>(), wa.as<float>()};
      if (blocks > 0) {
        const int64_t pg = s.groups == 1 ? 0 : s.per_group;
        int unit = std::min(copy_unit<T>(a->u, pg), copy_unit<T>(a->delta));
        unit = std::min(unit, copy_unit<T>(a->dout));
        if (a->z.ptr) unit = std::min(unit, copy_unit<T>(a->z));
        const int bc_unit = std::min(copy_unit<T>(a->B, a->B_group_stride),
                                     copy_unit<T>(a->C, a->C_group_stride));
        int out = std::min(copy_unit<T>(a->du, pg), copy_unit<T>(a->ddelta));
        if (a->z.ptr) out = std::min(out, copy_unit<T>(a->dz));
        ferrum_status r = with_states(s.states, [&](auto n) -> ferrum_status {
          constexpr int NP = decltype(n)::value;
          using C = BwdCfg<T, NP>;
          static std::atomic<uint64_t> done{0};
          cudaError_t e = launch_detail::ensure_smem(scan_bwd_kernel<T, NP>, C::BYTES, done);
          if (e != cudaSuccess) return cuda_error(e, what);
          launch_detail::clear_stale_error();
          scan_bwd_kernel<T, NP><<<(unsigned)blocks, C::THREADS, C::BYTES, st>>>(
              scan_in<T>(a), gr, s, group_blocks, unit, bc_unit,
              s.states == NP && aligned(a->saved_states, 16), out != kCopyScalar);
          return launched(what);
        });
        if (r) return r;
      }
      launch_detail::clear_stale_error();
      if (bc > 0)
        sum_bc_kernel<T><<<(unsigned)ceil_div(bc, 256), 256, 0, st>>>(
            wbc.as<float>(), (T*)a->dB, (T*)a->dC, a->lengths, s, group_blocks);
      sum_params_kernel<<<(unsigned)ceil_div(pa, 256), 256, 0, st>>>(wa.as<float>(), a->dA, a->dD,
                                                                    a->ddelta_bias, s);
      return launched(what);
    });
  });
}
