// RMSNorm of every q and k head and the rotation by position, in one pass over both:
//
//   t = x * rsqrt(sum_d x_d^2 / D + eps) * gamma_d
//   (t_a, t_b) -> (t_a c - t_b s, t_a s + t_b c)   for the pairs (a, b) among the first 2 P channels,
//                                                  (2j, 2j+1) or (j, j + P), c and s of the token's table row
//
// all in fp32, with one rounding at the end (prep.hip's norm over all heads of a token rounds where the
// DiT's graph does; this one has no graph to follow).
//
// Memory bound: every value is read and written once, and of the tables only the rows used.  A head lies
// in 8, 16 or 32 lanes (D up to 64, 128, 256), 8 channels each, so its sum is a few exchanges between
// lanes and never leaves the wave.  A wave works on one token's heads (several tokens' where they are
// fewer than its lanes hold), each lane on NCH of them: its channel pairs are the same in every head, so
// the angles are loaded once and the NCH reads are in flight together.  2 x 7854 tokens of 24 + 24 heads of 128
// channels: 68 us, 5.7 TB/s (a large copy: 5.1); 8 tokens: 2.9 us in a replayed graph, the launch.
#include "launchers.h"

namespace wan {

namespace {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x8 __attribute__((ext_vector_type(8)));

template <typename T> struct Vec8;
template <> struct Vec8<bf16> { typedef bf16x8 type; };
template <> struct Vec8<_Float16> { typedef f16x8 type; };
template <> struct Vec8<float> { typedef f32x8 type; };

// 8 values of 16-byte aligned memory
template <typename T>
__device__ __forceinline__ void load8(const T* p, float x[8]) {
  typedef typename Vec8<T>::type V __attribute__((aligned(16)));
  const V v = *reinterpret_cast<const V*>(p);
#pragma unroll
  for (int j = 0; j < 8; ++j) x[j] = (float)v[j];
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float x[8]) {
  typedef typename Vec8<T>::type V __attribute__((aligned(16)));
  V v;
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = (T)x[j];
  __builtin_nontemporal_store(v, reinterpret_cast<V*>(p));
}

// The sum over a head's lanes, in all of them: neighbours, pairs and halves of 8 by lane permutations, 16 by
// rotations.
template <int C>
__device__ __forceinline__ float lane_move(float v) {
  return __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(v), C, 0xf, 0xf, true));
}
template <int LPH>
__device__ __forceinline__ float head_sum(float v) {
  if constexpr (LPH == 8) {
    v += lane_move<0xb1>(v);      // the neighbour of 2
    v += lane_move<0x4e>(v);      // the other pair of 4
    v += lane_move<0x141>(v);     // the other four, mirrored
  } else {
    v += lane_move<0x128>(v);
    v += lane_move<0x124>(v);
    v += lane_move<0x122>(v);
    v += lane_move<0x121>(v);
    if constexpr (LPH == 32) v += __shfl_xor(v, 16);
  }
  return v;
}

// LPH lanes a head, NCH heads a lane.
template <typename T, int LPH, int NCH>
__global__ __launch_bounds__(256) void head_norm_kernel(const HeadNormArgs a) {
  typedef typename Vec8<T>::type V __attribute__((aligned(16)));
  const int lane = threadIdx.x & 63;
  const int wave = (int)(row_block(a.grid_x) * 4) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (wave >= a.waves) return;
  const int group = a.by_waves(wave);                 // tokens of one wave
  const int part = wave - group * a.waves_per_token;
  const int slot = lane / LPH, chunk = lane % LPH;
  const int64_t tok = ((int64_t)group << a.token_shift) + (slot >> a.slot_shift);
  const bool live = tok < (int64_t)a.B * a.L && chunk * 8 < a.D;
  const int heads = a.Hq + a.Hk;
  const int per_step = 1 << a.slot_shift;             // heads of a token that a wave works on at once
  const int h0 = part * (per_step * NCH) + (slot & (per_step - 1));
  const int d0 = chunk * 8;
  const int b = live ? a.by_tokens((int)tok) : 0, l = live ? (int)tok - b * a.L : 0;

  V xv[NCH];
#pragma unroll
  for (int i = 0; i < NCH; ++i) {
    const int h = h0 + i * per_step;
    xv[i] = V{};
    if (live && h < heads) {
      const T* p = h < a.Hq ? static_cast<const T*>(a.q) + b * a.q_sb + l * a.q_st + h * a.q_sh
                            : static_cast<const T*>(a.k) + b * a.k_sb + l * a.k_st + (h - a.Hq) * a.k_sh;
      xv[i] = *reinterpret_cast<const V*>(p + d0);
    }
  }
  // this lane's angles: of pairs d0/2 .. +3 (neighbours), or of d0 % P .. +7 (halves)
  const bool turned = a.cos != nullptr && live && d0 < 2 * a.P;
  float c[8] = {}, s[8] = {};
  bool outside = false;
  if (a.cos != nullptr && live) {
    const int row = a.positions != nullptr ? a.positions[tok] : l;
    outside = row < 0 || row >= a.rows;
    if (turned && !outside) {
      const int64_t at = (int64_t)row * a.P;
      if (a.interleaved) {
        const f32x4 c4 = *reinterpret_cast<const f32x4*>(a.cos + at + d0 / 2);
        const f32x4 s4 = *reinterpret_cast<const f32x4*>(a.sin + at + d0 / 2);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          c[j] = c4[j];
          s[j] = s4[j];
        }
      } else {
        const int p0 = d0 < a.P ? d0 : d0 - a.P;
        load8(a.cos + at + p0, c);
        load8(a.sin + at + p0, s);
      }
    }
  }
  V gq = V{}, gk = V{};
  if (chunk * 8 < a.D) {
    gq = *reinterpret_cast<const V*>(static_cast<const T*>(a.gamma_q) + d0);
    gk = *reinterpret_cast<const V*>(static_cast<const T*>(a.gamma_k) + d0);
  }

#pragma unroll
  for (int i = 0; i < NCH; ++i) {
    const int h = h0 + i * per_step;
    float u[8], ss = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      u[j] = (float)xv[i][j];
      ss = fmaf(u[j], u[j], ss);
    }
    ss = head_sum<LPH>(ss);
    const float inv = 1.0f / sqrtf(ss / (float)a.D + a.eps);
#pragma unroll
    for (int j = 0; j < 8; ++j) u[j] = u[j] * inv * (float)(h < a.Hq ? gq[j] : gk[j]);
    if (a.cos != nullptr) {
      if (a.interleaved) {
        if (turned) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float re = u[2 * j], im = u[2 * j + 1];
            u[2 * j] = re * c[j] - im * s[j];
            u[2 * j + 1] = re * s[j] + im * c[j];
          }
        }
      } else {
        // the other half of a pair is P / 8 lanes away, in the same head
        const bool first = d0 < a.P;
        const int other = first ? lane + a.P / 8 : lane - a.P / 8;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float w = __shfl(u[j], other & 63);
          if (turned) u[j] = first ? u[j] * c[j] - w * s[j] : w * s[j] + u[j] * c[j];
        }
      }
      // a position that the tables do not hold: the token's heads are NaN
      if (outside) {
#pragma unroll
        for (int j = 0; j < 8; ++j) u[j] = __builtin_nanf("");
      }
    }
    if (live && h < heads) {
      T* o = h < a.Hq ? static_cast<T*>(a.q_out) + (tok * a.Hq + h) * a.D
                      : static_cast<T*>(a.k_out) + (tok * a.Hk + (h - a.Hq)) * a.D;
      store8(o + d0, u);
    }
  }
}

template <typename T, int LPH, int NCH>
int launch(HeadNormArgs a, hipStream_t s) {
  const HeadNormPlan p = head_norm_plan((int64_t)a.B * a.L, a.Hq + a.Hk, LPH, NCH);
  if (p.waves > 0x7ff00000) return set_error(2, "head_norm: %lld waves is too many", (long long)p.waves);
  a.waves = (int)p.waves;
  a.waves_per_token = p.waves_per_token;
  a.by_waves = FastDiv(p.waves_per_token);
  a.by_tokens = FastDiv(a.L);
  a.slot_shift = p.slot_shift;
  a.token_shift = p.token_shift;
  const RowGrid g = row_grid((p.waves + 3) / 4, 256);
  a.grid_x = g.x;
  hipLaunchKernelGGL((head_norm_kernel<T, LPH, NCH>), dim3(g.x, g.y), dim3(256), 0, s, a);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? 0 : set_error(4, "head_norm launch: %s", hipGetErrorString(e));
}

template <typename T, int LPH>
int launch_lanes(const HeadNormArgs& a, hipStream_t s) {
  switch (head_norm_chunks((int64_t)a.B * a.L, a.Hq + a.Hk, LPH)) {
    case 1: return launch<T, LPH, 1>(a, s);
    case 2: return launch<T, LPH, 2>(a, s);
    case 3: return launch<T, LPH, 3>(a, s);
    default: return launch<T, LPH, 4>(a, s);
  }
}

template <typename T>
int launch_type(const HeadNormArgs& a, hipStream_t s) {
  if (a.D <= 64) return launch_lanes<T, 8>(a, s);
  if (a.D <= 128) return launch_lanes<T, 16>(a, s);
  return launch_lanes<T, 32>(a, s);
}

}  // namespace

int launch_head_norm(const HeadNormArgs& a, int dtype, hipStream_t s) {
  if ((int64_t)a.B * a.L == 0) return 0;
  switch (dtype) {
    case kBF16: return launch_type<bf16>(a, s);
    case kF16: return launch_type<_Float16>(a, s);
    default: return launch_type<float>(a, s);
  }
}

}  // namespace wan
