// Device helpers of the per-head norm and the position rotation: a 16-lane group holds one
// 128-channel head of one token, lane v channels 8v .. 8v + 7.
#pragma once

#include "skv_common.h"

namespace skv {

constexpr int kRowLanes = 16;  // lanes per 128-channel head row
constexpr int kHeadBlock = 4;  // heads of one token that a group works on with one table row
inline int head_blocks(int heads) { return heads / kHeadBlock + (heads % kHeadBlock > 0); }
constexpr int64_t kMaxThreads = (int64_t)1 << 32;  // a launch has fewer


// 8 channels as raw words: 4 of a 16-bit type, 8 of float.
template <typename T>
struct Raw8 {
  static constexpr int kWords = 2 * (int)sizeof(T);
  uint32_t w[kWords];

  __device__ static Raw8 load(const T* p) {
    Raw8 r;
#pragma unroll
    for (int i = 0; i < kWords / 4; ++i) {
      const u32x4 v = reinterpret_cast<const u32x4*>(p)[i];
#pragma unroll
      for (int j = 0; j < 4; ++j) r.w[4 * i + j] = v[j];
    }
    return r;
  }
  // nontemporal: outputs of many tokens do not push out what is still to be read (4680 tokens of 80 heads 45 ->
  // 40 us, the training step of 16380 tokens 203 -> 189; loads marked so as well 42)
  __device__ void store(T* p) const {
#pragma unroll
    for (int i = 0; i < kWords / 4; ++i)
      __builtin_nontemporal_store(u32x4{w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]}, reinterpret_cast<u32x4*>(p) + i);
  }
  __device__ static Raw8 zero() {
    Raw8 r;
#pragma unroll
    for (int i = 0; i < kWords; ++i) r.w[i] = 0u;
    return r;
  }
  __device__ Raw8 from_lane(int lane) const {
    Raw8 r;
#pragma unroll
    for (int i = 0; i < kWords; ++i) r.w[i] = (uint32_t)__shfl((int)w[i], lane, 64);
    return r;
  }
  __device__ void unpack(float (&o)[8]) const {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < 8; ++i) o[i] = __uint_as_float(w[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        typedef T t2 __attribute__((ext_vector_type(2)));
        const t2 p = __builtin_bit_cast(t2, w[i]);
        o[2 * i] = (float)p[0];
        o[2 * i + 1] = (float)p[1];
      }
    }
  }
  // the one rounding of the path: nearest even, to the tensor's type
  __device__ static Raw8 pack(const float (&o)[8]) {
    Raw8 r;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < 8; ++i) r.w[i] = __float_as_uint(o[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        typedef T t2 __attribute__((ext_vector_type(2)));
        t2 p;
        p[0] = (T)o[2 * i];
        p[1] = (T)o[2 * i + 1];
        r.w[i] = __builtin_bit_cast(uint32_t, p);
      }
    }
    return r;
  }
};

// Sum over the 16 lanes of a row, in every lane: four rotations inside the DPP row.
__device__ inline float row_sum(float x) {
#define SKV_ROW_ADD(ctrl) \
  x += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), ctrl, 0xf, 0xf, false))
  SKV_ROW_ADD(0x128);  // row_ror:8
  SKV_ROW_ADD(0x124);
  SKV_ROW_ADD(0x122);
  SKV_ROW_ADD(0x121);
#undef SKV_ROW_ADD
  return x;
}

// 8 norm weights at channel `c`, of any of the three types; ones without a weight tensor.
__device__ inline void load_weight8(const void* w, int dtype, int c, float (&o)[8]) {
  if (w == nullptr) {
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = 1.0f;
  } else if (dtype == SKV_F32) {
    Raw8<float>::load(static_cast<const float*>(w) + c).unpack(o);
  } else if (dtype == SKV_BF16) {
    Raw8<bf16>::load(static_cast<const bf16*>(w) + c).unpack(o);
  } else {
    Raw8<f16>::load(static_cast<const f16*>(w) + c).unpack(o);
  }
}

// Where a lane's channels turn: `half` pairs, (2i, 2i + 1) when INTER, (i, i + half) otherwise.
// half is a multiple of 8, so a lane's 8 channels lie in one half and its partner's in the other.
template <bool INTER>
struct TurnLane {
  bool turns;   // channels below 2 * half
  bool second;  // (not INTER) channels of the second half
  int at;       // first table column of the lane
  int partner;  // lane of the wave that holds the other channel of each pair (self when INTER)

  __device__ TurnLane(int half, int lane64) {
    const int v = lane64 & 15, lanes = half >> 3;
    turns = v < 2 * lanes;
    second = !INTER && turns && v >= lanes;
    if constexpr (INTER) {
      at = 4 * v;
      partner = lane64;
    } else {
      at = 8 * (second ? v - lanes : v);
      partner = turns ? (second ? lane64 - lanes : lane64 + lanes) : lane64;
    }
  }
};

// A token's cos / sin at a lane's channels.
template <bool INTER>
struct Turn {
  static constexpr int kN = INTER ? 4 : 8;
  float c[kN], s[kN];

  // pos outside the table's rows turns by NaN: the row it belongs to says so instead of reading
  // past the table.
  __device__ void load(const float* cos, const float* sin, int64_t stride, int64_t rows, int64_t pos,
                       const TurnLane<INTER>& lane) {
    if (!lane.turns) {
#pragma unroll
      for (int i = 0; i < kN; ++i) c[i] = 1.0f, s[i] = 0.0f;
      return;
    }
    if (pos < 0 || pos >= rows) {
#pragma unroll
      for (int i = 0; i < kN; ++i) c[i] = s[i] = __builtin_nanf("");
      return;
    }
    const f32x4* pc = reinterpret_cast<const f32x4*>(cos + pos * stride + lane.at);
    const f32x4* ps = reinterpret_cast<const f32x4*>(sin + pos * stride + lane.at);
#pragma unroll
    for (int i = 0; i < kN / 4; ++i) {
      const f32x4 a = pc[i], b = ps[i];
#pragma unroll
      for (int j = 0; j < 4; ++j) c[4 * i + j] = a[j], s[4 * i + j] = b[j];
    }
  }

  // y turned by +angle (BACK: by -angle, the transpose); yp holds the partner lane's channels.
  template <bool BACK>
  __device__ void apply(float (&y)[8], const float (&yp)[8], const TurnLane<INTER>& lane) const {
    if (!lane.turns) return;  // untouched, infinities and all
    if constexpr (INTER) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float a = y[2 * i], b = y[2 * i + 1], t = BACK ? -s[i] : s[i];
        y[2 * i] = a * c[i] - b * t;
        y[2 * i + 1] = b * c[i] + a * t;
      }
    } else {
      const bool minus = lane.second == BACK;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float t = minus ? -s[i] : s[i];
        y[i] = y[i] * c[i] + yp[i] * t;
      }
    }
  }
};

// One head row normalised, weighted and turned: w / wp are the weights of the lane's and of its
// partner's channels (their values come from the partner's raw words and the row's own 1 / rms).
template <typename T, bool INTER>
__device__ inline Raw8<T> norm_turn(const Raw8<T>& raw, bool norm, float eps, const float (&w)[8],
                                    const float (&wp)[8], const Turn<INTER>& turn,
                                    const TurnLane<INTER>& lane) {
  float y[8], yp[8];
  raw.unpack(y);
  if constexpr (!INTER) raw.from_lane(lane.partner).unpack(yp);
  if (norm) {
    float ss = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) ss += y[i] * y[i];
    const float r = rsqrtf(row_sum(ss) * (1.0f / kHeadDim) + eps);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      y[i] = y[i] * r * w[i];
      if constexpr (!INTER) yp[i] = yp[i] * r * wp[i];
    }
  }
  turn.template apply<false>(y, yp, lane);
  return Raw8<T>::pack(y);
}

}  // namespace skv
