// RMS norm of every query and key head with the position rotation in the same pass, and its
// gradient (skv_qk_norm_rope, skv_qk_norm_rope_grad).
//
// Per token and head, with x the head's 128 channels:
//   xh = x / sqrt(mean(x^2) + eps),  y = w . xh,  z = R(position) y
// where R turns the first 2 * half channels in pairs by the token's table row.  Backwards, with
// g = dL/dz:
//   dy = R^T g,  dw = sum over rows of dy . xh,  u = w . dy,
//   dx = r u - x r^3 mean(u . x),  r = 1 / sqrt(mean(x^2) + eps).
// A row is 16 lanes of 8 channels, so its sums are four DPP adds and nothing but the weights'
// gradient leaves the row.  Both passes are bound by bytes: q, k (and their gradients) once in and
// once out; four heads of a token share one load of its table row.
#include "skv_rowops.h"

namespace skv {

namespace {

struct QkSide {
  const void* x;
  int64_t sb, st, sh;
  const void* g;  // gradient of the output (backward)
  int64_t gb, gt, gh;
  void* out;  // z, or dx
  int64_t ob, ot, oh;
  const void* w;
  int w_dtype, norm, heads, blocks;  // blocks: groups of kHeadBlock heads
  float eps;
  float* dw_part;  // [workgroups of this side][128], or NULL
  void* dw;
  int dw_dtype;
};

struct QkArgs {
  QkSide q, k;
  const float *cos, *sin;
  int64_t tab_st, tab_rows;
  const void* pos;
  int64_t pos_sb, pos_st, pos0;
  int pos64, half, batch, rows;
  int n_units_q, n_units;  // (token, head block) units of q, and of q and k
  int n_groups_q;          // backward: workgroups of q (the others work on k)
};

__device__ inline int64_t position(const QkArgs& a, int b, int row) {
  if (a.pos == nullptr) return a.pos0 + row;
  const int64_t i = b * a.pos_sb + row * a.pos_st;
  return a.pos0 + (a.pos64 ? static_cast<const int64_t*>(a.pos)[i]
                           : (int64_t)static_cast<const int32_t*>(a.pos)[i]);
}

// grid ceil(n_units / 16), block 256: 16 lanes per unit of kHeadBlock heads of one token, every
// head's load issued before the first is worked on.  4680 tokens of 40 + 40 bf16 heads take 35.1 us, 5.5 TB/s,
// what a large copy reaches and part of the input in the last cache; a few tokens 3.9 us, which is the launch.
template <typename T, bool INTER>
__global__ __launch_bounds__(256) void qk_norm_rope_kernel(QkArgs a) {
  const int lane64 = threadIdx.x & 63;
  int unit = (int)blockIdx.x * 16 + (threadIdx.x >> 4);
  const TurnLane<INTER> lane(a.half, lane64);
  const bool live = unit < a.n_units;
  const bool is_q = !live || unit < a.n_units_q;  // lanes behind the last unit look at q's first
  unit = !live ? 0 : is_q ? unit : unit - a.n_units_q;
  const QkSide& s = is_q ? a.q : a.k;
  const int hb = unit % s.blocks, br = unit / s.blocks;
  const int row = br % a.rows, b = br / a.rows;
  const int h0 = hb * kHeadBlock, c = 8 * (lane64 & 15);
  const T* x = static_cast<const T*>(s.x) + b * s.sb + row * s.st + h0 * s.sh + c;
  Raw8<T> raw[kHeadBlock];
#pragma unroll
  for (int i = 0; i < kHeadBlock; ++i)
    raw[i] = live && h0 + i < s.heads ? Raw8<T>::load(x + i * s.sh) : Raw8<T>::zero();
  Turn<INTER> turn;
  turn.load(a.cos, a.sin, a.tab_st, a.tab_rows, position(a, b, row), lane);
  float w[8], wp[8];
  load_weight8(s.w, s.w_dtype, c, w);
  if constexpr (!INTER) load_weight8(s.w, s.w_dtype, 8 * (lane.partner & 15), wp);
  T* o = static_cast<T*>(s.out) + b * s.ob + row * s.ot + h0 * s.oh + c;
#pragma unroll
  for (int i = 0; i < kHeadBlock; ++i) {
    const Raw8<T> z = norm_turn<T, INTER>(raw[i], s.norm, s.eps, w, wp, turn, lane);
    if (live && h0 + i < s.heads) z.store(o + i * s.oh);
  }
}

// grid: n_groups_q workgroups that walk q's units, the rest k's.  A thread keeps the weight
// gradient of its 8 channels over all its rows; the workgroup's 16 rows of sums meet in LDS and go
// out as one row of partials, which qk_norm_dw_kernel adds in a fixed order.  16380 tokens of 24 + 24 bf16
// heads: 604 MB in 108 us, 5.6 TB/s (the forward pass 67 us, 6.0 TB/s; part of the inputs in the last cache).
template <typename T, bool INTER>
__global__ __launch_bounds__(256) void qk_norm_rope_grad_kernel(QkArgs a) {
  __shared__ float part[16][kHeadDim];
  const int lane64 = threadIdx.x & 63, group = threadIdx.x >> 4;
  const bool is_q = (int)blockIdx.x < a.n_groups_q;
  const QkSide& s = is_q ? a.q : a.k;
  const int wg = is_q ? blockIdx.x : blockIdx.x - a.n_groups_q;
  const int n_wg = is_q ? a.n_groups_q : gridDim.x - a.n_groups_q;
  const int n_units = is_q ? a.n_units_q : a.n_units - a.n_units_q;
  const TurnLane<INTER> lane(a.half, lane64);
  const int c = 8 * (lane64 & 15);
  float w[8], dw[8];
  load_weight8(s.w, s.w_dtype, c, w);
#pragma unroll
  for (int i = 0; i < 8; ++i) dw[i] = 0.0f;
  for (int u0 = wg * 16; u0 < n_units; u0 += n_wg * 16) {  // whole waves: partners shuffle
    const bool live = u0 + group < n_units;
    const int unit = live ? u0 + group : 0;
    const int hb = unit % s.blocks, br = unit / s.blocks;
    const int row = br % a.rows, b = br / a.rows;
    const int h0 = hb * kHeadBlock;
    const T* x = static_cast<const T*>(s.x) + b * s.sb + row * s.st + h0 * s.sh + c;
    const T* g = static_cast<const T*>(s.g) + b * s.gb + row * s.gt + h0 * s.gh + c;
    Raw8<T> xr[kHeadBlock], gr[kHeadBlock];
#pragma unroll
    for (int i = 0; i < kHeadBlock; ++i) {
      const bool there = live && h0 + i < s.heads;
      xr[i] = there ? Raw8<T>::load(x + i * s.sh) : Raw8<T>::zero();
      gr[i] = there ? Raw8<T>::load(g + i * s.gh) : Raw8<T>::zero();
    }
    Turn<INTER> turn;
    turn.load(a.cos, a.sin, a.tab_st, a.tab_rows, position(a, b, row), lane);
    T* o = static_cast<T*>(s.out) + b * s.ob + row * s.ot + h0 * s.oh + c;
#pragma unroll
    for (int i = 0; i < kHeadBlock; ++i) {
      float xf[8], dy[8], dyp[8];
      gr[i].unpack(dy);
      if constexpr (!INTER) gr[i].from_lane(lane.partner).unpack(dyp);
      turn.template apply<true>(dy, dyp, lane);
      const bool there = live && h0 + i < s.heads;
      if (s.norm) {
        xr[i].unpack(xf);
        float ss = 0.0f, ux = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          ss += xf[e] * xf[e];
          ux += dy[e] * w[e] * xf[e];
        }
        const float r = rsqrtf(row_sum(ss) * (1.0f / kHeadDim) + s.eps);
        const float m = row_sum(ux) * (1.0f / kHeadDim) * r * r;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          // a row that is not there adds nothing, whatever its table row holds
          dw[e] += there ? dy[e] * (xf[e] * r) : 0.0f;
          dy[e] = r * (dy[e] * w[e] - xf[e] * m);
        }
      }
      if (there) Raw8<T>::pack(dy).store(o + i * s.oh);
    }
  }
  if (s.dw_part == nullptr) return;  // the same for every thread of the workgroup
#pragma unroll
  for (int i = 0; i < 8; ++i) part[group][c + i] = dw[i];
  __syncthreads();
  if (threadIdx.x < kHeadDim) {
    float t = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; ++i) t += part[i][threadIdx.x];
    s.dw_part[(int64_t)wg * kHeadDim + threadIdx.x] = t;
  }
}

// grid (4, 2): 32 channels of q's or k's weight gradient from the workgroups' partials, in a fixed order
// (2048 rows of partials 4.4 us).
__global__ __launch_bounds__(1024) void qk_norm_dw_kernel(QkArgs a, int n_groups_k) {
  __shared__ float part[128][33];
  const QkSide& s = blockIdx.y == 0 ? a.q : a.k;
  if (s.dw == nullptr) return;
  const int n = blockIdx.y == 0 ? a.n_groups_q : n_groups_k;
  const int c = 4 * (threadIdx.x & 7), j = threadIdx.x >> 3, c0 = 32 * blockIdx.x;
  f32x4 t = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
  for (int i = j; i < n; i += 128)
    t += *reinterpret_cast<const f32x4*>(s.dw_part + (int64_t)i * kHeadDim + c0 + c);
#pragma unroll
  for (int i = 0; i < 4; ++i) part[j][c + i] = t[i];
  __syncthreads();
  // 32 threads a channel, four rows each, then across them
  const int ch = threadIdx.x >> 5, k = threadIdx.x & 31;
  float sum = part[k][ch] + part[k + 32][ch] + part[k + 64][ch] + part[k + 96][ch];
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) sum += __shfl_xor(sum, d, 64);
  if (k == 0) {
    if (s.dw_dtype == SKV_F32) static_cast<float*>(s.dw)[c0 + ch] = sum;
    else if (s.dw_dtype == SKV_BF16) static_cast<bf16*>(s.dw)[c0 + ch] = (bf16)sum;
    else static_cast<f16*>(s.dw)[c0 + ch] = (f16)sum;
  }
}

bool float_dtype(int t) { return t == SKV_F32 || t == SKV_BF16 || t == SKV_F16; }

bool aligned(const void* p, int64_t sb, int64_t st, int64_t sh) {
  return p && reinterpret_cast<uintptr_t>(p) % 16 == 0 && sb >= 0 && st >= 0 && sh >= 0 &&
         sb % 8 == 0 && st % 8 == 0 && sh % 8 == 0;
}

// byte extent [lo, hi) of a [batch][rows][heads][128] view
void extent(const void* p, int64_t sb, int64_t st, int64_t sh, const skv_qk_norm_rope_desc* d,
            int heads, int esz, uintptr_t& lo, uintptr_t& hi) {
  lo = reinterpret_cast<uintptr_t>(p);
  hi = lo + (uintptr_t)esz * ((d->batch - 1) * sb + (d->rows - 1) * st + (heads - 1) * sh + kHeadDim);
}

int check_side(const char* fn, const char* name, const skv_qk_norm_rope_desc* d,
               const skv_norm_side* s, bool grad) {
  if (s->heads <= 0) {
    set_error("%s: %s has %d heads", fn, name, s->heads);
    return SKV_E_ARG;
  }
  if (!aligned(s->x, s->x_sb, s->x_st, s->x_sh) || !aligned(s->out, s->out_sb, s->out_st, s->out_sh) ||
      (grad && !aligned(s->grad, s->grad_sb, s->grad_st, s->grad_sh))) {
    set_error("%s: %s tensors must be 16-byte aligned with non-negative strides that are multiples "
              "of 8 elements", fn, name);
    return SKV_E_ARG;
  }
  if (s->norm && s->weight && (!float_dtype(s->weight_dtype) ||
                               reinterpret_cast<uintptr_t>(s->weight) % 16)) {
    set_error("%s: %s norm weight must be 16-byte aligned f32, bf16 or f16", fn, name);
    return SKV_E_ARG;
  }
  if (s->norm && !(s->eps >= 0.0f)) {
    set_error("%s: %s eps must not be negative", fn, name);
    return SKV_E_ARG;
  }
  if (d->rows > 0 && d->batch > 0) {
    const int esz = d->dtype == SKV_F32 ? 4 : 2;
    uintptr_t xl, xh, ol, oh;
    extent(s->x, s->x_sb, s->x_st, s->x_sh, d, s->heads, esz, xl, xh);
    extent(s->out, s->out_sb, s->out_st, s->out_sh, d, s->heads, esz, ol, oh);
    const bool same = s->x == s->out && s->x_sb == s->out_sb && s->x_st == s->out_st &&
                      s->x_sh == s->out_sh;
    if (!same && xl < oh && ol < xh) {
      set_error("%s: %s out overlaps the input without being the input itself", fn, name);
      return SKV_E_ARG;
    }
  }
  if (grad && s->grad_weight &&
      (!s->norm || !float_dtype(s->grad_weight_dtype) ||
       reinterpret_cast<uintptr_t>(s->grad_weight) % 4)) {
    set_error("%s: %s grad_weight needs a norm and an f32, bf16 or f16 tensor", fn, name);
    return SKV_E_ARG;
  }
  return SKV_OK;
}

QkSide side(const skv_norm_side& s) {
  QkSide o{};
  o.x = s.x, o.sb = s.x_sb, o.st = s.x_st, o.sh = s.x_sh;
  o.g = s.grad, o.gb = s.grad_sb, o.gt = s.grad_st, o.gh = s.grad_sh;
  o.out = s.out, o.ob = s.out_sb, o.ot = s.out_st, o.oh = s.out_sh;
  o.w = s.norm ? s.weight : nullptr, o.w_dtype = s.weight_dtype, o.norm = s.norm != 0;
  o.heads = s.heads, o.blocks = head_blocks(s.heads), o.eps = s.eps;
  o.dw = s.grad_weight, o.dw_dtype = s.grad_weight_dtype;
  return o;
}

// Checks a descriptor and fills the kernels' arguments.
int fill(const char* fn, const skv_qk_norm_rope_desc* d, bool grad, QkArgs* a) {
  clear_error();
  if (!d) {
    set_error("%s: null descriptor", fn);
    return SKV_E_ARG;
  }
  if (d->head_dim != kHeadDim) {
    set_error("%s: head_dim=%d unsupported (built for %d)", fn, d->head_dim, kHeadDim);
    return SKV_E_UNSUPPORTED;
  }
  if (!float_dtype(d->dtype)) {
    set_error("%s: dtype %d unsupported (f32, bf16 or f16)", fn, d->dtype);
    return SKV_E_UNSUPPORTED;
  }
  if (d->batch < 0 || d->rows < 0) {
    set_error("%s: bad sizes (batch=%d rows=%d)", fn, d->batch, d->rows);
    return SKV_E_ARG;
  }
  if (d->half < 0 || d->half > kHeadDim / 2 || d->half % 8 || (d->half > 0) != (d->cos != nullptr) ||
      (d->cos == nullptr) != (d->sin == nullptr)) {
    set_error("%s: the rotation takes cos and sin of 8, 16 .. 64 columns, or neither", fn);
    return SKV_E_ARG;
  }
  if (d->half && (d->table_rows <= 0 || d->table_stride < d->half || d->table_stride % 4 ||
                  reinterpret_cast<uintptr_t>(d->cos) % 16 || reinterpret_cast<uintptr_t>(d->sin) % 16)) {
    set_error("%s: cos / sin need rows, 16-byte aligned pointers and a row stride that is a "
              "multiple of 4 and holds the columns", fn);
    return SKV_E_ARG;
  }
  int st = check_side(fn, "q", d, &d->q, grad);
  if (st == SKV_OK && d->k.heads != 0) st = check_side(fn, "k", d, &d->k, grad);
  if (st != SKV_OK) return st;
  *a = QkArgs{};
  a->q = side(d->q);
  if (d->k.heads) a->k = side(d->k);
  const int64_t tokens = (int64_t)d->batch * d->rows;
  if (tokens >= ((int64_t)1 << 31) || (tokens * (a->q.blocks + (int64_t)a->k.blocks) + 15) / 16 * 256 >= kMaxThreads) {
    set_error("%s: too many rows (batch=%d rows=%d)", fn, d->batch, d->rows);
    return SKV_E_ARG;
  }
  a->cos = d->cos, a->sin = d->sin, a->tab_st = d->table_stride, a->tab_rows = d->table_rows;
  a->pos = d->positions, a->pos_sb = d->pos_sb, a->pos_st = d->pos_st, a->pos0 = d->position0;
  a->pos64 = d->pos_is_int64, a->half = d->half, a->batch = d->batch, a->rows = d->rows;
  a->n_units_q = (int)(tokens * a->q.blocks);
  a->n_units = a->n_units_q + (int)(tokens * a->k.blocks);
  return SKV_OK;
}

template <typename T>
void launch_norm_rope(const QkArgs& a, bool interleaved, hipStream_t s) {
  const dim3 grid((unsigned)((a.n_units + 15) / 16)), block(256);
  if (interleaved) hipLaunchKernelGGL((qk_norm_rope_kernel<T, true>), grid, block, 0, s, a);
  else hipLaunchKernelGGL((qk_norm_rope_kernel<T, false>), grid, block, 0, s, a);
}

template <typename T>
void launch_grad(const QkArgs& a, bool interleaved, int groups, hipStream_t s) {
  const dim3 grid((unsigned)groups), block(256);
  if (interleaved) hipLaunchKernelGGL((qk_norm_rope_grad_kernel<T, true>), grid, block, 0, s, a);
  else hipLaunchKernelGGL((qk_norm_rope_grad_kernel<T, false>), grid, block, 0, s, a);
}

int launched(const char* fn) {
  const hipError_t e = hipGetLastError();
  if (e == hipSuccess) return SKV_OK;
  set_error("%s: launch failed: %s", fn, hipGetErrorString(e));
  return SKV_E_LAUNCH;
}

// Workgroups of one side of the backward pass: 8 per CU keep enough loads in flight to stream, and
// more would only add rows of partial sums.
int grad_groups(int n_units, int share) {
  const int need = (n_units + 15) / 16, most = cu_count() * 8;
  return n_units == 0 ? 0 : need < most * share / 16 ? need : (most * share / 16 > 0 ? most * share / 16 : 1);
}

void grad_grid(const QkArgs& a, int* nq, int* nk) {
  const int share = a.n_units ? (int)(((int64_t)a.n_units_q * 16 + a.n_units / 2) / a.n_units) : 16;
  *nq = grad_groups(a.n_units_q, share < 1 ? 1 : share);
  *nk = grad_groups(a.n_units - a.n_units_q, 16 - share < 1 ? 1 : 16 - share);
}

}  // namespace

}  // namespace skv

using namespace skv;

extern "C" int skv_qk_norm_rope(const skv_qk_norm_rope_desc* d, skv_stream_t stream) {
  QkArgs a;
  const int st = fill("skv_qk_norm_rope", d, false, &a);
  if (st != SKV_OK || a.n_units == 0) return st;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (d->dtype == SKV_F32) launch_norm_rope<float>(a, d->interleaved, s);
  else if (d->dtype == SKV_BF16) launch_norm_rope<bf16>(a, d->interleaved, s);
  else launch_norm_rope<f16>(a, d->interleaved, s);
  return launched("skv_qk_norm_rope");
}

extern "C" int skv_qk_norm_rope_grad_workspace(const skv_qk_norm_rope_desc* d, int64_t* bytes) {
  QkArgs a;
  const int st = fill("skv_qk_norm_rope_grad_workspace", d, true, &a);
  if (st != SKV_OK) return st;
  if (!bytes) {
    set_error("skv_qk_norm_rope_grad_workspace: null result");
    return SKV_E_ARG;
  }
  int nq, nk;
  grad_grid(a, &nq, &nk);
  *bytes = (int64_t)((a.q.dw ? nq : 0) + (a.k.dw ? nk : 0)) * kHeadDim * (int64_t)sizeof(float);
  return SKV_OK;
}

extern "C" int skv_qk_norm_rope_grad(const skv_qk_norm_rope_desc* d, skv_stream_t stream) {
  const char* fn = "skv_qk_norm_rope_grad";
  QkArgs a;
  const int st = fill(fn, d, true, &a);
  if (st != SKV_OK) return st;
  int nq, nk;
  grad_grid(a, &nq, &nk);
  a.n_groups_q = nq;
  const int64_t need = (int64_t)((a.q.dw ? nq : 0) + (a.k.dw ? nk : 0)) * kHeadDim * (int64_t)sizeof(float);
  if (need > 0 && (!d->workspace || d->workspace_bytes < need ||
                   reinterpret_cast<uintptr_t>(d->workspace) % 16)) {
    set_error("%s: needs a 16-byte aligned workspace of %lld bytes", fn, (long long)need);
    return SKV_E_ARG;
  }
  float* ws = static_cast<float*>(d->workspace);
  if (a.q.dw) a.q.dw_part = ws, ws += (int64_t)nq * kHeadDim;
  if (a.k.dw) a.k.dw_part = ws;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (a.n_units > 0) {
    if (d->dtype == SKV_F32) launch_grad<float>(a, d->interleaved, nq + nk, s);
    else if (d->dtype == SKV_BF16) launch_grad<bf16>(a, d->interleaved, nq + nk, s);
    else launch_grad<f16>(a, d->interleaved, nq + nk, s);
    const int e = launched(fn);
    if (e != SKV_OK) return e;
  }
  if (a.q.dw || a.k.dw) {
    hipLaunchKernelGGL(qk_norm_dw_kernel, dim3(4, 2), dim3(1024), 0, s, a, nk);
    return launched(fn);
  }
  return SKV_OK;
}
