// The 8-bit key/value cache: rotary embedding + quantisation of new rows into
// their slots, reading rows back, and moving an accepted path's rows.
// (Row format: kvq8.cuh. The attention over it: attention_q8.cu.)
#include <algorithm>
#include <array>

#include "host.cuh"
#include "kvq8.cuh"

namespace ssd {

struct WriteQ8Args {
  const void* q;
  const void* k;
  const void* v;
  int64_t ldq, ldk, ldv;
  int n_q, n_kv, hd;  // n_q: query heads to rotate (0: cache write only)
  const float* cos;
  const float* sin;
  int max_pos, rot, interleaved, kv_shift;
  const int32_t* positions;
  const int32_t* slots;
  uint8_t* kc;
  uint8_t* vc;
  uint8_t* ks;
  uint8_t* vs;
  int64_t head_stride, scale_head_stride;
  int max_slots;
  void* q_out;
  int64_t ldqo;
  uint32_t* status;
};

// Four elements as loaded or stored, and their values.
template <typename T>
struct Quad {
  uint32_t w[sizeof(T)];
};
template <typename T>
__device__ __forceinline__ void quad_values(const Quad<T>& r, float* x) {
#pragma unroll
  for (int i = 0; i < (int)sizeof(T); ++i) {
    if constexpr (sizeof(T) == 2) {
      x[2 * i] = __uint_as_float(r.w[i] << 16);
      x[2 * i + 1] = __uint_as_float(r.w[i] & 0xffff0000u);
    } else {
      x[i] = __uint_as_float(r.w[i]);
    }
  }
}
template <typename T>
__device__ __forceinline__ Quad<T> quad_of(const float* x) {
  Quad<T> r;
#pragma unroll
  for (int i = 0; i < (int)sizeof(T); ++i) {
    if constexpr (sizeof(T) == 2) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
      r.w[i] = *reinterpret_cast<const uint32_t*>(&h);
    } else {
      r.w[i] = __float_as_uint(x[i]);
    }
  }
  return r;
}
template <typename T>
__device__ __forceinline__ Quad<T> load_quad(const T* p) {
  Quad<T> r;
  if constexpr (sizeof(T) == 2) {
    const uint2 u = *reinterpret_cast<const uint2*>(p);
    r.w[0] = u.x, r.w[1] = u.y;
  } else {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    r.w[0] = u.x, r.w[1] = u.y, r.w[2] = u.z, r.w[3] = u.w;
  }
  return r;
}
template <typename T>
__device__ __forceinline__ void store_quad(T* p, const Quad<T>& r) {
  if constexpr (sizeof(T) == 2)
    *reinterpret_cast<uint2*>(p) = make_uint2(r.w[0], r.w[1]);
  else
    *reinterpret_cast<uint4*>(p) = make_uint4(r.w[0], r.w[1], r.w[2], r.w[3]);
}
template <typename T, bool VEC>
__device__ __forceinline__ void store8(T* p, const float* x) {
  if constexpr (!VEC) {
#pragma unroll
    for (int i = 0; i < 8; ++i) p[i] = from_f32<T>(x[i]);
  } else if constexpr (sizeof(T) == 2) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  } else {
    reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
  }
}

// One token's rows: query heads rotated into q_out, key heads rotated and
// quantised, value heads quantised into cache slot slots[t].
//   (a, b) -> (a cos - b sin, b cos + a sin) for the pair (i, i + rot / 2)
//   (half layout) or (2i, 2i + 1) (interleaved), i < rot / 2; elements from
//   rot on pass through. Products and sums round one by one, as the formula
//   written out does, so that the codes do not depend on contraction.
// A row is LPR lanes x 4 pairs: a lane holds both elements of its pairs, so
// that nothing is read twice and a row may be rotated in place, and keeps its
// 4 cos / sin for all rows of the token. U passes of query rows and one of key
// and value rows are loaded before the position is known. VEC: rows and tables
// in aligned vectors (rot a multiple of 8).
// Bound by bytes, 2 H hd + 2 Hkv hd elements and the codes of each token, once
// the instructions are few (4096 tokens of 64 + 8 + 8 heads of 128, 178 MB, 27 us at
// the copy rate: 32 us; lanes of 8 neighbouring elements that also read their
// partners issued 1.6 times as many and took 47). Five CTAs per SM want 48
// registers: U = 1 with six 34 us, U = 2 with four 34, U = 4 with two 48.
// T: of the rows. TO: of q_out, T or bf16 of fp32 rows (a projection's accumulators:
// the rotated query is rounded once).
template <typename T, typename TO, int LPR, bool INTER, bool VEC>
__global__ void __launch_bounds__(256, VEC && sizeof(T) == 2 ? 5 : 3) rope_kv_write_q8_kernel(const WriteQ8Args a) {
  constexpr int RPC = 256 / LPR;  // rows per pass of the CTA
  constexpr int U = 2;
  pdl_wait();
  pdl_trigger();
  const int t = blockIdx.x;
  const int l = threadIdx.x % LPR, sub = threadIdx.x / LPR;
  const bool on = 8 * l < a.hd;
  const int half = a.rot >> 1;
  const int slot = a.slots[t];
  int pos = a.rot ? a.positions[t] : 0;
  // Pair p = 4 l + j: elements (p, p + half), or (2p, 2p + 1) if interleaved or
  // not rotated. VEC: the quads at lo and hi.
  const bool split = !INTER && 4 * l < half;
  const uint32_t lo = split ? 4 * l : 8 * l, hi = split ? half + 4 * l : 8 * l + 4;
  auto first_of = [&](int p) { return !INTER && p < half ? p : 2 * p; };
  auto second_of = [&](int p) { return !INTER && p < half ? p + half : 2 * p + 1; };
  // x[0 .. 3], x[4 .. 7]: the quads, or without VEC the pairs' first and second elements
  struct Raw {
    Quad<T> q[2];
  };
  auto load = [&](const T* src, uint32_t at) {  // the row at element `at` of src
    Raw r;
    if constexpr (!VEC) {
      T* e = reinterpret_cast<T*>(r.q);
#pragma unroll
      for (int j = 0; j < 4; ++j) e[j] = src[at + first_of(4 * l + j)], e[4 + j] = src[at + second_of(4 * l + j)];
    } else if constexpr (INTER && sizeof(T) == 2) {
      const uint4 w = *reinterpret_cast<const uint4*>(src + (at + lo));
      r.q[0].w[0] = w.x, r.q[0].w[1] = w.y, r.q[1].w[0] = w.z, r.q[1].w[1] = w.w;
    } else {
      r.q[0] = load_quad(src + (at + lo));
      r.q[1] = load_quad(src + (at + hi));
    }
    return r;
  };
  // Passes over the query rows and then the key and value rows (r < n_kv: key),
  // pass i by the CTA i % gridDim.y (kv_shift: the query rows' passes % gridDim.y).
  // The loads of the first ones come first.
  const int step = gridDim.y * RPC;
  int rq = blockIdx.y * RPC + sub;
  int rkv = ((int)blockIdx.y - a.kv_shift + ((int)blockIdx.y < a.kv_shift ? (int)gridDim.y : 0)) * RPC + sub;
  // (a token's own offsets are 32-bit: the entry point checks)
  const T* q_src = static_cast<const T*>(a.q) + (int64_t)t * a.ldq;
  TO* q_dst = static_cast<TO*>(a.q_out) + (int64_t)t * a.ldqo;
  auto load_kv = [&](int r) {
    const T* src = r < a.n_kv ? static_cast<const T*>(a.k) + (int64_t)t * a.ldk : static_cast<const T*>(a.v) + (int64_t)t * a.ldv;
    return load(src, (r < a.n_kv ? r : r - a.n_kv) * a.hd);
  };
  Raw kv{}, q[U];
  if (on && rkv < 2 * a.n_kv) kv = load_kv(rkv);
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (on && rq + u * step < a.n_q) q[u] = load(q_src, (rq + u * step) * a.hd);
  const bool slot_ok = slot >= 0 && slot < a.max_slots;
  if (a.rot && (pos < 0 || pos >= a.max_pos)) {
    if (threadIdx.x == 0 && blockIdx.y == 0) report_error(a.status, kErrBadIndex);
    pos = 0;
  }
  if (!slot_ok && threadIdx.x == 0 && blockIdx.y == 0) report_error(a.status, kErrBadIndex);
  const bool turns = on && 4 * l < half;
  float c[4] = {}, s[4] = {};
  if (turns) {
    const int64_t at = (int64_t)pos * half + 4 * l;
    if constexpr (VEC) {
      const float4 c4 = *reinterpret_cast<const float4*>(a.cos + at), s4 = *reinterpret_cast<const float4*>(a.sin + at);
      c[0] = c4.x, c[1] = c4.y, c[2] = c4.z, c[3] = c4.w;
      s[0] = s4.x, s[1] = s4.y, s[2] = s4.z, s[3] = s4.w;
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (4 * l + j < half) c[j] = a.cos[at + j], s[j] = a.sin[at + j];
    }
  }
  auto values = [&](const Raw& r, bool turn, float* x) {
    quad_values<T>(r.q[0], x);
    quad_values<T>(r.q[1], x + 4);
    if (!turn) return;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float& xa = VEC && INTER ? x[2 * j] : x[j];
      float& xb = VEC && INTER ? x[2 * j + 1] : x[4 + j];
      const float va = xa, vb = xb;
      if (VEC || 4 * l + j < half) {
        xa = __fsub_rn(__fmul_rn(va, c[j]), __fmul_rn(vb, s[j]));
        xb = __fadd_rn(__fmul_rn(vb, c[j]), __fmul_rn(va, s[j]));
      }
    }
  };
  while (rkv - sub < 2 * a.n_kv) {  // uniform
    const bool live = on && rkv < 2 * a.n_kv, is_v = rkv >= a.n_kv;
    const int head = is_v ? rkv - a.n_kv : rkv;
    float x[8] = {};
    if (live) values(kv, turns && !is_v, x);
    float amax = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float m = fabsf(x[j]);
      amax = m <= 3.402823466e38f ? fmaxf(amax, m) : amax;  // Inf and NaN do not set the scale
    }
#pragma unroll
    for (int o = LPR / 2; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    if (live && slot_ok) {
      const int byte = q8_scale_byte(amax);
      const float inv = q8_inv_scale(byte);
      const uint32_t c0 = q8_pack4(x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv);
      const uint32_t c1 = q8_pack4(x[4] * inv, x[5] * inv, x[6] * inv, x[7] * inv);
      uint8_t* dst = (is_v ? a.vc : a.kc) + (int64_t)head * a.head_stride + (int64_t)slot * a.hd;
      if constexpr (!VEC) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          dst[first_of(4 * l + j)] = static_cast<uint8_t>(c0 >> (8 * j));
          dst[second_of(4 * l + j)] = static_cast<uint8_t>(c1 >> (8 * j));
        }
      } else if constexpr (INTER) {
        *reinterpret_cast<uint2*>(dst + lo) = make_uint2(c0, c1);
      } else {
        *reinterpret_cast<uint32_t*>(dst + lo) = c0;
        *reinterpret_cast<uint32_t*>(dst + hi) = c1;
      }
      if (l == 0) (is_v ? a.vs : a.ks)[(int64_t)head * a.scale_head_stride + slot] = static_cast<uint8_t>(byte);
    }
    rkv += step;
    if (on && rkv < 2 * a.n_kv) kv = load_kv(rkv);
  }
  if (!on) return;
  for (; rq < a.n_q; rq += U * step) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (rq + u * step >= a.n_q) break;
      float x[8];
      values(q[u], turns, x);
      const uint32_t at = (rq + u * step) * a.hd;
      if constexpr (!VEC) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          q_dst[at + first_of(4 * l + j)] = from_f32<TO>(x[j]);
          q_dst[at + second_of(4 * l + j)] = from_f32<TO>(x[4 + j]);
        }
      } else {
        const Quad<TO> y0 = quad_of<TO>(x), y1 = quad_of<TO>(x + 4);
        if constexpr (INTER && sizeof(TO) == 2) {
          *reinterpret_cast<uint4*>(q_dst + (at + lo)) = make_uint4(y0.w[0], y0.w[1], y1.w[0], y1.w[1]);
        } else {
          store_quad(q_dst + (at + lo), y0);
          store_quad(q_dst + (at + hi), y1);
        }
      }
      if (rq + (u + U) * step < a.n_q) q[u] = load(q_src, (rq + (u + U) * step) * a.hd);
    }
  }
}

// Rows of the cache as values: k_out / v_out [N, n_kv * hd], value =
// code * 2^e rounded to T (exact for bf16 and fp32). Bound by bytes: hd + 1
// read and hd * sizeof(T) written per row. A lane converts 16 codes.
struct ReadQ8Args {
  const uint8_t* kc;
  const uint8_t* vc;
  const uint8_t* ks;
  const uint8_t* vs;
  int64_t head_stride, scale_head_stride;
  int n_kv, hd, max_slots;
  const int32_t* slots;
  int64_t first, n;
  void* k_out;
  void* v_out;
  int64_t ldk, ldv;
  uint32_t* status;
};

template <typename T, bool VEC>
__global__ void __launch_bounds__(256) kv_read_q8_kernel(const ReadQ8Args a) {
  pdl_wait();
  pdl_trigger();
  const int cpr = a.hd >> 4;  // 16-code chunks per row
  const int64_t per_slot = (int64_t)a.n_kv * cpr;
  const int64_t total = a.n * per_slot;
  const uint8_t* codes = blockIdx.y ? a.vc : a.kc;
  const uint8_t* scales = blockIdx.y ? a.vs : a.ks;
  T* out = static_cast<T*>(blockIdx.y ? a.v_out : a.k_out);
  const int64_t ldo = blockIdx.y ? a.ldv : a.ldk;
  if (!out) return;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t n = i / per_slot;
    const int rest = (int)(i - n * per_slot);
    const int head = rest / cpr, ch = rest - head * cpr;
    const int64_t slot = a.slots ? a.slots[n] : a.first + n;
    uint4 u = make_uint4(0, 0, 0, 0);
    float sc = 0.f;
    if (slot >= 0 && slot < a.max_slots) {
      u = *reinterpret_cast<const uint4*>(codes + (int64_t)head * a.head_stride + slot * a.hd + ch * 16);
      sc = q8_scale(scales[(int64_t)head * a.scale_head_stride + slot]);
    } else if (rest == 0) {
      report_error(a.status, kErrBadIndex);
    }
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
    float x[16];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 lo = q8_unpack2(w[j]), hi = q8_unpack2(w[j] >> 16);
      x[4 * j] = lo.x * sc;
      x[4 * j + 1] = lo.y * sc;
      x[4 * j + 2] = hi.x * sc;
      x[4 * j + 3] = hi.y * sc;
    }
    T* dst = out + n * ldo + (int64_t)head * a.hd + ch * 16;
    store8<T, VEC>(dst, x);
    store8<T, VEC>(dst + 8, x + 8);
  }
}

// keep_positions for the 8-bit cache: one thread per (layer, K/V, head,
// 16-code chunk) and one per row's scale bytes; each reads all kept slots
// before it writes (as kv_compact_kernel).
__global__ void __launch_bounds__(256)
    kv_compact_q8_kernel(uint8_t* codes, uint8_t* scales, int64_t n_layers, int64_t layer_stride, int64_t kv_stride,
                         int64_t head_stride, int64_t s_layer_stride, int64_t s_kv_stride, int64_t s_head_stride,
                         int n_kv, int hd, int max_slots, const int32_t* start, const int32_t* keep_slots,
                         const int32_t* n_keep, int max_keep, uint32_t* status) {
  constexpr int kMaxKeep = 32;
  pdl_wait();
  pdl_trigger();
  const int parts = hd / 16 + 1;
  const int64_t tid = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (tid >= n_layers * 2 * n_kv * parts) return;
  const int want = *n_keep;
  const int nk = min(min(want, max_keep), kMaxKeep);
  const int s0 = start[0];
  bool bad = want < 0 || want > max_keep || s0 < 0 || s0 + nk > max_slots;
  for (int j = 0; j < nk && !bad; ++j) bad = keep_slots[j] < 0 || keep_slots[j] >= max_slots;
  if (bad) {
    if (tid == 0) report_error(status, kErrBadIndex);
    return;
  }
  const int part = (int)(tid % parts);
  const int64_t row = tid / parts;
  const int head = (int)(row % n_kv);
  const int kv = (int)(row / n_kv % 2);
  const int64_t layer = row / n_kv / 2;
  if (part < parts - 1) {
    uint8_t* base = codes + layer * layer_stride + kv * kv_stride + head * head_stride + part * 16;
    uint4 buf[kMaxKeep];
#pragma unroll
    for (int j = 0; j < kMaxKeep; ++j)
      if (j < nk) buf[j] = *reinterpret_cast<const uint4*>(base + (int64_t)keep_slots[j] * hd);
#pragma unroll
    for (int j = 0; j < kMaxKeep; ++j)
      if (j < nk && keep_slots[j] != s0 + j) *reinterpret_cast<uint4*>(base + (int64_t)(s0 + j) * hd) = buf[j];
  } else {
    uint8_t* base = scales + layer * s_layer_stride + kv * s_kv_stride + head * s_head_stride;
    uint8_t buf[kMaxKeep];
#pragma unroll
    for (int j = 0; j < kMaxKeep; ++j)
      if (j < nk) buf[j] = base[keep_slots[j]];
#pragma unroll
    for (int j = 0; j < kMaxKeep; ++j)
      if (j < nk && keep_slots[j] != s0 + j) base[s0 + j] = buf[j];
  }
}

static bool aligned16(const void* p, int64_t ld_bytes) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && ld_bytes % 16 == 0;
}

// Checks shared by the entry points over one layer of the cache.
int check_kv_q8(const SsdKvQ8* c, const char* who) {
  if (!c || !c->k || !c->v || !c->k_scale || !c->v_scale) return fail(SSD_ERR_INVALID, "%s: NULL cache", who);
  if (c->n_kv_heads <= 0 || c->max_slots <= 0 || c->head_dim <= 0)
    return fail(SSD_ERR_INVALID, "%s: bad cache shape", who);
  if (c->head_dim % 16 || c->head_dim > 128)
    return fail(SSD_ERR_UNSUPPORTED, "%s: head_dim must be a multiple of 16 up to 128", who);
  if (c->max_slots > kQ8MaxSlots) return fail(SSD_ERR_UNSUPPORTED, "%s: too many slots", who);
  if (c->head_stride < c->max_slots * c->head_dim || c->scale_head_stride < c->max_slots)
    return fail(SSD_ERR_INVALID, "%s: cache heads overlap", who);
  if (!aligned16(c->k, c->head_stride) || !aligned16(c->v, c->head_stride))
    return fail(SSD_ERR_INVALID, "%s: cache rows must be 16-byte aligned", who);
  return SSD_OK;
}

// Whether blocks of `extent` bytes at the given strides (of layers, K / V and
// heads, in any order of size) overlap. A dimension of one has no stride.
static bool blocks_overlap(int64_t extent, std::array<std::pair<int64_t, int64_t>, 3> dims) {
  std::sort(dims.begin(), dims.end());
  __int128 end = extent;  // bytes from the first block's start to the last one's end so far
  for (const auto& [stride, n] : dims) {
    if (n == 1) continue;
    if (stride < end) return true;
    end += static_cast<__int128>(stride) * (n - 1);
  }
  return false;
}

template <typename T, typename TO, bool INTER, bool VEC>
int launch_write_q8(WriteQ8Args& a, int64_t T_rows, cudaStream_t stream) {
  const int lanes = a.hd / 8;
  auto go = [&](auto kern, int lpr) {
    // Few tokens: spread a token's rows over CTAs (one pass each) until the
    // SMs are covered; many tokens: one CTA walks all rows of its token and
    // reuses the cos / sin registers.
    const int rpc = 256 / lpr;
    const int q_passes = (a.n_q + rpc - 1) / rpc;
    int64_t gy = q_passes + (2 * a.n_kv + rpc - 1) / rpc;
    const int64_t cover = (2 * device_sms() + T_rows - 1) / T_rows;
    if (gy > cover) gy = cover;
    a.kv_shift = (int)(q_passes % gy);
    return launch_kernel("rope_kv_write_q8_kernel", kern, dim3((unsigned)T_rows, (unsigned)gy), dim3(256), 0, stream,
                         1, 1, a);
  };
  if (lanes <= 2) return go(rope_kv_write_q8_kernel<T, TO, 2, INTER, VEC>, 2);
  if (lanes <= 4) return go(rope_kv_write_q8_kernel<T, TO, 4, INTER, VEC>, 4);
  if (lanes <= 8) return go(rope_kv_write_q8_kernel<T, TO, 8, INTER, VEC>, 8);
  return go(rope_kv_write_q8_kernel<T, TO, 16, INTER, VEC>, 16);
}
template <typename T, typename TO>
int launch_write_q8(WriteQ8Args& a, bool vec, int64_t T_rows, cudaStream_t stream) {
  if (a.interleaved)
    return vec ? launch_write_q8<T, TO, true, true>(a, T_rows, stream)
               : launch_write_q8<T, TO, true, false>(a, T_rows, stream);
  return vec ? launch_write_q8<T, TO, false, true>(a, T_rows, stream)
             : launch_write_q8<T, TO, false, false>(a, T_rows, stream);
}

}  // namespace ssd

using namespace ssd;

extern "C" {

int ssd_rope_kv_write_q8(const void* q, int64_t ldq, const void* k, int64_t ldk, const void* v, int64_t ldv, int64_t T,
                         int64_t n_heads, const float* rope_cos, const float* rope_sin, int64_t max_pos,
                         int64_t rot_dim, int interleaved, const int32_t* positions, const int32_t* slots,
                         const SsdKvQ8* cache, void* q_out, int64_t ldqo, int dtype, uint32_t* status, void* stream) {
  const char* who = "ssd_rope_kv_write_q8";
  if (const int rc = check_kv_q8(cache, who)) return rc;
  if (T <= 0 || T > INT32_MAX) return fail(SSD_ERR_INVALID, "%s: T must be positive", who);
  if (!k || !v || !slots) return fail(SSD_ERR_INVALID, "%s: NULL k, v or slots", who);
  if (q && (!q_out || n_heads <= 0)) return fail(SSD_ERR_INVALID, "%s: q needs q_out and n_heads", who);
  const int64_t hd = cache->head_dim;
  if ((q && n_heads >= (1 << 30) / hd) || cache->n_kv_heads >= (1 << 30) / hd)
    return fail(SSD_ERR_UNSUPPORTED, "%s: rows too long", who);
  if (rot_dim < 0 || rot_dim > hd || (rot_dim & 1))
    return fail(SSD_ERR_INVALID, "%s: rot_dim must be even, 0 .. head_dim", who);
  if (rot_dim && (!rope_cos || !rope_sin || !positions || max_pos <= 0))
    return fail(SSD_ERR_INVALID, "%s: rotation needs tables and positions", who);
  const int out_dtype = dtype & ~SSD_ROWS_F32;
  if (out_dtype != SSD_F32 && out_dtype != SSD_BF16) return fail(SSD_ERR_UNSUPPORTED, "%s: dtype %d", who, dtype);
  const bool rows_f32 = out_dtype == SSD_F32 || (dtype & SSD_ROWS_F32);
  if (q && q == q_out && rows_f32 && out_dtype == SSD_BF16)
    return fail(SSD_ERR_INVALID, "%s: fp32 rows cannot be rotated in place into bf16", who);
  if (T > 1 && ((q && (ldq < n_heads * hd || ldqo < n_heads * hd)) || ldk < cache->n_kv_heads * hd ||
                ldv < cache->n_kv_heads * hd))
    return fail(SSD_ERR_INVALID, "%s: rows overlap", who);
  WriteQ8Args a{};
  a.q = q;
  a.k = k;
  a.v = v;
  a.ldq = ldq;
  a.ldk = ldk;
  a.ldv = ldv;
  a.n_q = q ? (int)n_heads : 0;
  a.n_kv = (int)cache->n_kv_heads;
  a.hd = (int)hd;
  a.cos = rope_cos;
  a.sin = rope_sin;
  a.max_pos = (int)(max_pos > INT32_MAX ? INT32_MAX : max_pos);
  a.rot = (int)rot_dim;
  a.interleaved = interleaved ? 1 : 0;
  a.positions = positions;
  a.slots = slots;
  a.kc = static_cast<uint8_t*>(cache->k);
  a.vc = static_cast<uint8_t*>(cache->v);
  a.ks = cache->k_scale;
  a.vs = cache->v_scale;
  a.head_stride = cache->head_stride;
  a.scale_head_stride = cache->scale_head_stride;
  a.max_slots = (int)cache->max_slots;
  a.q_out = q_out;
  a.ldqo = ldqo;
  a.status = status;
  const int64_t es = rows_f32 ? 4 : 2, es_out = out_dtype == SSD_F32 ? 4 : 2;
  const bool vec = rot_dim % 8 == 0 && aligned16(rope_cos, 0) && aligned16(rope_sin, 0) && aligned16(k, ldk * es) &&
                   aligned16(v, ldv * es) &&
                   (!q || (aligned16(q, ldq * es) && aligned16(q_out, ldqo * es_out)));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (out_dtype == SSD_F32) return launch_write_q8<float, float>(a, vec, T, s);
  return rows_f32 ? launch_write_q8<float, bf16>(a, vec, T, s) : launch_write_q8<bf16, bf16>(a, vec, T, s);
}

int ssd_kv_read_q8(const SsdKvQ8* cache, const int32_t* slots, int64_t first, int64_t n, void* k_out, int64_t ldk,
                   void* v_out, int64_t ldv, int dtype, uint32_t* status, void* stream) {
  const char* who = "ssd_kv_read_q8";
  if (const int rc = check_kv_q8(cache, who)) return rc;
  if (n <= 0) return fail(SSD_ERR_INVALID, "%s: n must be positive", who);
  if (!k_out && !v_out) return fail(SSD_ERR_INVALID, "%s: NULL k_out and v_out", who);
  if (!slots && (first < 0 || first > cache->max_slots || n > cache->max_slots - first))
    return fail(SSD_ERR_INVALID, "%s: slots outside the cache", who);
  if (dtype != SSD_F32 && dtype != SSD_BF16) return fail(SSD_ERR_UNSUPPORTED, "%s: dtype %d", who, dtype);
  const int64_t width = cache->n_kv_heads * cache->head_dim;
  if (n > 1 && ((k_out && ldk < width) || (v_out && ldv < width)))
    return fail(SSD_ERR_INVALID, "%s: rows overlap", who);
  ReadQ8Args a{};
  a.kc = static_cast<const uint8_t*>(cache->k);
  a.vc = static_cast<const uint8_t*>(cache->v);
  a.ks = cache->k_scale;
  a.vs = cache->v_scale;
  a.head_stride = cache->head_stride;
  a.scale_head_stride = cache->scale_head_stride;
  a.n_kv = (int)cache->n_kv_heads;
  a.hd = (int)cache->head_dim;
  a.max_slots = (int)cache->max_slots;
  a.slots = slots;
  a.first = first;
  a.n = n;
  a.k_out = k_out;
  a.v_out = v_out;
  a.ldk = ldk;
  a.ldv = ldv;
  a.status = status;
  const int64_t es = dtype == SSD_F32 ? 4 : 2;
  const bool vec = (!k_out || aligned16(k_out, ldk * es)) && (!v_out || aligned16(v_out, ldv * es));
  const int64_t total = n * (width / 16);
  int64_t blocks = (total + 255) / 256;
  const int64_t most = 8LL * device_sms();
  if (blocks > most) blocks = most;
  const dim3 grid((unsigned)blocks, 2);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  auto go = [&](auto kern) { return launch_kernel("kv_read_q8_kernel", kern, grid, dim3(256), 0, s, 1, 1, a); };
  if (dtype == SSD_F32) return vec ? go(kv_read_q8_kernel<float, true>) : go(kv_read_q8_kernel<float, false>);
  return vec ? go(kv_read_q8_kernel<bf16, true>) : go(kv_read_q8_kernel<bf16, false>);
}

int ssd_kv_compact_q8(void* codes, uint8_t* scales, int64_t n_layers, int64_t layer_stride, int64_t kv_stride,
                      int64_t head_stride, int64_t scale_layer_stride, int64_t scale_kv_stride,
                      int64_t scale_head_stride, int64_t n_kv_heads, int64_t head_dim, int64_t max_slots,
                      const int32_t* start, const int32_t* keep_slots, const int32_t* n_keep, int64_t max_keep,
                      uint32_t* status, void* stream) {
  const char* who = "ssd_kv_compact_q8";
  if (max_keep <= 0 || max_keep > 32) return fail(SSD_ERR_UNSUPPORTED, "%s: max_keep must be 1..32", who);
  if (!codes || !scales || !start || !keep_slots || !n_keep) return fail(SSD_ERR_INVALID, "%s: NULL argument", who);
  if (n_layers <= 0 || n_kv_heads <= 0 || max_slots <= 0 || max_slots > kQ8MaxSlots)
    return fail(SSD_ERR_INVALID, "%s: bad cache shape", who);
  if (head_dim <= 0 || head_dim % 16 || head_dim > 128)
    return fail(SSD_ERR_UNSUPPORTED, "%s: head_dim must be a multiple of 16 up to 128", who);
  if (!aligned16(codes, head_stride) || kv_stride % 16 || layer_stride % 16)
    return fail(SSD_ERR_INVALID, "%s: cache rows must be 16-byte aligned", who);
  if (blocks_overlap(max_slots * head_dim, {{{layer_stride, n_layers}, {kv_stride, 2}, {head_stride, n_kv_heads}}}) ||
      blocks_overlap(max_slots, {{{scale_layer_stride, n_layers}, {scale_kv_stride, 2}, {scale_head_stride, n_kv_heads}}}))
    return fail(SSD_ERR_INVALID, "%s: cache layers, K and V or heads overlap", who);
  const int64_t total = n_layers * 2 * n_kv_heads * (head_dim / 16 + 1);
  return launch_kernel("kv_compact_q8_kernel", kv_compact_q8_kernel, dim3((unsigned)((total + 255) / 256)), dim3(256),
                       0, static_cast<cudaStream_t>(stream), 1, 1, static_cast<uint8_t*>(codes), scales, n_layers,
                       layer_stride, kv_stride, head_stride, scale_layer_stride, scale_kv_stride, scale_head_stride,
                       (int)n_kv_heads, (int)head_dim, (int)max_slots, start, keep_slots, n_keep, (int)max_keep,
                       status);
}

}  // extern "C"
