// Tree attention over the 8-bit key/value cache (row format: kvq8.cuh).
//
// Query row r = t * G + g (token t, head g of the KV head's group) attends
// the slots [prefix_start[t], prefix_len[t]) and slot spec_base + j for every
// set bit j of token t's mask; a row that sees nothing gives zeros.
//   s = (q . k8) 2^ek / sqrt(hd),  o = sum p 2^ev v8 / sum p,  p = 2^(s log2 e - m)
#include "host.cuh"
#include "kvq8.cuh"

namespace ssd {

int check_kv_q8(const SsdKvQ8* c, const char* who);  // kvq8.cu

constexpr int kAttnQ8CounterBase = 49152;  // counter slots of the attention kernels in a workspace
constexpr int kAttnQ8MaxBlocks = 16384;
constexpr int kAttnQ8MaxWords = 4;         // mask words per token

struct AttnQ8Args {
  const void* q;
  int64_t ldq;
  int T, G, M;  // tokens, query heads per KV head, T * G query rows per KV head
  int n_kv, hd;
  const uint8_t* kc;
  const uint8_t* vc;
  const uint8_t* ks;
  const uint8_t* vs;
  int64_t head_stride, scale_head_stride;
  int kv_end;  // slots the call may attend: [0, kv_end)
  const int32_t* prefix_len;
  const int32_t* prefix_start;
  const int32_t* spec_base;
  const uint64_t* mask;
  int mask_words;
  int n_splits, tiles;  // key slices; row tiles per KV head
  void* out;
  int64_t ldo;
  float* part;
  uint32_t* counters;
  uint32_t* status;
  float scale;
};

// ------------------------------------------------------------- CUDA cores
// fp32 queries (the exact tier) and head sizes other than 64 and 128. A CTA =
// one KV head x 32 query rows x one slice of the live key range: 8 warps x 4
// rows, keys staged 64 at a time as fp32 in shared memory. Scores: a lane owns
// keys lane and lane + 32 (float4 reads, row pitch hd + 4 floats: conflict
// free); outputs: a lane owns dims lane, lane + 32, ... Softmax statistics and
// accumulators are fp32. Slices write (max, sum, acc) records; the last CTA of
// a row tile merges them in slice order.
constexpr int kSimtWarps = 8;
constexpr int kSimtRows = 32;   // query rows per CTA
constexpr int kSimtKeys = 64;   // keys per block

__host__ __device__ constexpr int simt_q8_smem(int hd) {
  return (2 * kSimtKeys * (hd + 4) + kSimtRows * hd + kSimtWarps * kSimtKeys * 4) * 4;
}

template <typename T>
__global__ void __launch_bounds__(256) attn_q8_simt_kernel(const AttnQ8Args a) {
  extern __shared__ __align__(16) float simt_sm[];
  const int hd = a.hd, pitch = hd + 4;
  float* Ks = simt_sm;                           // [64][hd + 4]
  float* Vs = Ks + kSimtKeys * pitch;            // [64][hd + 4]
  float* Qs = Vs + kSimtKeys * pitch;            // [32][hd]
  float* Ps = Qs + kSimtRows * hd;               // [8 warps][64 keys][4 rows]
  __shared__ int s_len[kSimtRows], s_start[kSimtRows], s_lo, s_hi, s_last;
  __shared__ uint64_t s_mask[kSimtRows][kAttnQ8MaxWords];

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int h = blockIdx.x / a.tiles, tile = blockIdx.x % a.tiles, split = blockIdx.y;
  const int q0 = tile * kSimtRows;
  const int nq = min(kSimtRows, a.M - q0);
  const int t0 = q0 / a.G, ntok = (q0 + nq - 1) / a.G - t0 + 1;
  pdl_wait();
  pdl_trigger();
  const int sb = a.mask ? a.spec_base[0] : 0;
  if (threadIdx.x == 0) {
    s_lo = INT32_MAX;
    s_hi = 0;
  }
  __syncthreads();
  if (threadIdx.x < ntok) {
    const int t = t0 + threadIdx.x;
    const int start = max(a.prefix_start ? a.prefix_start[t] : 0, 0);
    const int len = min(a.prefix_len[t], a.kv_end);
    int64_t lo = start, hi = len;
    if (len <= start) lo = INT32_MAX, hi = 0;
    for (int w = 0; w < a.mask_words; ++w) {
      const uint64_t m = a.mask[(int64_t)t * a.mask_words + w];
      s_mask[threadIdx.x][w] = m;
      if (m) {
        lo = min(lo, (int64_t)sb + w * 64 + __ffsll(m) - 1);
        hi = max(hi, (int64_t)sb + w * 64 + 64 - __clzll(m));
      }
    }
    s_len[threadIdx.x] = len;
    s_start[threadIdx.x] = start;
    atomicMin(&s_lo, (int)max(lo, (int64_t)0));
    atomicMax(&s_hi, (int)min(hi, (int64_t)a.kv_end));
  }
  for (int i = threadIdx.x; i < kSimtRows * hd; i += blockDim.x) {
    const int r = i / hd, d = i % hd;
    float v = 0.f;
    if (r < nq) {
      const int qr = q0 + r;
      v = to_f32<T>(static_cast<const T*>(a.q)[(int64_t)(qr / a.G) * a.ldq + (int64_t)(h * a.G + qr % a.G) * hd + d]);
    }
    Qs[i] = v * a.scale;
  }
  __syncthreads();
  // the live range, cut into n_splits slices of whole key blocks
  const int lo = s_hi > s_lo ? s_lo / kSimtKeys * kSimtKeys : 0, hi = s_hi > s_lo ? s_hi : 0;
  const int per = ((hi - lo + kSimtKeys - 1) / kSimtKeys + a.n_splits - 1) / a.n_splits * kSimtKeys;
  const int k_lo = (int)min((int64_t)lo + (int64_t)split * per, (int64_t)hi), k_hi = min(k_lo + per, hi);

  float m[4], l[4], acc[4][4];
  int tok[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    m[i] = -INFINITY;
    l[i] = 0.f;
    tok[i] = min(q0 + warp * 4 + i, a.M - 1) / a.G - t0;
    if (tok[i] >= ntok) tok[i] = ntok - 1;
#pragma unroll
    for (int u = 0; u < 4; ++u) acc[i][u] = 0.f;
  }
  const bool warp_on = warp * 4 < nq;
  const int cpr = hd >> 4;
  for (int kb = k_lo; kb < k_hi; kb += kSimtKeys) {
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * kSimtKeys * cpr; i += blockDim.x) {
      const bool is_v = i >= kSimtKeys * cpr;
      const int idx = is_v ? i - kSimtKeys * cpr : i;
      const int j = idx / cpr, c = idx % cpr;
      const int slot = kb + j;
      uint4 u = make_uint4(0, 0, 0, 0);
      float sc = 0.f;
      if (slot < k_hi) {
        u = *reinterpret_cast<const uint4*>((is_v ? a.vc : a.kc) + (int64_t)h * a.head_stride + (int64_t)slot * hd + c * 16);
        sc = q8_scale((is_v ? a.vs : a.ks)[(int64_t)h * a.scale_head_stride + slot]);
      }
      float* dst = (is_v ? Vs : Ks) + j * pitch + c * 16;
      const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const float2 p = q8_unpack2(w[x]), q = q8_unpack2(w[x] >> 16);
        *reinterpret_cast<float4*>(dst + 4 * x) = make_float4(p.x * sc, p.y * sc, q.x * sc, q.y * sc);
      }
    }
    __syncthreads();
    if (!warp_on) continue;
    float s[4][2];
#pragma unroll
    for (int i = 0; i < 4; ++i) s[i][0] = s[i][1] = 0.f;
    const float* k0 = Ks + lane * pitch;
    const float* k1 = k0 + 32 * pitch;
    const float* qw = Qs + warp * 4 * hd;
    for (int d = 0; d < hd; d += 4) {
      const float4 x = *reinterpret_cast<const float4*>(k0 + d), y = *reinterpret_cast<const float4*>(k1 + d);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float4 q = *reinterpret_cast<const float4*>(qw + i * hd + d);
        s[i][0] = fmaf(q.x, x.x, fmaf(q.y, x.y, fmaf(q.z, x.z, fmaf(q.w, x.w, s[i][0]))));
        s[i][1] = fmaf(q.x, y.x, fmaf(q.y, y.y, fmaf(q.z, y.z, fmaf(q.w, y.w, s[i][1]))));
      }
    }
    // visibility of the lane's two keys per row, then one softmax step
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int tk = tok[i];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int slot = kb + lane + 32 * u;
        bool ok = slot < k_hi && slot >= s_start[tk] && slot < s_len[tk];
        if (!ok && slot < k_hi && a.mask_words) {
          const int64_t bit = (int64_t)slot - sb;
          if (bit >= 0 && bit < a.mask_words * 64) ok = (s_mask[tk][bit >> 6] >> (bit & 63)) & 1ull;
        }
        if (!ok) s[i][u] = -INFINITY;
      }
      const float top = warp_max(fmaxf(s[i][0], s[i][1]));
      const float mn = fmaxf(m[i], top);
      const float ref = mn == -INFINITY ? 0.f : mn;  // nothing seen yet: every p below is 0
      const float alpha = m[i] == -INFINITY ? 0.f : expf(m[i] - ref);
      const float p0 = s[i][0] == -INFINITY ? 0.f : expf(s[i][0] - ref);
      const float p1 = s[i][1] == -INFINITY ? 0.f : expf(s[i][1] - ref);
      m[i] = mn;
      l[i] = fmaf(l[i], alpha, warp_sum(p0 + p1));
#pragma unroll
      for (int u = 0; u < 4; ++u) acc[i][u] *= alpha;
      Ps[(warp * kSimtKeys + lane) * 4 + i] = p0;
      Ps[(warp * kSimtKeys + lane + 32) * 4 + i] = p1;
    }
    __syncwarp();
    const int nk = min(kSimtKeys, k_hi - kb);
    for (int j = 0; j < nk; ++j) {
      const float4 p = *reinterpret_cast<const float4*>(Ps + (warp * kSimtKeys + j) * 4);
      // a key that no row of this warp sees adds nothing, whatever its value
      if (p.x == 0.f && p.y == 0.f && p.z == 0.f && p.w == 0.f) continue;
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int d = lane + 32 * u;
        if (d < hd) {
          const float v = Vs[j * pitch + d];
          acc[0][u] = fmaf(p.x, v, acc[0][u]);
          acc[1][u] = fmaf(p.y, v, acc[1][u]);
          acc[2][u] = fmaf(p.z, v, acc[2][u]);
          acc[3][u] = fmaf(p.w, v, acc[3][u]);
        }
      }
    }
    __syncwarp();
  }
  T* outp = static_cast<T*>(a.out);
  auto store_row = [&](int r, const float* o, float sum) {
    const int qr = q0 + r;
    const float inv = sum == 0.f ? 0.f : 1.f / sum;  // (a NaN sum stays NaN)
    T* dst = outp + (int64_t)(qr / a.G) * a.ldo + (int64_t)(h * a.G + qr % a.G) * hd;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int d = lane + 32 * u;
      if (d < hd) dst[d] = from_f32<T>(o[u] * inv);
    }
  };
  if (a.n_splits == 1) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (warp * 4 + i < nq) store_row(warp * 4 + i, acc[i], l[i]);
    return;
  }
  const int rec = hd + 2;
  float* mine = a.part + ((int64_t)blockIdx.x * a.n_splits + split) * kSimtRows * rec;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (warp * 4 + i >= nq) continue;
    float* p = mine + (warp * 4 + i) * rec;
    if (lane == 0) {
      p[0] = m[i];
      p[1] = l[i];
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int d = lane + 32 * u;
      if (d < hd) p[2 + d] = acc[i][u];
    }
  }
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0)
    s_last = atomicAdd(&a.counters[kAttnQ8CounterBase + blockIdx.x], 1u) == (uint32_t)(a.n_splits - 1);
  __syncthreads();
  if (!s_last) return;
  __threadfence();
  const float* all = a.part + (int64_t)blockIdx.x * a.n_splits * kSimtRows * rec;
  for (int i = 0; i < 4; ++i) {
    const int r = warp * 4 + i;
    if (r >= nq) continue;
    float top = -INFINITY;
    for (int sp = 0; sp < a.n_splits; ++sp) top = fmaxf(top, __ldcg(all + ((int64_t)sp * kSimtRows + r) * rec));
    float sum = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
    for (int sp = 0; sp < a.n_splits; ++sp) {
      const float* p = all + ((int64_t)sp * kSimtRows + r) * rec;
      const float ls = __ldcg(p + 1), ms = __ldcg(p);
      if (ls == 0.f) continue;
      const float w = ms == -INFINITY ? 1.f : expf(ms - top);  // NaN scores: their sum is NaN, kept
      sum = fmaf(ls, w, sum);
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int d = lane + 32 * u;
        if (d < hd) o[u] = fmaf(__ldcg(p + 2 + d), w, o[u]);
      }
    }
    store_row(r, o, sum);
  }
  if (threadIdx.x == 0) a.counters[kAttnQ8CounterBase + blockIdx.x] = 0u;
}

static int launch_simt(AttnQ8Args& a, int dtype, void* workspace, int64_t workspace_bytes, cudaStream_t stream) {
  a.tiles = (a.M + kSimtRows - 1) / kSimtRows;
  const int64_t blocks = (int64_t)a.n_kv * a.tiles;
  if (blocks > INT32_MAX) return fail(SSD_ERR_UNSUPPORTED, "ssd_tree_attention_q8: too many row tiles");
  // Slices of at least 128 keys until the SMs hold two CTAs each.
  int64_t splits = (2 * device_sms() + blocks - 1) / blocks;
  const int64_t by_len = (a.kv_end + 127) / 128;
  if (splits > by_len) splits = by_len;
  if (splits < 1 || blocks > kAttnQ8MaxBlocks) splits = 1;
  a.n_splits = (int)splits;
  if (splits > 1) {
    const int64_t need = kCounterBytes + blocks * splits * kSimtRows * (a.hd + 2) * 4;
    if (!workspace || need > workspace_bytes)
      return fail(SSD_ERR_WORKSPACE, "ssd_tree_attention_q8: workspace too small (need %lld)", (long long)need);
    a.counters = static_cast<uint32_t*>(workspace);
    a.part = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + kCounterBytes);
  }
  auto go = [&](auto kern, bool& set) {
    if (!set) {
      allow_max_dynamic_smem(kern);
      set = true;
    }
    return launch_kernel("attn_q8_simt_kernel", kern, dim3((unsigned)blocks, (unsigned)splits), dim3(256),
                         (size_t)simt_q8_smem(a.hd), stream, 1u, 1u, a);
  };
  static bool set_f32 = false, set_bf16 = false;
  if (dtype == SSD_F32) return go(attn_q8_simt_kernel<float>, set_f32);
  return go(attn_q8_simt_kernel<bf16>, set_bf16);
}

}  // namespace ssd

using namespace ssd;

extern "C" int ssd_tree_attention_q8(const void* q, int64_t ldq, int64_t T, int64_t n_heads, const SsdKvQ8* cache,
                                     const int32_t* prefix_len, const int32_t* prefix_start, const int32_t* spec_base,
                                     const uint64_t* spec_mask, int64_t mask_words, int64_t kv_bound, void* out,
                                     int64_t ldo, int dtype, void* workspace, int64_t workspace_bytes,
                                     uint32_t* status, void* stream) {
  const char* who = "ssd_tree_attention_q8";
  if (const int rc = check_kv_q8(cache, who)) return rc;
  const int64_t n_kv = cache->n_kv_heads, hd = cache->head_dim;
  if (T <= 0 || n_heads <= 0 || n_heads % n_kv) return fail(SSD_ERR_INVALID, "%s: bad head configuration", who);
  if (!q || !prefix_len || !out) return fail(SSD_ERR_INVALID, "%s: NULL argument", who);
  if (spec_mask && (!spec_base || mask_words <= 0 || mask_words > kAttnQ8MaxWords))
    return fail(SSD_ERR_INVALID, "%s: mask needs spec_base and 1..4 words", who);
  if (dtype != SSD_F32 && dtype != SSD_BF16) return fail(SSD_ERR_UNSUPPORTED, "%s: dtype %d", who, dtype);
  if (T > 1 && (ldq < n_heads * hd || ldo < n_heads * hd)) return fail(SSD_ERR_INVALID, "%s: rows overlap", who);
  if (T * (n_heads / n_kv) > INT32_MAX / 2) return fail(SSD_ERR_UNSUPPORTED, "%s: too many rows", who);
  AttnQ8Args a{};
  a.q = q;
  a.ldq = ldq;
  a.T = (int)T;
  a.G = (int)(n_heads / n_kv);
  a.M = a.T * a.G;
  a.n_kv = (int)n_kv;
  a.hd = (int)hd;
  a.kc = static_cast<const uint8_t*>(cache->k);
  a.vc = static_cast<const uint8_t*>(cache->v);
  a.ks = cache->k_scale;
  a.vs = cache->v_scale;
  a.head_stride = cache->head_stride;
  a.scale_head_stride = cache->scale_head_stride;
  a.kv_end = (int)(kv_bound > 0 && kv_bound < cache->max_slots ? kv_bound : cache->max_slots);
  a.prefix_len = prefix_len;
  a.prefix_start = prefix_start;
  a.spec_base = spec_mask ? spec_base : nullptr;
  a.mask = spec_mask;
  a.mask_words = spec_mask ? (int)mask_words : 0;
  a.out = out;
  a.ldo = ldo;
  a.status = status;
  a.scale = 1.0f / sqrtf((float)hd);
  return launch_simt(a, dtype, workspace, workspace_bytes, static_cast<cudaStream_t>(stream));
}
