// Tree attention over the 8-bit key/value cache (row format: kvq8.cuh).
//
// Query row r = t * G + g (token t, head g of the KV head's group) attends
// the slots [prefix_start[t], prefix_len[t]) and slot spec_base + j for every
// set bit j of token t's mask; a row that sees nothing gives zeros.
//   s = (q . k8) 2^ek / sqrt(hd),  o = sum p 2^ev v8 / sum p,  p = 2^(s log2 e - m)
#include <algorithm>
#include <atomic>

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
// a row tile merges them in slice order. With few rows it is one block's chain
// of latencies: 5 tokens of 32 + 8 heads of 64 over 160 keys take 20 us (31 with
// slices of two blocks, integer divisions in the staging loops and a merge that
// waits for each record in turn).
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
#pragma unroll
  for (int r = warp; r < kSimtRows; r += kSimtWarps) {
    const int qr = q0 + r, tok = qr / a.G;
    const T* src = static_cast<const T*>(a.q) + (int64_t)tok * a.ldq + (int64_t)(h * a.G + qr - tok * a.G) * hd;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int d = lane + 32 * u;
      if (d < hd) Qs[r * hd + d] = r < nq ? to_f32<T>(src[d]) * a.scale : 0.f;
    }
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
#pragma unroll
    for (int i = threadIdx.x; i < 2 * kSimtKeys * 8; i += 256) {  // 8 lanes a row, cpr of them with work
      const bool is_v = i >= kSimtKeys * 8;
      const int j = (i >> 3) & (kSimtKeys - 1), c = i & 7;
      if (c >= cpr) continue;
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
#pragma unroll 4
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
    // (keys past k_hi: P and V are zero)
#pragma unroll 8
    for (int j = 0; j < kSimtKeys; ++j) {
      const float4 p = *reinterpret_cast<const float4*>(Ps + (warp * kSimtKeys + j) * 4);
      // a key that no row of this warp sees adds nothing, whatever its value
      const bool none = p.x == 0.f && p.y == 0.f && p.z == 0.f && p.w == 0.f;
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int d = lane + 32 * u;
        if (32 * u < hd) {  // uniform; lanes past hd read the pitch's padding or the next row and are not stored
          const float v = none ? 0.f : Vs[j * pitch + d];
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
  // A warp joins a row: lane = slice for the weights, lane = dims for the sums.
  const int64_t pitch_rec = (int64_t)kSimtRows * rec;
  for (int r = warp; r < nq; r += kSimtWarps) {
    const float* row = a.part + (int64_t)blockIdx.x * a.n_splits * pitch_rec + (int64_t)r * rec;
    float top = -INFINITY;
    for (int sp = lane; sp < a.n_splits; sp += 32) top = fmaxf(top, __ldcg(row + sp * pitch_rec));
    top = warp_max(top);
    float sum = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
    for (int s0 = 0; s0 < a.n_splits; s0 += 32) {
      float ls = 0.f, w = 0.f;
      if (s0 + lane < a.n_splits) {
        const float ms = __ldcg(row + (s0 + lane) * pitch_rec);
        ls = __ldcg(row + (s0 + lane) * pitch_rec + 1);
        w = ls == 0.f ? 0.f : ms == -INFINITY ? 1.f : expf(ms - top);  // NaN scores: their sum is NaN, kept
      }
      sum += warp_sum(ls * w);
      const uint32_t live = __ballot_sync(0xffffffffu, ls != 0.f);
      const int n = min(32, a.n_splits - s0);
#pragma unroll 4
      for (int b = 0; b < n; ++b) {
        const float ws = __shfl_sync(0xffffffffu, w, b);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int d = lane + 32 * u;
          if (d < hd && ((live >> b) & 1u)) o[u] = fmaf(__ldcg(row + (s0 + b) * pitch_rec + 2 + d), ws, o[u]);
        }
      }
    }
    store_row(r, o, sum);
  }
  if (threadIdx.x == 0) a.counters[kAttnQ8CounterBase + blockIdx.x] = 0u;
}

// Lets the kernels use all shared memory, once per device (a kernel's attributes
// are set per device). `done`: a bit per device, set only after the attributes
// are: a call from another thread meanwhile sets them again, which is harmless,
// and never launches without them.
template <typename... Kerns>
static void allow_smem_on_device(std::atomic<uint64_t>& done, Kerns... kerns) {
  int dev = 0;
  const bool known = cudaGetDevice(&dev) == cudaSuccess && dev >= 0 && dev < 64;
  if (known && (done.load(std::memory_order_acquire) >> dev & 1u)) return;
  (allow_max_dynamic_smem(kerns), ...);
  if (known) done.fetch_or(1ull << dev, std::memory_order_release);
}

static int launch_simt(AttnQ8Args& a, int dtype, void* workspace, int64_t workspace_bytes, cudaStream_t stream) {
  a.tiles = (a.M + kSimtRows - 1) / kSimtRows;
  const int64_t blocks = (int64_t)a.n_kv * a.tiles;
  if (blocks > INT32_MAX) return fail(SSD_ERR_UNSUPPORTED, "ssd_tree_attention_q8: too many row tiles");
  // Slices of at least one key block until the SMs hold two CTAs each.
  int64_t splits = (2 * device_sms() + blocks - 1) / blocks;
  const int64_t by_len = (a.kv_end + kSimtKeys - 1) / kSimtKeys;
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
  auto go = [&](auto kern, std::atomic<uint64_t>& done) {
    allow_smem_on_device(done, kern);
    return launch_kernel("attn_q8_simt_kernel", kern, dim3((unsigned)blocks, (unsigned)splits), dim3(256),
                         (size_t)simt_q8_smem(a.hd), stream, 1u, 1u, a);
  };
  static std::atomic<uint64_t> done_f32{0}, done_bf16{0};
  if (dtype == SSD_F32) return go(attn_q8_simt_kernel<float>, done_f32);
  return go(attn_q8_simt_kernel<bf16>, done_bf16);
}

// ------------------------------------------------------------ tensor cores
// bf16 queries, head_dim 64 or 128, in the transposed form: keys are the
// M = 128 rows of the tensor-core tiles, query rows their N columns, so that
// a block of 128 keys costs what its N = 16 .. 144 query rows need and no
// padding of few query rows to 128 (decode has 4 .. 132).
//   S^T [128 keys x N]  = K8 [128 x hd] Q^T          (K8: codes as stored)
//   O^T [hd x N]       += V8^T [hd x 128] P'^T       (V8: codes as stored)
// The cache's codes feed the tensor cores untouched (kind::f8f6f4); what they
// multiply is split into 8-bit terms. A bf16 query element has 8 significant
// bits: q = (hi + lo) 2^eq with hi its nearest e4m3 (4 bits) and lo the rest in
// e5m2: exact down to 2^-13 of the row's largest, off by 2^-21 of that at most below.
// P' is the sum of three e5m2 terms, 3 significant bits each, taken from its fp16
// form (whose upper byte is an e5m2 code): off by 2^-10 of it at most, and by
// 2^-16 below 2^-6. Two terms do not do: hi in e5m2 and the rest in e4m3 hold 8
// bits down to 2^-2 only, and 3 where the rest vanishes, below 2^-7; the weights of
// an even tail beside one strong key are then off by up to 1/8, all to the same side.
// Scales never touch the operands: a softmax thread owns one key (= TMEM
// lane), so 2^ek is a factor of its scores and 2^ev an addend in its exponent,
//   t = s log2 e + ev,  P' = 2^(t - M + kBias),  l += P' 2^-ev,
// with M a whole number per row that scales O and l. A block's column maxima
// (one warp reduction instruction per column and warp, joined in shared memory)
// move M only when some t exceeds it by kGrow; then O and l shift by whole
// powers of two. P' <= 2^(kBias + kGrow) = 2^15.75 stays below the largest e5m2.
// The largest weight is above 2^(kBias - 1), so that what the last term cuts off
// comes to at most n 2^-27 of it over n keys. l sums the uncut P' in fp32 per thread
// until the end.
//
// A CTA = one KV head x up to 144 query rows (whole tokens) x one slice of the
// key blocks that some row sees (a bitmap in shared memory: slot ranges of
// other sequences in between are not read). Warps 0 / 1 stream K / V blocks by
// TMA; 2 issues the MMAs, S^T(b + 1) and O(b) as each is ready; 3 fetches the
// scale bytes, works out the visibility of blocks that not every row sees whole
// and zeroes V rows that none does (0 * NaN). The other warps prepare the queries and then run the
// softmax, as warpgroups of 128 threads = 128 keys. One warpgroup's block is a
// long chain (two waits, TMEM loads, one barrier, 2^x, stores, a fence), so
// several run side by side: CG of them share a block's columns, 16 CH each, and
// A such sets take the blocks in turn, each with its own S^T and P' buffers,
// references, l and O^T, joined at the end. What CH, CG and A are for N columns
// follows from registers (l: 16 CH), TMEM (N (2 A + A) <= 512 columns)
// and threads: see q8_shape.
constexpr int kQ8Keys = 128;
constexpr int kQ8MaxRows = 144;       // query rows per CTA: three ring stages fit next to their Q and P'
constexpr int kQ8MaxStages = 6;
constexpr int kQ8MapWords = 128;      // bitmap of key blocks (units of 2^unit_shift blocks)
constexpr int kQ8Helpers = 128;       // threads of warps 0 .. 3
constexpr float kQ8Bias = 12.f;
constexpr float kQ8Grow = 3.75f;
constexpr int kQ8Terms = 3;           // e5m2 terms of a weight
constexpr float kQ8Unset = 1e30f;     // reference of a row that saw no key yet: every t exceeds it
constexpr int kQ8BarSoftmax = 8, kQ8BarHelpers = 9;  // named barriers (1 .. 5: the warpgroups')

// Column chunks of 16 -> chunks per warpgroup, warpgroups that share a block,
// sets of them that take blocks in turn: as many warpgroups as registers and
// TMEM allow (up to four; three where l takes 48 registers), as sets where a
// block's columns do not fill them. Measured over 32k keys of 8 heads, us: 36 rows a
// head {2, 2, 2} 35.4, {2, 2, 1} 41.4, {3, 1, 1} 48.2; 88 rows {2, 3, 1} 50.6, {3, 2, 1}
// 54.8; 120 rows {2, 4, 1} 61.5, {3, 3, 1} 65.1. Up to 32 rows {2, 1, 4} and {2, 1, 2}
// come out even: 20 rows 31.0 and 31.7, 32 rows 33.4 and 31.9, heads of 64 27.7
// and 28.7, 340 slots 10.0 and 10.7, but 8k keys 20.0 and 17.8.
// P' has a buffer a set. A set alone of up to 96 columns has a second one: over few
// key blocks the softmax would wait for the first values (33 rows over 2k keys,
// 80 columns: 18.4 us with two, 20.0 with one). Of 128 columns one does: 2k prefill
// 119.8 us with two, 117.6 with one, and with head_dim 64 40.0 and 39.2 for 1k.
struct Q8Shape {
  int ch, cg, sets, p_buffers;
};
static Q8Shape q8_shape(int chunks) {
  if (chunks <= 2) return {chunks, 1, 4, 4};
  if (chunks <= 4) return {2, 2, 2, 2};
  if (chunks <= 8) return {2, (chunks + 1) / 2, 1, chunks <= 6 ? 2 : 1};
  return {3, 3, 1, 1};
}

struct AttnQ8Maps {
  CUtensorMap k, v;  // [n_kv][max_slots][hd] bytes, box {hd, 128, 1}
};

struct AttnQ8Meta {
  float rowc[kQ8MaxRows];                      // 2^eq scale log2 e per query row
  int len[kQ8MaxRows], start[kQ8MaxRows];      // per token
  uint32_t map[kQ8MapWords];
  int max_start, min_len;                      // a block inside [max_start, min_len) is visible to every row
  int first, count;                            // this CTA's units of the bitmap
  int part[8];                                 // per block buffer: not every row sees the whole block
  int abort;
  uint32_t tmem;
  uint64_t k_full[kQ8MaxStages], k_empty[kQ8MaxStages], v_full[kQ8MaxStages], v_clean[kQ8MaxStages],
      v_empty[kQ8MaxStages];
  uint64_t s_full[8], s_free[8], info_full[8], p_full[4], p_free[4], meta_ready, q_ready, o_full;
};
static_assert(sizeof(AttnQ8Meta) % 16 == 0, "the arrays behind it are read 16 bytes at a time");

// S^T runs one block of each set ahead of the softmax.
__host__ __device__ constexpr int q8_s_buffers(int sets) { return 2 * sets; }
__host__ __device__ constexpr int q8_p_bytes(int n) { return (n + 31) / 32 * 4096; }    // one term of one buffer
// Behind AttnQ8Meta: per softmax warp and column {kBias - M, the last move as
// a bf16 factor}, per warpgroup {column maxima of each warp's 32 keys}, and per
// block buffer {per token, the 128 bits of which of the block's keys it sees;
// per key, K's scale byte and V's in the high half}.
static int q8_fixed_smem(int hd, int n, const Q8Shape& f) {
  const int state = 4 * f.cg * f.sets * 16 * f.ch;
  return 1024 + 2 * n * hd + f.p_buffers * kQ8Terms * q8_p_bytes(n) + (int)sizeof(AttnQ8Meta) + state * 10 +
         q8_s_buffers(f.sets) * (n * 16 + kQ8Keys * 2);
}

// D[tmem] (+)= A[smem] * B[smem]^T, e4m3 in, fp32 accumulate.
__device__ __forceinline__ void umma_f8(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                        uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(tmem_d),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// Shared-memory matrix descriptor in two words: address and leading offset in
// the low one (an operand's later parts add (bytes >> 4) there), stride offset,
// version and swizzle (2 = 128 B, 4 = 64 B, 6 = 32 B) in the high one.
__device__ __forceinline__ uint32_t q8_desc_lo(uint32_t saddr, uint32_t lbo) {
  return ((saddr >> 4) & 0x3FFFu) | ((lbo >> 4) << 16);
}
__device__ __forceinline__ uint32_t q8_desc_hi(uint32_t sbo, uint32_t swizzle) {
  return (sbo >> 4) | (1u << 14) | (swizzle << 29);
}
__device__ __forceinline__ uint64_t q8_desc(uint32_t lo, uint32_t hi) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "r"(lo), "r"(hi));
  return d;
}
// e4m3 A, e4m3 or e5m2 B, fp32 D, M x N; mn: both operands MN-major.
__host__ __device__ constexpr uint32_t idesc_f8(int M, int N, bool mn, bool b_e5m2 = false) {
  return (1u << 4) | (b_e5m2 ? 1u << 10 : 0u) | (mn ? (1u << 15) | (1u << 16) : 0u) | (static_cast<uint32_t>(N >> 3) << 17) |
         (static_cast<uint32_t>(M >> 4) << 24);
}
// mbar_wait that sleeps between polls, for the warps that run ahead of the
// others (the copies, the scale bytes): polling takes instruction fetch from the
// warps that work. Waking up is slow, so the warps on the critical path poll.
// Gives up after seconds.
__device__ __forceinline__ bool q8_wait(uint64_t* bar, uint32_t parity) {
  for (uint32_t i = 0; i < 1u << 17; ++i) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}\n"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity), "r"(20000u)
        : "memory");
    if (ok) return true;
  }
  return false;
}
__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}\n"
      : "=r"(r));
  return r != 0;
}
__device__ __forceinline__ float q8_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Which of the slots kb .. kb + 63 a token sees: its range [start, len) plus
// the mask bits (bit i = slot sb + i) below kv_end.
__device__ __forceinline__ uint64_t q8_low_bits(int n) { return n <= 0 ? 0ull : n >= 64 ? ~0ull : (1ull << n) - 1ull; }
__device__ __forceinline__ uint64_t q8_seen_bits(int kb, int start, int len, const uint64_t* mask, int words, int sb,
                                                 int kv_end) {
  const uint64_t range = len > start ? q8_low_bits(len - kb) & ~q8_low_bits(start - kb) : 0ull;
  const int64_t off = (int64_t)kb - sb;  // mask bit of slot kb
  if (off <= -64 || off >= words * 64) return range;
  const int w = off >= 0 ? (int)(off >> 6) : -1, sh = (int)(off - (int64_t)w * 64);  // 0 .. 63
  const uint64_t lo = w >= 0 ? mask[w] : 0ull, up = w + 1 < words ? mask[w + 1] : 0ull;
  const uint64_t spec = sh == 0 ? lo : (lo >> sh) | (up << (64 - sh));
  return range | (spec & q8_low_bits(kv_end - kb));
}

// Walks the key blocks of this CTA's slice in ascending order.
struct Q8Blocks {
  const uint32_t* map;
  uint32_t bits;
  int word, shift, sub, unit;
  __device__ Q8Blocks(const uint32_t* m, int first, int count, int unit_shift)
      : map(m), shift(unit_shift), sub(0), unit(0) {
    word = first >> 5;
    bits = count ? map[word] & (~0u << (first & 31)) : 0u;
  }
  __device__ __forceinline__ int next() {  // first slot of the next block
    if (sub == 0) {
      while (bits == 0u) bits = map[++word];
      unit = word * 32 + __ffs(bits) - 1;
      bits &= bits - 1;
    }
    const int block = (unit << shift) + sub;
    sub = sub + 1 < (1 << shift) ? sub + 1 : 0;
    return block * kQ8Keys;
  }
};

// The CTA's tokens (by warps 0 .. 3): slot ranges, and the bitmap of key
// blocks that some row sees.
__device__ __forceinline__ void q8_tokens(const AttnQ8Args& a, AttnQ8Meta& m, int t0, int ntok, int sb,
                                          int unit_shift) {
  auto mark = [&](int lo, int hi) {  // slots lo .. hi
    const int u0 = (lo / kQ8Keys) >> unit_shift, u1 = (hi / kQ8Keys) >> unit_shift;
    for (int w = u0 >> 5; w <= u1 >> 5; ++w) {
      uint32_t bits = ~0u;
      if (w == u0 >> 5) bits &= ~0u << (u0 & 31);
      if (w == u1 >> 5) bits &= ~0u >> (31 - (u1 & 31));
      if ((m.map[w] & bits) != bits) atomicOr(&m.map[w], bits);
    }
  };
  for (int i = threadIdx.x; i < ntok; i += kQ8Helpers) {
    const int t = t0 + i;
    const int start = max(a.prefix_start ? a.prefix_start[t] : 0, 0);
    const int len = min(a.prefix_len[t], a.kv_end);
    m.start[i] = start;
    m.len[i] = len;
    atomicMax(&m.max_start, start);
    atomicMin(&m.min_len, len);
    if (len > start) mark(start, len - 1);
    for (int w = 0; w < a.mask_words; ++w) {
      const uint64_t bits = a.mask[(int64_t)t * a.mask_words + w];
      if (!bits) continue;
      const int64_t lo = (int64_t)sb + w * 64 + __ffsll(bits) - 1, hi = (int64_t)sb + w * 64 + 63 - __clzll(bits);
      if (hi < 0 || lo >= a.kv_end) continue;
      mark((int)max(lo, (int64_t)0), (int)min(hi, (int64_t)a.kv_end - 1));
    }
  }
}
// Slice `split` of the marked units, in equal shares: its first unit and how
// many (computed alike by each warp that asks).
__device__ __forceinline__ void q8_slice(const AttnQ8Meta& m, int split, int n_splits, int& first, int& count) {
  constexpr int PER = kQ8MapWords / 32;
  const int lane = threadIdx.x & 31;
  int mine = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) mine += __popc(m.map[lane * PER + i]);
  int before = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, before, o);
    if (lane >= o) before += up;
  }
  const int total = __shfl_sync(0xffffffffu, before, 31);
  before -= mine;
  const int u0 = (int)((int64_t)total * split / n_splits);
  count = (int)((int64_t)total * (split + 1) / n_splits) - u0;
  const bool here = count > 0 && u0 >= before && u0 < before + mine;
  int at = 0;
  if (here) {
    int skip = u0 - before;
    for (int i = 0; i < PER; ++i) {
      uint32_t bits = m.map[lane * PER + i];
      const int n = __popc(bits);
      if (skip >= n) {
        skip -= n;
        continue;
      }
      for (; skip > 0; --skip) bits &= bits - 1;
      at = (lane * PER + i) * 32 + __ffs(bits) - 1;
      break;
    }
  }
  const uint32_t who = __ballot_sync(0xffffffffu, here);
  first = who ? __shfl_sync(0xffffffffu, at, __ffs(who) - 1) : 0;
}

// Rows per token G: r / G for r < 2^20 / G as a product (0 <= r < 144, G <= 144).
__device__ __forceinline__ int q8_token(int r, uint32_t inv_g) { return static_cast<int>((r * inv_g) >> 20); }

// The CTA's query rows as an e4m3 and an e5m2 term per element, K-major rows of HD bytes
// (by the softmax warps). A row is LPR lanes x 8 elements; a lane loads a batch
// of rows (all it has, in every shape) before it converts the first.
template <int HD>
__device__ __forceinline__ void q8_queries(const AttnQ8Args& a, AttnQ8Meta& m, uint8_t* q_hi, uint8_t* q_lo, int N,
                                           int nrows, int t0, int h) {
  constexpr int LPR = HD / 8, BATCH = 4;
  const int rows_per_pass = (blockDim.x - kQ8Helpers) / LPR;
  const bf16* qb = static_cast<const bf16*>(a.q);
  const bool wide = (reinterpret_cast<uintptr_t>(a.q) & 15) == 0 && a.ldq % 8 == 0;
  const uint32_t inv_g = ((1u << 20) + a.G - 1) / a.G;
  const int l8 = threadIdx.x % LPR, r0 = (threadIdx.x - kQ8Helpers) / LPR;
  for (int rb = 0; rb < N; rb += rows_per_pass * BATCH) {
    uint32_t raw[BATCH][4];
#pragma unroll
    for (int u = 0; u < BATCH; ++u) {
      const int r = rb + u * rows_per_pass + r0;
      raw[u][0] = raw[u][1] = raw[u][2] = raw[u][3] = 0u;
      if (r < nrows) {
        const int tok = q8_token(r, inv_g);
        const bf16* src = qb + (int64_t)(t0 + tok) * a.ldq + (int64_t)(h * a.G + r - tok * a.G) * HD + l8 * 8;
        if (wide) {
          const uint4 v = *reinterpret_cast<const uint4*>(src);
          raw[u][0] = v.x, raw[u][1] = v.y, raw[u][2] = v.z, raw[u][3] = v.w;
        } else {
          const uint16_t* s16 = reinterpret_cast<const uint16_t*>(src);
#pragma unroll
          for (int e = 0; e < 4; ++e) raw[u][e] = s16[2 * e] | (static_cast<uint32_t>(s16[2 * e + 1]) << 16);
        }
      }
    }
#pragma unroll
    for (int u = 0; u < BATCH; ++u) {
      const int r = rb + u * rows_per_pass + r0;
      if (rb + u * rows_per_pass >= N) break;  // uniform
      float x[8], amax = 0.f;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[2 * e] = __uint_as_float(raw[u][e] << 16);
        x[2 * e + 1] = __uint_as_float(raw[u][e] & 0xffff0000u);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {  // Inf and NaN become the row's amax: they compare above every finite value
        const float v = fabsf(x[e]);
        amax = v <= 3.402823466e38f ? fmaxf(amax, v) : INFINITY;
      }
#pragma unroll
      for (int o = LPR / 2; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
      const bool fine = amax <= 3.402823466e38f;
      const int byte = q8_scale_byte(fine ? amax : 0.f);
      const float inv = q8_inv_scale(byte);
      uint32_t hi[2] = {0u, 0u}, lo[2] = {0u, 0u};
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        const float y0 = x[e] * inv, y1 = x[e + 1] * inv;
        const uint32_t c = q8_pack2(y0, y1);
        const float2 back = q8_unpack2(c);
        hi[e >> 2] |= c << (8 * (e & 3));
        const float2 rest = make_float2(y0 - back.x, y1 - back.y);
        lo[e >> 2] |= static_cast<uint32_t>(__nv_cvt_float2_to_fp8x2(rest, __NV_SATFINITE, __NV_E5M2)) << (8 * (e & 3));
      }
      if (r < N) {
        const int sw = HD == 128 ? (r & 7) : ((r >> 1) & 3);  // swizzled place of the lane's 8 bytes
        const int at = r * HD + (((l8 >> 1) ^ sw) << 4) + (l8 & 1) * 8;
        *reinterpret_cast<uint2*>(q_hi + at) = make_uint2(hi[0], hi[1]);
        *reinterpret_cast<uint2*>(q_lo + at) = make_uint2(lo[0], lo[1]);
        if (l8 == 0) {
          m.rowc[r] = fine ? q8_scale(byte) * (a.scale * 1.4426950408889634f) : __int_as_float(0x7fffffff);
        }
      }
    }
}
}

// Visibility of the 16 columns from `col` for the thread's key (bit j = column
// col + j), from the block's per-token key masks.
__device__ __forceinline__ uint32_t q8_chunk_vis(const uint32_t* vis_buf, int col, int G, int ntok, int quarter,
                                                 int lane) {
  uint32_t vis = 0u;
  const int last = min((col + 15) / G, ntok - 1);
  for (int t = col / G; t <= last; ++t)
    if ((vis_buf[t * 4 + quarter] >> lane) & 1u) {
      const int lo = max(t * G - col, 0), hi = min((t + 1) * G - col, 16);
      vis |= ((1u << hi) - 1u) & ~((1u << lo) - 1u);
    }
  return vis;
}

// Scores of a block that not every row sees whole: -inf where the thread's key
// is not seen, in place in TMEM. Out of line, like q8_rescale: the main loop's
// instructions have to fit the instruction cache (with this code in it the
// loop ran 20 % longer on blocks that never execute it).
__device__ __noinline__ void q8_mask_scores(uint32_t ts, const uint32_t* vis_buf, int col, int chunks, int G, int ntok,
                                            int quarter, int lane) {
#pragma unroll 1
  for (int c = 0; c < chunks; ++c) {
    const uint32_t vis = q8_chunk_vis(vis_buf, col + c * 16, G, ntok, quarter, lane);
    float x[16];
    tmem_ld16(ts + c * 16, x);
#pragma unroll
    for (int j = 0; j < 16; ++j) x[j] = (vis >> j) & 1u ? x[j] : -INFINITY;
    tmem_st16(ts + c * 16, x);
  }
  tmem_wait_st();
}

// Maximum (or sum) of 16 columns over 32 lanes, halving the columns a lane
// holds at every step: lane i (and i + 16) returns column i & 15's.
template <bool MAX>
__device__ __forceinline__ float q8_columns_reduce(float* v, int lane) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) {
#pragma unroll
    for (int j = 0; j < o; ++j) {
      const bool up = lane & o;
      const float give = up ? v[j] : v[j + o], keep = up ? v[j + o] : v[j];
      const float got = __shfl_xor_sync(0xffffffffu, give, o);
      v[j] = MAX ? fmaxf(keep, got) : keep + got;
    }
  }
  const float got = __shfl_xor_sync(0xffffffffu, v[0], 16);
  return MAX ? fmaxf(v[0], got) : v[0] + got;
}

// 8 columns of O^T, with the wait, and back.
__device__ __forceinline__ void q8_tmem_ld8(uint32_t taddr, float* v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void q8_tmem_st8(uint32_t taddr, const float* v) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "f"(v[0]),
               "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7])
               : "memory");
}
// O^T's columns times the last moves' factors (bf16 pairs in shared memory).
__device__ __noinline__ void q8_rescale(uint32_t to, const uint16_t* factors, int chunks) {
  constexpr uint32_t one = 0x3f803f80u;
#pragma unroll 1
  for (int c = 0; c < 2 * chunks; ++c) {
    const uint4 f = *reinterpret_cast<const uint4*>(factors + c * 8);
    if (f.x == one && f.y == one && f.z == one && f.w == one) continue;  // none of the eight moved
    const uint32_t w[4] = {f.x, f.y, f.z, f.w};
    float o[8];
    q8_tmem_ld8(to + c * 8, o);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      o[2 * j] *= __uint_as_float(w[j] << 16);
      o[2 * j + 1] *= __uint_as_float(w[j] & 0xffff0000u);
    }
    q8_tmem_st8(to + c * 8, o);
  }
  tmem_wait_st();
}

// TMEM load without its wait; the wait takes the registers along so that
// nothing reads them before it.
__device__ __forceinline__ void q8_tmem_ld16(uint32_t taddr, float* v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]),
        "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void q8_tmem_wait16(float* v) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]),
                 "+f"(v[8]), "+f"(v[9]), "+f"(v[10]), "+f"(v[11]), "+f"(v[12]), "+f"(v[13]), "+f"(v[14]), "+f"(v[15])
               :
               : "memory");
}

// t of 16 columns from their raw products x, in place. (Paired fp32
// instructions measured no faster: same rate, more register moves.)
__device__ __forceinline__ void q8_scores(const float* rowc, float* x, float ck, float ev) {
#pragma unroll
  for (int j = 0; j < 16; j += 4) {
    const float4 r = *reinterpret_cast<const float4*>(rowc + j);
    x[j] = fmaf(x[j] * r.x, ck, ev);
    x[j + 1] = fmaf(x[j + 1] * r.y, ck, ev);
    x[j + 2] = fmaf(x[j + 2] * r.z, ck, ev);
    x[j + 3] = fmaf(x[j + 3] * r.w, ck, ev);
  }
}
// Four weights (>= 0) as three e5m2 codes each. Through fp16, whose upper byte
// is an e5m2 code: hi is the weight cut to 3 significant bits, mid what is left
// rounded to 3 (half a step added, the lower byte cut off), lo what is left then,
// of either sign, cut to 3. Of the fp16's 11 bits that leaves a unit off at most.
// A NaN stays in hi.
__device__ __forceinline__ void q8_split4(const float* p, uint32_t& hi, uint32_t& mid, uint32_t& lo) {
  const __half2 w[2] = {__floats2half2_rn(p[0], p[1]), __floats2half2_rn(p[2], p[3])};
  uint32_t h[2], m[2], r[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    uint32_t bits;
    __half2 x;
    memcpy(&bits, &w[i], 4);
    h[i] = bits & 0xff00ff00u;
    memcpy(&x, &h[i], 4);
    const __half2 left = __hsub2(w[i], x);
    memcpy(&bits, &left, 4);
    m[i] = (bits + 0x00800080u) & 0xff00ff00u;
    memcpy(&x, &m[i], 4);
    const __half2 rest = __hsub2(left, x);
    memcpy(&r[i], &rest, 4);
  }
  hi = __byte_perm(h[0], h[1], 0x7531);
  mid = __byte_perm(m[0], m[1], 0x7531);
  lo = __byte_perm(r[0], r[1], 0x7531);
}
__device__ __forceinline__ float q8_warp_max(float v) {  // NaN gives way to numbers, as in fmaxf
  float r;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}

// N floats of one lane, from L2 (another CTA of this launch may have written
// them), zeros where `on` is false.
template <int N>
__device__ __forceinline__ void q8_ldcg(const float* p, bool on, float* v) {
  if constexpr (N == 4) {
    const float4 x = on ? __ldcg(reinterpret_cast<const float4*>(p)) : make_float4(0.f, 0.f, 0.f, 0.f);
    v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w;
  } else {
    const float2 x = on ? __ldcg(reinterpret_cast<const float2*>(p)) : make_float2(0.f, 0.f);
    v[0] = x.x, v[1] = x.y;
  }
}

// Joins the key slices' records {O 2^(..M), M, l} of query row r of CTA column
// `blk` of `blks` into dst: one warp, weights 2^(M_s - max M), in slice order. Slices that saw
// nothing have l = 0 and no O.
template <int HD>
__device__ __noinline__ void q8_join_row(const float* part, int n_splits, int blk, int blks, int r, bf16* dst) {
  constexpr int DPL = HD / 32;
  const int lane = threadIdx.x & 31;
  const float* ml_part = part + (int64_t)blks * n_splits * kQ8MaxRows * HD;
  const int64_t rec0 = (int64_t)blk * n_splits * kQ8MaxRows + r;
  float top = -INFINITY;
  for (int s = lane; s < n_splits; s += 32) {
    const float2 ml = __ldcg(reinterpret_cast<const float2*>(ml_part + (rec0 + (int64_t)s * kQ8MaxRows) * 2));
    if (ml.y != 0.f) top = fmaxf(top, ml.x);
  }
  top = warp_max(top);
  float sum = 0.f, acc[DPL];
#pragma unroll
  for (int i = 0; i < DPL; ++i) acc[i] = 0.f;
  for (int s0 = 0; s0 < n_splits; s0 += 32) {
    float w = 0.f, ls = 0.f;
    if (s0 + lane < n_splits) {
      const float2 ml = __ldcg(reinterpret_cast<const float2*>(ml_part + (rec0 + (int64_t)(s0 + lane) * kQ8MaxRows) * 2));
      ls = ml.y;
      w = ls != 0.f ? exp2f(ml.x - top) : 0.f;
    }
    sum += warp_sum(ls * w);
    const uint32_t live = __ballot_sync(0xffffffffu, ls != 0.f);
    const int n = min(32, n_splits - s0);
    const float* o0 = part + (rec0 + (int64_t)s0 * kQ8MaxRows) * HD + lane * DPL;
    for (int b = 0; b < n; b += 8) {  // eight records in flight
      float v[8][DPL];
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const bool on = b + u < n && ((live >> (b + u)) & 1u);
        q8_ldcg<DPL>(o0 + (int64_t)(b + u) * kQ8MaxRows * HD, on, v[u]);
      }
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const float ws = __shfl_sync(0xffffffffu, w, (b + u) & 31);
#pragma unroll
        for (int i = 0; i < DPL; ++i) acc[i] = fmaf(ws, v[u][i], acc[i]);
      }
    }
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  dst += lane * DPL;
#pragma unroll
  for (int i = 0; i < DPL; ++i) dst[i] = f2bf(acc[i] * inv);
}

template <int HD, int CH, int A, int PB>
__global__ void __launch_bounds__(CH == 3 ? 512 : 640, 1)
    attn_q8_tc_kernel(const __grid_constant__ AttnQ8Maps maps, const AttnQ8Args a, const int n_chunks, const int cgs,
                      const int tok_per_group, const int stages, const int unit_shift) {
  constexpr int TILE = kQ8Keys * HD;              // bytes of a K or V block
  constexpr uint32_t SW = HD == 128 ? 2u : 4u;    // 128-byte or 64-byte swizzle: one atom row per cache row
  constexpr uint32_t SBO = 8 * HD;                // 8 rows of HD bytes
  constexpr int SB = q8_s_buffers(A);             // S^T buffers; like PB, P' buffers, a power of two
  constexpr int SSH = SB == 8 ? 3 : SB == 4 ? 2 : 1;
  constexpr int PSH = PB == 4 ? 2 : PB == 2 ? 1 : 0;
  constexpr int WC = 16 * CH;                     // columns of a warpgroup
  constexpr bool KEEP = CH == 1;
  extern __shared__ uint8_t q8_smem_raw[];
  // (an offset, not a rounded address: the compiler keeps knowing that this is shared memory)
  uint8_t* sm = q8_smem_raw + ((1024u - (smem_u32(q8_smem_raw) & 1023u)) & 1023u);
  const int N = 16 * n_chunks;
  const int p_bytes = q8_p_bytes(N), atoms = (N + 31) / 32;
  const int wgs = cgs * A;
  uint8_t* k_ring = sm;
  uint8_t* v_ring = k_ring + stages * TILE;
  uint8_t* p_buf = v_ring + stages * TILE;        // [PB][terms][keys / 8][atoms][8 keys x 32 rows]
  uint8_t* q_hi = p_buf + PB * kQ8Terms * p_bytes;       // [N][HD]
  uint8_t* q_lo = q_hi + N * HD;
  AttnQ8Meta& m = *reinterpret_cast<AttnQ8Meta*>(q_lo + N * HD);
  float* refs = reinterpret_cast<float*>(&m + 1);                            // [softmax warps][WC]
  float* wmax = refs + 4 * wgs * WC;                                         // [warpgroups][4][WC]
  uint32_t* vis = reinterpret_cast<uint32_t*>(wmax + 4 * wgs * WC);          // [SB][N tokens][4]
  uint16_t* scales = reinterpret_cast<uint16_t*>(vis + SB * N * 4);          // [SB][keys]
  uint16_t* factors = scales + SB * kQ8Keys;                                 // [softmax warps][WC]
  volatile int* abort_flag = &m.abort;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int h = blockIdx.x % a.n_kv, group = a.tiles - 1 - blockIdx.x / a.n_kv;  // longest causal rows first
  const int split = blockIdx.y;
  const int t0 = group * tok_per_group;
  const int ntok = min(tok_per_group, a.T - t0);
  const int nrows = ntok * a.G;

  if (threadIdx.x == 0) {
    m.max_start = 0;
    m.min_len = INT32_MAX;
    m.abort = 0;
    for (int i = 0; i < stages; ++i) {
      mbar_init(&m.k_full[i], 1);
      mbar_init(&m.k_empty[i], 1);
      mbar_init(&m.v_full[i], 1);
      mbar_init(&m.v_clean[i], 1);
      mbar_init(&m.v_empty[i], 1);
    }
    for (int i = 0; i < SB; ++i) {
      mbar_init(&m.s_full[i], 1);
      mbar_init(&m.s_free[i], 4 * cgs);
      mbar_init(&m.info_full[i], 1);
    }
    for (int i = 0; i < PB; ++i) {
      mbar_init(&m.p_full[i], 4 * cgs);
      mbar_init(&m.p_free[i], 1);
    }
    mbar_init(&m.meta_ready, 1);
    mbar_init(&m.q_ready, 4 * wgs);
    mbar_init(&m.o_full, 1);
    fence_mbar_init();
  }
  if (threadIdx.x < kQ8MapWords) m.map[threadIdx.x] = 0u;
  if (warp == 2) {
    tmem_alloc(&m.tmem, 512);
    tmem_relinquish();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&maps.k);
    tma_prefetch_desc(&maps.v);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = m.tmem, tmem_o = tmem + SB * N;  // SB S^T buffers, then A O^T, N columns each
  pdl_wait();
  pdl_trigger();
  const uint32_t p_s = smem_u32(p_buf);
  auto give_up = [&] {
    report_error(a.status, kErrWaitTimeout);
    *abort_flag = 1;
  };

  if (warp < 4) {
    const int sb = a.mask ? a.spec_base[0] : 0;
    q8_tokens(a, m, t0, ntok, sb, unit_shift);
    __syncwarp();
    named_bar_sync(kQ8BarHelpers, kQ8Helpers);
    int first, count;
    q8_slice(m, split, a.n_splits, first, count);
    const int nblocks = count << unit_shift;
    const int max_start = m.max_start, min_len = m.min_len;
    if (warp == 3 && lane == 0) {
      m.first = first;
      m.count = count;
      mbar_arrive(&m.meta_ready);
    }
    Q8Blocks it(m.map, first, count, unit_shift);
    if (warp < 2) {
      if (lane == 0) {
        const bool is_v = warp == 1;
        uint64_t* full = is_v ? m.v_full : m.k_full;
        uint64_t* empty = is_v ? m.v_empty : m.k_empty;
        uint8_t* ring = is_v ? v_ring : k_ring;
        const CUtensorMap* map = is_v ? &maps.v : &maps.k;
        const uint64_t pol = l2_policy_evict_first();
        int st = 0, issued = 0;
        uint32_t phase = 0;
        for (int b = 0; b < nblocks; ++b) {
          if ((b >= stages && !q8_wait(&empty[st], phase ^ 1u)) || *abort_flag) {
            give_up();
            break;
          }
          mbar_arrive_expect_tx(&full[st], TILE);
          tma_load_3d(ring + st * TILE, map, &full[st], 0, it.next(), h, pol);
          ++issued;
          if (++st == stages) st = 0, phase ^= 1u;
        }
        if (*abort_flag)  // copies in flight land before the CTA leaves
          for (int b = max(issued - stages, 0); b < issued; ++b) (void)mbar_wait(&full[b % stages], (b / stages) & 1);
      }
    } else if (warp == 2) {
      // The whole warp runs the loop (its addresses stay uniform), one lane
      // issues. The softmax frees S^T's buffer and fills P' at the same time, so
      // a fixed order loses nothing: S^T runs SB blocks ahead of O. (A loop
      // that polled for whichever is ready cost the softmax warps their
      // instruction fetch: 20 % of the kernel.) O(b) goes first: it frees the P'
      // buffer, while S^T(b + SB) is wanted a whole softmax block later (the other
      // way round: 65 rows over 32k keys 105 us against 101.5, 2k prefill 120.5
      // against 117.6). Descriptors of later parts of an operand add to the low word.
      const bool leader = elect_one();
      if (nblocks > 0) {
        const uint32_t id_s = idesc_f8(128, N, false), id_s5 = idesc_f8(128, N, false, true), id_o = idesc_f8(128, N, true, true);
        const uint32_t rows_hi = q8_desc_hi(SBO, SW), p_hi = q8_desc_hi(atoms * 256, 6u);
        const uint32_t k_lo = q8_desc_lo(smem_u32(k_ring), 16), v_lo = q8_desc_lo(smem_u32(v_ring), 0);
        const uint32_t qh_lo = q8_desc_lo(smem_u32(q_hi), 16), ql_lo = q8_desc_lo(smem_u32(q_lo), 16);
        const uint32_t p_lo = q8_desc_lo(p_s, 256);
        int sS = 0, sP = 0;
        uint32_t phS = 0, phP = 0;
        bool ok = mbar_wait(&m.q_ready, 0);
#pragma unroll 1
        for (int nS = 0; nS < nblocks + SB; ++nS) {
          const int nP = nS - SB, buf = nS & (SB - 1), pbuf = nP & (PB - 1);
          if (nP >= 0)
            ok = ok && mbar_wait(&m.s_free[buf], (nP >> SSH) & 1) && mbar_wait(&m.p_full[pbuf], (nP >> PSH) & 1);
          if (__any_sync(0xffffffffu, !ok || *abort_flag)) {
            if (lane == 0) give_up();
            break;
          }
          tc_fence_after();
          if (nP >= 0) {
            ok = mbar_wait(&m.v_clean[sP], phP);
            tc_fence_after();
            if (leader && ok) {
              // V8^T: MN-major, one atom of HD head dims x 8 keys per 8 HD bytes; for HD = 64 the second half of
              // M = 128 repeats the first (lanes 64 .. 127 are not read). P': MN-major, atoms of 32 rows x 8 keys.
              const uint32_t d = tmem_o + (nP & (A - 1)) * N;
              const uint32_t v = v_lo + sP * (TILE >> 4), pl = p_lo + pbuf * (kQ8Terms * p_bytes >> 4);
#pragma unroll
              for (int term = 0; term < kQ8Terms; ++term)
#pragma unroll
                for (int kk = 0; kk < kQ8Keys / 32; ++kk)
                  umma_f8(d, q8_desc(v + kk * 2 * HD, rows_hi),
                          q8_desc(pl + term * (p_bytes >> 4) + kk * (atoms * 64), p_hi), id_o,
                          (nP >= A || term > 0 || kk > 0) ? 1u : 0u);
              umma_commit(&m.p_free[pbuf]);
              umma_commit(&m.v_empty[sP]);
            }
            __syncwarp();
            if (++sP == stages) sP = 0, phP ^= 1u;
          }
          if (nS < nblocks) {
            ok = ok && mbar_wait(&m.k_full[sS], phS);
            tc_fence_after();
            if (leader && ok) {
              const uint32_t d = tmem + buf * N, k = k_lo + sS * (TILE >> 4);
#pragma unroll
              for (int ks = 0; ks < HD / 32; ++ks)
                umma_f8(d, q8_desc(k + ks * 2, rows_hi), q8_desc(qh_lo + ks * 2, rows_hi), id_s, ks > 0);
#pragma unroll
              for (int ks = 0; ks < HD / 32; ++ks)
                umma_f8(d, q8_desc(k + ks * 2, rows_hi), q8_desc(ql_lo + ks * 2, rows_hi), id_s5, 1u);
              umma_commit(&m.s_full[buf]);
              umma_commit(&m.k_empty[sS]);
            }
            __syncwarp();
            if (++sS == stages) sS = 0, phS ^= 1u;
          }
        }
      }
      if (leader) umma_commit(&m.o_full);
    } else {
      // Scale bytes of every block (loaded one block ahead); for blocks that not
      // every row sees whole, the keys that each token sees, for the softmax
      // warps, and zeros in the V rows that none does.
      const uint8_t* ksc = a.ks + (int64_t)h * a.scale_head_stride;
      const uint8_t* vsc = a.vs + (int64_t)h * a.scale_head_stride;
      uint32_t bytes[4] = {0u, 0u, 0u, 0u};
      int next_kb = 0;
      auto fetch = [&] {
        next_kb = it.next();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int slot = next_kb + i * 32 + lane;
          bytes[i] = slot < a.kv_end ? ksc[slot] | (static_cast<uint32_t>(vsc[slot]) << 8) : 0u;
        }
      };
      if (nblocks > 0) fetch();
      int st = 0;
      uint32_t phase = 0;
      for (int b = 0; b < nblocks; ++b) {
        const int kb = next_kb, buf = b & (SB - 1);
        const bool part = kb < max_start || kb + kQ8Keys > min_len;
        bool bad = b >= SB && !q8_wait(&m.s_free[buf], ((b >> SSH) - 1) & 1);  // block b - SB is done with them
#pragma unroll
        for (int i = 0; i < 4; ++i) scales[buf * kQ8Keys + i * 32 + lane] = static_cast<uint16_t>(bytes[i]);
        if (b + 1 < nblocks) fetch();
        if (lane == 0) m.part[buf] = part;
        uint32_t seen[4] = {~0u, ~0u, ~0u, ~0u};
        if (part) {
          seen[0] = seen[1] = seen[2] = seen[3] = 0u;
          for (int i = lane; i < ntok; i += 32) {
            const uint64_t* mask = a.mask + (int64_t)(t0 + i) * a.mask_words;
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              const uint64_t v = q8_seen_bits(kb + 64 * half, m.start[i], m.len[i], mask, a.mask_words, sb, a.kv_end);
              vis[(buf * N + i) * 4 + 2 * half] = static_cast<uint32_t>(v);
              vis[(buf * N + i) * 4 + 2 * half + 1] = static_cast<uint32_t>(v >> 32);
              seen[2 * half] |= static_cast<uint32_t>(v);
              seen[2 * half + 1] |= static_cast<uint32_t>(v >> 32);
            }
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&m.info_full[buf]);
        bad = bad || !q8_wait(&m.v_full[st], phase);
        if (__any_sync(0xffffffffu, bad || *abort_flag)) {
          if (lane == 0) give_up();
          break;
        }
        if (part) {
          bool wrote = false;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if (!((__reduce_or_sync(0xffffffffu, seen[i]) >> lane) & 1u)) {
              uint4* row = reinterpret_cast<uint4*>(v_ring + st * TILE + (i * 32 + lane) * HD);
#pragma unroll
              for (int c = 0; c < HD / 16; ++c) row[c] = make_uint4(0, 0, 0, 0);
              wrote = true;
            }
          }
          if (wrote) fence_proxy_async_smem();
          __syncwarp();
        }
        if (lane == 0) mbar_arrive(&m.v_clean[st]);
        if (++st == stages) st = 0, phase ^= 1u;
      }
    }
  } else {
    // ---- softmax warps: the queries, then thread = key
    const int sw = warp - 4, wg = sw >> 2, quarter = warp & 3;
    const int cg = wg % cgs, turn = wg / cgs;     // columns [WC cg, ..), blocks turn, turn + A, ..
    const int my_chunks = min(CH, n_chunks - cg * CH);
    const int col_base = cg * WC;
    const uint32_t lane_base = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t to = tmem_o + turn * N + lane_base + col_base;
    const int key = quarter * 32 + lane;
    float* const my_ref = refs + sw * WC;
    float* const my_max = wmax + (wg * 4 + quarter) * WC;
    const float* const all_max = wmax + wg * 4 * WC;
    uint16_t* const my_fac = factors + sw * WC;
    const uint32_t p_at = p_s + (key >> 3) * atoms * 256 + (key & 7) * 32;
    const uint32_t p_flip = (key >> 2) & 1;
    q8_queries<HD>(a, m, q_hi, q_lo, N, nrows, t0, h);
    for (int i = lane; i < WC; i += 32)  // columns past the rows: P' = 0
      my_ref[i] = col_base + i < nrows ? kQ8Unset : -kQ8Unset;
    fence_proxy_async_smem();
    __syncwarp();
    named_bar_sync(kQ8BarSoftmax, 128 * wgs);  // the rows' scales are read by other warps than wrote them
    if (lane == 0) mbar_arrive(&m.q_ready);
    bool bad = !mbar_wait(&m.meta_ready, 0);
    if (bad) give_up();
    const int nblocks = bad ? 0 : m.count << unit_shift;
    float l[WC];
#pragma unroll
    for (int i = 0; i < WC; ++i) l[i] = 0.f;
    for (int b = turn; b < nblocks; b += A) {
      const int buf = b & (SB - 1), pbuf = b & (PB - 1);
      const uint32_t use = (b >> SSH) & 1;        // parity of the S^T buffer's use by block b
      // After a timeout the loop runs on without waiting: the warpgroup's barriers stay matched.
      if (!bad && !(mbar_wait(&m.info_full[buf], use) && mbar_wait(&m.s_full[buf], use))) {
        bad = true;
        give_up();
      }
      const bool part = m.part[buf];
      const uint32_t bytes = scales[buf * kQ8Keys + key];
      const float ck = q8_scale(max(bytes & 0xffu, 1u));  // (not 0: a masked score is -inf times this)
      // (inside the bytes ever written: an unseen slot's may be any, and 255 would make inv_v -Inf, 0 * Inf NaN)
      const int vb = min(max(static_cast<int>(bytes >> 8), kQ8MinScale), kQ8MaxScale);
      const float ev = static_cast<float>(vb - 127), inv_v = q8_inv_scale(vb);
      tc_fence_after();
      const uint32_t ts = tmem + buf * N + lane_base + col_base;
      if (part) q8_mask_scores(ts, vis + buf * N * 4, col_base, my_chunks, a.G, ntok, quarter, lane);
      // t of every column and its maximum over the warp's keys. The registers
      // hold one chunk's t next to l: the loop runs down to chunk 0, whose t stays
      // for the weights below; the others' are computed again (all of them: 3 %
      // longer). It is rolled for the instruction cache.
      float x[16];
      q8_tmem_ld16(ts + (my_chunks - 1) * 16, x);
      named_bar_sync(1 + wg, 128);  // the other warps have read the last block's maxima
#pragma unroll 1
      for (int c = my_chunks - 1; c >= 0; --c) {
        if (c + 1 < my_chunks) q8_tmem_ld16(ts + c * 16, x);
        q8_tmem_wait16(x);
        q8_scores(m.rowc + col_base + c * 16, x, ck, ev);
#pragma unroll
        for (int j = 0; j < 16; j += 4) {
          const float4 top = make_float4(q8_warp_max(x[j]), q8_warp_max(x[j + 1]), q8_warp_max(x[j + 2]),
                                         q8_warp_max(x[j + 3]));
          *reinterpret_cast<float4*>(my_max + c * 16 + j) = top;  // (all lanes the same: no branch)
        }
      }
      tc_fence_before();
      __syncwarp();
      if (KEEP && lane == 0) mbar_arrive(&m.s_free[buf]);  // the scores are in registers
      named_bar_sync(1 + wg, 128);
      // lane i: columns i, i + 32 (each warp for itself, all alike)
      constexpr int PER = (WC + 31) / 32;
      float now[PER], factor[PER];
      bool moves = false;
#pragma unroll
      for (int k = 0; k < PER; ++k) {
        const int i = lane + 32 * k;
        factor[k] = 1.f;
        now[k] = -kQ8Unset;
        if (i < 16 * my_chunks) {
          const float mx = fmaxf(fmaxf(all_max[i], all_max[WC + i]), fmaxf(all_max[2 * WC + i], all_max[3 * WC + i]));
          const float old = my_ref[i];
          now[k] = old;
          if (mx + old > kQ8Bias + kQ8Grow) {
            now[k] = kQ8Bias - ceilf(mx);
            const float by = old - now[k];  // a whole number
            factor[k] = old == kQ8Unset || by > 126.f ? 0.f : __uint_as_float((127u - static_cast<uint32_t>(by)) << 23);
            moves = true;
          }
        }
      }
      if (__any_sync(0xffffffffu, moves)) {
#pragma unroll
        for (int k = 0; k < PER; ++k) {
          const int i = lane + 32 * k;
          if (i < WC) {
            my_ref[i] = now[k];
            my_fac[i] = static_cast<uint16_t>(__float_as_uint(factor[k]) >> 16);  // a power of two or 0: exact
          }
        }
        __syncwarp();
        if (b >= A) {  // the last P V into this O is block b - A's
          if (!bad && !mbar_wait(&m.p_free[(b - A) & (PB - 1)], ((b - A) >> PSH) & 1)) {
            bad = true;
            give_up();
          }
          tc_fence_after();
          q8_rescale(to, my_fac, my_chunks);
        }
#pragma unroll
        for (int i = 0; i < WC; i += 2) {
          const uint32_t w = reinterpret_cast<const uint32_t*>(my_fac)[i / 2];  // (columns past my_chunks: l = 0)
          l[i] *= __uint_as_float(w << 16);
          l[i + 1] *= __uint_as_float(w & 0xffff0000u);
        }
      }
      if (b >= PB && !bad && !mbar_wait(&m.p_free[pbuf], ((b >> PSH) - 1) & 1)) {  // P V of block b - PB read this buffer
        bad = true;
        give_up();
      }
      const uint32_t pb = p_at + pbuf * kQ8Terms * p_bytes;
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        if (c < my_chunks) {
          const int col = col_base + c * 16;
          float* p = x;
          if (c > 0) {
            q8_tmem_ld16(ts + c * 16, p);
            q8_tmem_wait16(p);
            q8_scores(m.rowc + col, p, ck, ev);
          }
          uint32_t w[kQ8Terms][4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float4 ref = *reinterpret_cast<const float4*>(my_ref + c * 16 + 4 * j);
            const float r[4] = {ref.x, ref.y, ref.z, ref.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              p[4 * j + e] = q8_ex2(p[4 * j + e] + r[e]);
              l[c * 16 + 4 * j + e] = fmaf(p[4 * j + e], inv_v, l[c * 16 + 4 * j + e]);
            }
            q8_split4(p + 4 * j, w[0][j], w[1][j], w[2][j]);
          }
          const uint32_t at = pb + (col >> 5) * 256 + ((((col >> 4) & 1u) ^ p_flip) << 4);
#pragma unroll
          for (int k = 0; k < kQ8Terms; ++k)
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at + k * p_bytes), "r"(w[k][0]), "r"(w[k][1]),
                         "r"(w[k][2]), "r"(w[k][3])
                         : "memory");
        }
      }
      fence_proxy_async_smem();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if (!KEEP) mbar_arrive(&m.s_free[buf]);
        mbar_arrive(&m.p_full[pbuf]);
      }
    }
    // ---- results: l summed over the 128 keys' threads, O^T read back (lane = head dim)
    const int parties = 128 * wgs;
    if (!mbar_wait(&m.o_full, 0)) give_up();
    tc_fence_after();
    __syncwarp();
    named_bar_sync(kQ8BarSoftmax, parties);
    float* s_l = reinterpret_cast<float*>(p_buf);  // [softmax warps][WC]: the P buffers are free once every MMA retired
    float* s_f = s_l + 4 * wgs * WC;                // [A][N] factors of the O accumulators
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const float sum = q8_columns_reduce<false>(l + c * 16, lane);
      if (lane < 16) s_l[sw * WC + c * 16 + lane] = sum;
    }
    __syncwarp();
    named_bar_sync(kQ8BarSoftmax, parties);
    // thread i: row i's factors, and the record {M, l} of a slice
    const int64_t rec0 = ((int64_t)blockIdx.x * a.n_splits + split) * kQ8MaxRows;
    const int i = threadIdx.x - kQ8Helpers;
    if (i < N) {
      const int g = i / WC, c = i - g * WC;
      float ls[A], ms[A], top = -kQ8Unset, sum = 0.f;
#pragma unroll
      for (int u = 0; u < A; ++u) {  // join the sets' shares of the slice
        const float* pl = s_l + (u * cgs + g) * 4 * WC + c;
        ls[u] = (pl[0] + pl[WC]) + (pl[2 * WC] + pl[3 * WC]);
        ms[u] = kQ8Bias - refs[(u * cgs + g) * 4 * WC + c];
        if (ls[u] != 0.f) top = fmaxf(top, ms[u]);
      }
#pragma unroll
      for (int u = 0; u < A; ++u) {
        ms[u] = ls[u] == 0.f ? 0.f : exp2f(ms[u] - top);
        sum = fmaf(ls[u], ms[u], sum);
      }
      float scale = 1.f;
      if (a.n_splits > 1) {
        if (i < nrows) {
          float* ml = a.part + (int64_t)gridDim.x * a.n_splits * kQ8MaxRows * HD + (rec0 + i) * 2;
          *reinterpret_cast<float2*>(ml) = make_float2(top, sum);
        }
      } else {
        scale = sum == 0.f ? 0.f : 1.f / sum;
      }
#pragma unroll
      for (int u = 0; u < A; ++u) s_f[u * N + i] = nblocks > u ? ms[u] * scale : 0.f;  // (O without a block: not read)
    }
    __syncwarp();
    named_bar_sync(kQ8BarSoftmax, parties);
    const int d = quarter * 32 + lane;
    if (quarter * 32 < HD) {
#pragma unroll 1
      for (int c = wg; c < n_chunks; c += wgs) {
        const int col = c * 16;
        float o[16];
#pragma unroll
        for (int u = 0; u < A; ++u) {
          float x[16];
          tmem_ld16(tmem_o + u * N + lane_base + col, x);
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            const float f = s_f[u * N + col + j];
            const float y = f == 0.f ? 0.f : f * x[j];
            o[j] = u == 0 ? y : o[j] + y;
          }
        }
        if (a.n_splits > 1) {
          float* dst = a.part + (rec0 + col) * HD + d;
#pragma unroll
          for (int j = 0; j < 16; ++j)
            if (col + j < nrows) dst[j * HD] = o[j];
        } else {
          int tok = col / a.G, g = col - tok * a.G;
          bf16* base = static_cast<bf16*>(a.out) + (int64_t)h * a.G * HD + d;
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            if (col + j < nrows) base[(int64_t)(t0 + tok) * a.ldo + g * HD] = f2bf(o[j]);
            if (++g == a.G) g = 0, ++tok;
          }
        }
      }
    }
    if constexpr (CH == 1) {  // few rows: the last slice to finish joins the column's records
      if (a.n_splits > 1) {
        __threadfence();
        __syncwarp();
        named_bar_sync(kQ8BarSoftmax, parties);
        if (threadIdx.x == kQ8Helpers) {
          const uint32_t before = atomicAdd(&a.counters[kAttnQ8CounterBase + blockIdx.x], 1u);
          m.first = before == (uint32_t)(a.n_splits - 1);
          if (m.first) a.counters[kAttnQ8CounterBase + blockIdx.x] = 0u;
        }
        __syncwarp();
        named_bar_sync(kQ8BarSoftmax, parties);
        if (m.first) {
          __threadfence();
          for (int r = sw; r < nrows; r += 4 * wgs) {
            const int tok = r / a.G;
            bf16* dst = static_cast<bf16*>(a.out) + (int64_t)(t0 + tok) * a.ldo + (int64_t)(h * a.G + r - tok * a.G) * HD;
            q8_join_row<HD>(a.part, a.n_splits, blockIdx.x, gridDim.x, r, dst);
          }
        }
      }
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == 2) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// The join as a launch of its own, one warp a row. With up to 16 query rows
// the last CTA of a column joins its records itself, which the device hardly
// notices (one token over 2k keys: 11.2 us against 11.6 replayed from a graph)
// but the host does: 13.6 -> 12.1 us launched call by call, where the second
// launch was the bound. With 36 rows over 32k keys, 18 slices, the one CTA
// takes 2.4 us longer than the launch (37.8 us against 35.4).
template <int HD>
__global__ void __launch_bounds__(256) attn_q8_join_kernel(const AttnQ8Args a, const int tok_per_group) {
  pdl_wait();
  pdl_trigger();
  const int h = blockIdx.x % a.n_kv, group = a.tiles - 1 - blockIdx.x / a.n_kv;
  const int t0 = group * tok_per_group;
  const int r = blockIdx.y * 8 + (threadIdx.x >> 5);
  if (r >= min(tok_per_group, a.T - t0) * a.G) return;
  const int tok = r / a.G;
  bf16* dst = static_cast<bf16*>(a.out) + (int64_t)(t0 + tok) * a.ldo + (int64_t)(h * a.G + r - tok * a.G) * HD;
  q8_join_row<HD>(a.part, a.n_splits, blockIdx.x, gridDim.x, r, dst);
}

static int q8_tensor_map(const void* base, const SsdKvQ8& c, CUtensorMap* out) {
  TensorMapEncodeFn encode = tensor_map_encoder();
  if (!encode) return fail(SSD_ERR_CUDA, "cuTensorMapEncodeTiled is unavailable");
  cuuint64_t dims[3] = {(cuuint64_t)c.head_dim, (cuuint64_t)c.max_slots, (cuuint64_t)c.n_kv_heads};
  cuuint64_t strides[2] = {(cuuint64_t)c.head_dim, (cuuint64_t)c.head_stride};
  cuuint32_t box[3] = {(cuuint32_t)c.head_dim, (cuuint32_t)kQ8Keys, 1u};
  cuuint32_t estr[3] = {1u, 1u, 1u};
  const CUresult r = encode(out, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void*>(base), dims, strides, box, estr,
                            CU_TENSOR_MAP_INTERLEAVE_NONE,
                            c.head_dim == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
                            CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(SSD_ERR_CUDA, "ssd_tree_attention_q8: tensor map (%d)", (int)r);
  return SSD_OK;
}

// Query rows in groups of whole tokens, evenly, and key slices: one CTA per SM,
// slices of at least two key blocks (one block each: 12.4 us against 11.2 for one
// token over 2k keys), and no join at all for as many blocks as the warpgroup
// sets, or one more, take side by side (one token over 340 slots 8.8 us in one
// slice, 10.2 in two; 600 slots 10.2 and 10.3 in three; 1100 slots 13.8 and 10.5 in
// five). Groups of up to 144 rows or of up to 128, whichever the
// estimate takes for shorter: key blocks of a CTA, and two for the queries and
// the results, x the measured time of one at that many columns, in 30 ns. (144
// against 128 rows of 8 heads, us: 2048 tokens 128 and 118; 65 tokens over 2k
// keys 23.7 and 20.3, 33 tokens 19.4 and 17.7, as SMs are left; 65 tokens over
// 32k keys 101 and 108, as they fill two groups but not three; 33 tokens 67 and 74.)
struct Q8Plan {
  int tiles, tokens, chunks, key_blocks;
  int64_t splits;
};
static Q8Plan q8_plan(int T, int G, int n_kv, int kv_end, int sms) {
  constexpr int kCost[10] = {0, 18, 18, 35, 35, 60, 60, 71, 71, 87};
  Q8Plan best{};
  double least = 0.;
  for (const int rows : {kQ8MaxRows, 128}) {
    if (G > rows) break;
    Q8Plan p;
    const int fit = rows / G, few = (T + fit - 1) / fit;
    p.tokens = (T + few - 1) / few;
    p.tiles = (T + p.tokens - 1) / p.tokens;
    p.chunks = (p.tokens * G + 15) / 16;
    p.key_blocks = (kv_end + kQ8Keys - 1) / kQ8Keys;
    const int64_t blocks = (int64_t)n_kv * p.tiles;
    p.splits = p.key_blocks <= q8_shape(p.chunks).sets + 1
                   ? 1
                   : std::max<int64_t>(1, std::min<int64_t>(sms / blocks, (p.key_blocks + 1) / 2));
    const double waves = std::max(1., static_cast<double>(blocks) / sms);
    const double cost = waves * static_cast<double>((p.key_blocks + p.splits - 1) / p.splits + 2) * kCost[p.chunks];
    if (rows == kQ8MaxRows || cost < least) best = p, least = cost;
  }
  return best;
}

template <int HD>
static int launch_tc(AttnQ8Args& a, const SsdKvQ8& cache, void* workspace, int64_t workspace_bytes,
                     cudaStream_t stream) {
  const Q8Plan plan = q8_plan(a.T, a.G, a.n_kv, a.kv_end, device_sms());
  a.tiles = plan.tiles;
  const int tpg = plan.tokens, chunks = plan.chunks, key_blocks = plan.key_blocks;
  const int64_t blocks = (int64_t)a.n_kv * a.tiles, splits = plan.splits;
  if (blocks > INT32_MAX) return fail(SSD_ERR_UNSUPPORTED, "ssd_tree_attention_q8: too many row groups");
  int shift = 0;
  while ((key_blocks >> shift) >= kQ8MapWords * 32) ++shift;
  a.n_splits = (int)splits;
  if (splits > 1) {
    const int64_t need = kCounterBytes + blocks * splits * kQ8MaxRows * (HD + 2) * 4;
    if (!workspace || need > workspace_bytes)
      return fail(SSD_ERR_WORKSPACE, "ssd_tree_attention_q8: workspace too small (need %lld)", (long long)need);
    a.part = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + kCounterBytes);
    a.counters = static_cast<uint32_t*>(workspace);
  }
  AttnQ8Maps maps;
  if (const int rc = q8_tensor_map(cache.k, cache, &maps.k)) return rc;
  if (const int rc = q8_tensor_map(cache.v, cache, &maps.v)) return rc;
  const Q8Shape f = q8_shape(chunks);
  const int fixed = q8_fixed_smem(HD, chunks * 16, f);
  int stages = (232448 - fixed) / (2 * kQ8Keys * HD);
  if (stages > kQ8MaxStages) stages = kQ8MaxStages;
  const size_t smem = (size_t)fixed + (size_t)stages * 2 * kQ8Keys * HD;
  typedef void (*Kern)(const AttnQ8Maps, const AttnQ8Args, int, int, int, int, int);
  const Kern kerns[6] = {attn_q8_tc_kernel<HD, 1, 4, 4>, attn_q8_tc_kernel<HD, 2, 4, 4>, attn_q8_tc_kernel<HD, 2, 2, 2>,
                         attn_q8_tc_kernel<HD, 2, 1, 2>, attn_q8_tc_kernel<HD, 2, 1, 1>, attn_q8_tc_kernel<HD, 3, 1, 1>};
  static std::atomic<uint64_t> done{0};
  allow_smem_on_device(done, kerns[0], kerns[1], kerns[2], kerns[3], kerns[4], kerns[5]);
  const Kern kern = kerns[f.ch == 3 ? 5 : f.sets == 4 ? f.ch - 1 : f.sets == 2 ? 2 : f.p_buffers == 2 ? 3 : 4];
  int rc = launch_kernel("attn_q8_tc_kernel", kern, dim3((unsigned)blocks, (unsigned)splits),
                         dim3((unsigned)(kQ8Helpers + 128 * f.cg * f.sets)), smem, stream, 1u, 1u, maps, a, chunks, f.cg,
                         tpg, stages, shift);
  if (rc || splits == 1 || chunks == 1) return rc;
  return launch_kernel("attn_q8_join_kernel", attn_q8_join_kernel<HD>,
                       dim3((unsigned)blocks, (unsigned)((tpg * a.G + 7) / 8)), dim3(256), 0, stream, 1u, 1u, a, tpg);
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
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == SSD_BF16 && a.G <= kQ8MaxRows) {
    if (hd == 128) return launch_tc<128>(a, *cache, workspace, workspace_bytes, s);
    if (hd == 64) return launch_tc<64>(a, *cache, workspace, workspace_bytes, s);
  }
  return launch_simt(a, dtype, workspace, workspace_bytes, s);
}
