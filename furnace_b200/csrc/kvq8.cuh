// The 8-bit paged KV cache: append with rotation, attention, read-back.
// Included by kernels.cu (shares the launch and PTX helpers).
//
// Layout (fz_kvq8 in include/furnace.h): a page holds 64 positions of every
// KV head; page p, head h, side w (0 keys, 1 values) is the 64 * HD bytes at
// ((p * nkv + h) * 2 + w) * 64 * HD, four blocks of 16 positions back to back.
// A byte is code + 128, code in [-127, 127]; the value is code * scale with one
// f32 scale per (page, head, side, block).
//
// Inside a block the bytes lie in the order in which a warp's lanes (g = lane /
// 4, t = lane % 4) want them as B operands of mma.m16n8k16, so that a lane's
// operands are whole 16-byte pieces and a warp's pieces are consecutive:
//   keys    [8 positions][64 dims] tiles: piece (position g, dims 16t..16t+15)
//   values  [32 dims] tiles: piece (g, t) = 4 words i, the word's bytes being
//           positions 2t, 2t + 1, 8 + 2t, 9 + 2t of dim 8i + g
constexpr uint32_t KQ_PAGE = 64;   // positions of a page
constexpr uint32_t KQ_BLOCK = 16;  // positions that share a scale
constexpr uint32_t KQ_NB = KQ_PAGE / KQ_BLOCK;

// Byte offset inside a block of key (tok, dim) and value (tok, dim).
template <int HD>
__device__ __forceinline__ uint32_t kq_koff(uint32_t tok, uint32_t dim) {
  return (tok >> 3) * 8 * HD + (dim >> 6) * 512 + (tok & 7) * 64 + (dim & 63);
}
__device__ __forceinline__ uint32_t kq_voff(uint32_t tok, uint32_t dim) {
  return (dim >> 5) * 512 + (dim & 7) * 64 + ((tok & 7) >> 1) * 16 + ((dim & 31) >> 3) * 4 + (tok >> 3) * 2 + (tok & 1);
}

struct KqSeq {
  int32_t len, n_new, row0;  // positions held, of these new, first row
};

// Sequence i's lengths, checked: a sequence whose numbers are out of range is
// treated as having no rows, and the status word says so.
__device__ __forceinline__ KqSeq kq_seq(const KvQ8Batch& b, uint32_t i, uint32_t* status) {
  KqSeq s;
  const int64_t len = (b.lens ? (int64_t)b.lens[i] : 0) + b.len_add;
  int64_t r0 = (int64_t)i * b.max_new, n = b.max_new;
  if (b.starts) {
    r0 = b.starts[i];
    n = (int64_t)b.starts[i + 1] - r0;
  }
  if (len < 0 || len > (int64_t)b.max_pages * KQ_PAGE || n < 0 || n > b.max_new || n > len || r0 < 0 ||
      r0 + n > b.n_rows) {
    atomicOr(status, KQ_BAD_LEN);
    return KqSeq{0, 0, 0};
  }
  s.len = (int32_t)len;
  s.n_new = (int32_t)n;
  s.row0 = (int32_t)r0;
  return s;
}

// Physical page of sequence i's page j, or -1 (status) when it is none.
__device__ __forceinline__ int32_t kq_page(const KvQ8Dev& c, const KvQ8Batch& b, uint32_t i, uint32_t j) {
  const int64_t at = (int64_t)i * b.max_pages + j;
  const int64_t p = b.pages ? (int64_t)b.pages[at] : at;
  if (p < 0 || p >= c.n_pages) {
    atomicOr(c.status, KQ_BAD_PAGE);
    return -1;
  }
  return (int32_t)p;
}

__device__ __forceinline__ float kq_ld(const float* p) { return *p; }
__device__ __forceinline__ float kq_ld(const __half* p) { return __half2float(*p); }
__device__ __forceinline__ void kq_st(float* p, float v) { *p = v; }
__device__ __forceinline__ void kq_st(__half* p, float v) { *p = __float2half_rn(v); }

// Element d of a head's row, rotated at a position's factors cs (null: as it
// is): pairs half a head apart, every product rounded by itself (the
// reference's uncontracted a*c - b*s / a*s + b*c, src/model.rs:193-217).
template <int HD, typename T>
__device__ __forceinline__ float kq_rotated(const T* x, const float2* cs, uint32_t d) {
  constexpr uint32_t half = HD / 2;
  const float own = kq_ld(x + d);
  if (!cs) return own;
  const float2 f = cs[d % half];
  const float other = kq_ld(x + (d < half ? d + half : d - half));
  return d < half ? __fsub_rn(__fmul_rn(own, f.x), __fmul_rn(other, f.y))
                  : __fadd_rn(__fmul_rn(other, f.y), __fmul_rn(own, f.x));
}

// code of x at scale s (0 for an empty scale)
__device__ __forceinline__ int kq_code(float x, float s) {
  return s > 0.f ? __float2int_rn(fminf(fmaxf(__fdiv_rn(x, s), -127.f), 127.f)) : 0;
}

// ---------------------------------------------------------------------------
// Append.  Grid (blocks a sequence can touch, nkv, n_seqs): a CTA quantizes
// one block of one head, keys and values.  The scale is the largest magnitude
// of the call's values / 127, and at least the block's older scale when
// positions before this call's are kept; those take the codes of the larger
// scale.  Every position of the block is one step of a plain loop here.
// ---------------------------------------------------------------------------
constexpr int KQ_AP_THREADS = 128;

template <int HD, typename T>
__global__ void __launch_bounds__(KQ_AP_THREADS) k_kvq8_append(KvQ8Dev c, KvQ8Batch b, const T* __restrict__ k,
                                                               const T* __restrict__ v, uint64_t ld) {
  pdl_trigger();
  pdl_wait();
  const KqSeq s = kq_seq(b, blockIdx.z, c.status);
  const int32_t p0 = s.len - s.n_new;
  const int32_t blk = p0 / (int32_t)KQ_BLOCK + (int32_t)blockIdx.x, base = blk * (int32_t)KQ_BLOCK;
  if (s.n_new == 0 || base >= s.len) return;
  const int32_t page = kq_page(c, b, blockIdx.z, blk / KQ_NB);
  if (page < 0) return;
  if (c.rope && s.len > (int32_t)c.n_rope) {
    if (threadIdx.x == 0) atomicOr(c.status, KQ_BAD_POS);
    return;
  }
  const uint32_t h = blockIdx.y, tid = threadIdx.x, sub = blk % KQ_NB;
  const int32_t a = max(p0 - base, 0), e = min(s.len - base, (int32_t)KQ_BLOCK);  // new positions [a, e)
  __shared__ float red[KQ_AP_THREADS / 32];
  for (int w = 0; w < 2; w++) {
    uint8_t* codes = c.codes + (((uint64_t)page * c.nkv + h) * 2 + w) * KQ_PAGE * HD + sub * KQ_BLOCK * HD;
    float* sc = c.scales + (((uint64_t)page * c.nkv + h) * 2 + w) * KQ_NB + sub;
    auto value = [&](int32_t tok, uint32_t d) {
      const uint64_t at = (uint64_t)(s.row0 + base + tok - p0) * ld + (uint64_t)h * HD;
      return w ? kq_ld(v + at + d)
               : kq_rotated<HD>(k + at, c.rope ? c.rope + (uint64_t)(base + tok) * (HD / 2) : nullptr, d);
    };
    float m = 0.f;
    bool bad = false;
    for (int32_t tok = a; tok < e; tok++)
      for (uint32_t d = tid; d < HD; d += KQ_AP_THREADS) {
        const float x = fabsf(value(tok, d));
        bad |= !(x <= 3.402823466e38f);
        m = fmaxf(m, x);
      }
    if (bad) atomicOr(c.status, KQ_NOT_FINITE);
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (__syncthreads_or(bad)) m = __int_as_float(0x7fffffff);  // a scale that is no number, not a wrong one
    if (tid % 32 == 0) red[tid / 32] = m;
    const float before = *sc;
    __syncthreads();
    bool nan = false;
    for (int i = 0; i < KQ_AP_THREADS / 32; i++) {
      nan |= red[i] != red[i];
      m = fmaxf(m, red[i]);
    }
    float scale = __fdiv_rn(m, 127.f);
    if (a > 0 && !(scale > before)) scale = before;
    if (nan) scale = __int_as_float(0x7fffffff);
    const bool grew = a > 0 && scale > before;
    const float ratio = __fdiv_rn(before, scale);
    for (int32_t tok = 0; tok < e; tok++)
      for (uint32_t d = tid; d < HD; d += KQ_AP_THREADS) {
        uint8_t* p = codes + (w ? kq_voff(tok, d) : kq_koff<HD>(tok, d));
        if (tok >= a)
          *p = (uint8_t)(128 + kq_code(value(tok, d), scale));
        else if (grew)
          *p = (uint8_t)(128 + __float2int_rn(__fmul_rn((float)((int)*p - 128), ratio)));
      }
    __syncthreads();  // every thread has read *sc and red
    if (tid == 0) *sc = scale;
  }
}

// ---------------------------------------------------------------------------
// Read-back: the rows a batch names as values.  Grid (max_new, nkv, n_seqs).
// ---------------------------------------------------------------------------
template <int HD, typename T>
__global__ void __launch_bounds__(HD) k_kvq8_read(KvQ8Dev c, KvQ8Batch b, T* __restrict__ k, T* __restrict__ v,
                                                  uint64_t ld) {
  pdl_trigger();
  pdl_wait();
  const KqSeq s = kq_seq(b, blockIdx.z, c.status);
  const uint32_t h = blockIdx.y, d = threadIdx.x;
  if ((int32_t)blockIdx.x >= s.n_new) return;
  const uint32_t pos = s.len - s.n_new + blockIdx.x;
  const int32_t page = kq_page(c, b, blockIdx.z, pos / KQ_PAGE);
  if (page < 0) return;
  const uint32_t sub = pos / KQ_BLOCK % KQ_NB, tok = pos % KQ_BLOCK;
  for (int w = 0; w < 2; w++) {
    T* out = w ? v : k;
    if (!out) continue;
    const uint64_t side = ((uint64_t)page * c.nkv + h) * 2 + w;
    const uint8_t code = c.codes[side * KQ_PAGE * HD + sub * KQ_BLOCK * HD + (w ? kq_voff(tok, d) : kq_koff<HD>(tok, d))];
    kq_st(out + (uint64_t)(s.row0 + blockIdx.x) * ld + (uint64_t)h * HD + d,
          __fmul_rn((float)((int)code - 128), c.scales[side * KQ_NB + sub]));
  }
}

// ---------------------------------------------------------------------------
// Attention: one CTA of four warps per (row, query head); a warp takes every
// fourth visible position, its lanes the dims, with an online softmax, and
// the four warps' sums meet in shared memory.
// ---------------------------------------------------------------------------
constexpr int KQ_AT_THREADS = 128;

template <int HD, typename T>
__global__ void __launch_bounds__(KQ_AT_THREADS) k_kvq8_attend(KvQ8Dev c, KvQ8Batch b, const T* __restrict__ q,
                                                               uint64_t ldq, T* __restrict__ out, uint64_t ldo,
                                                               uint32_t window, uint32_t sinks, float scale) {
  pdl_trigger();
  pdl_wait();
  constexpr int DPL = HD / 32;
  const KqSeq s = kq_seq(b, blockIdx.z, c.status);
  if ((int32_t)blockIdx.x >= s.n_new) return;
  const uint32_t head = blockIdx.y, h = head / c.group, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t pos = s.len - s.n_new + blockIdx.x, row = s.row0 + blockIdx.x;
  if (c.rope && pos >= c.n_rope) {
    if (threadIdx.x == 0) atomicOr(c.status, KQ_BAD_POS);
    return;
  }
  float qv[DPL], acc[DPL], m = -INFINITY, l = 0.f;
  for (int i = 0; i < DPL; i++) {
    qv[i] = kq_rotated<HD>(q + (uint64_t)row * ldq + (uint64_t)head * HD,
                           c.rope ? c.rope + (uint64_t)pos * (HD / 2) : nullptr, lane + 32 * i);
    acc[i] = 0.f;
  }
  for (uint32_t t = warp; t <= pos; t += 4) {
    if (window && pos - t >= window && t >= sinks) continue;
    const int32_t page = kq_page(c, b, blockIdx.z, t / KQ_PAGE);
    if (page < 0) continue;
    const uint32_t sub = t / KQ_BLOCK % KQ_NB, tok = t % KQ_BLOCK;
    const uint64_t side = ((uint64_t)page * c.nkv + h) * 2;
    const uint8_t* kc = c.codes + side * KQ_PAGE * HD + sub * KQ_BLOCK * HD;
    float d = 0.f;
    for (int i = 0; i < DPL; i++) d = fmaf(qv[i], (float)((int)kc[kq_koff<HD>(tok, lane + 32 * i)] - 128), d);
    for (int o = 16; o > 0; o >>= 1) d += __shfl_xor_sync(0xffffffffu, d, o);
    d *= scale * c.scales[side * KQ_NB + sub];
    const float mn = fmaxf(m, d), alpha = expf(m - mn), p = expf(d - mn);
    const float pv = p * c.scales[(side + 1) * KQ_NB + sub];
    l = fmaf(l, alpha, p);
    m = mn;
    for (int i = 0; i < DPL; i++)
      acc[i] = fmaf(acc[i], alpha, pv * (float)((int)kc[KQ_PAGE * HD + kq_voff(tok, lane + 32 * i)] - 128));
  }
  __shared__ float sm[4], sl[4], sa[4][HD];
  if (lane == 0) sm[warp] = m, sl[warp] = l;
  for (int i = 0; i < DPL; i++) sa[warp][lane + 32 * i] = acc[i];
  __syncthreads();
  const float top = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
  for (uint32_t d = threadIdx.x; d < HD; d += KQ_AT_THREADS) {
    float num = 0.f, den = 0.f;
    for (int w = 0; w < 4; w++) {
      const float f = sm[w] == -INFINITY ? 0.f : expf(sm[w] - top);
      num = fmaf(f, sa[w][d], num);
      den = fmaf(f, sl[w], den);
    }
    kq_st(out + (uint64_t)row * ldo + (uint64_t)head * HD + d, den == 0.f ? 0.f : __fdiv_rn(num, den));
  }
}

// ---------------------------------------------------------------------------
// Launches
// ---------------------------------------------------------------------------
template <int HD, typename T>
static void kvq8_append_t(const KvQ8Dev& c, const KvQ8Batch& b, const void* k, const void* v, uint64_t ld,
                          cudaStream_t s) {
  const dim3 grid((b.max_new + 2 * KQ_BLOCK - 2) / KQ_BLOCK, c.nkv, b.n_seqs);
  launch_pdl(k_kvq8_append<HD, T>, grid, dim3(KQ_AP_THREADS), 0, s, c, b, static_cast<const T*>(k),
             static_cast<const T*>(v), ld);
}

void launch_kvq8_append(const KvQ8Dev& c, const KvQ8Batch& b, bool f16, const void* k, const void* v, uint64_t ld,
                        cudaStream_t s) {
  if (!b.n_seqs) return;
  if (c.hd == 128)
    f16 ? kvq8_append_t<128, __half>(c, b, k, v, ld, s) : kvq8_append_t<128, float>(c, b, k, v, ld, s);
  else
    f16 ? kvq8_append_t<64, __half>(c, b, k, v, ld, s) : kvq8_append_t<64, float>(c, b, k, v, ld, s);
}

template <int HD, typename T>
static void kvq8_read_t(const KvQ8Dev& c, const KvQ8Batch& b, void* k, void* v, uint64_t ld, cudaStream_t s) {
  launch_pdl(k_kvq8_read<HD, T>, dim3(b.max_new, c.nkv, b.n_seqs), dim3(HD), 0, s, c, b, static_cast<T*>(k),
             static_cast<T*>(v), ld);
}

void launch_kvq8_read(const KvQ8Dev& c, const KvQ8Batch& b, bool f16, void* k, void* v, uint64_t ld, cudaStream_t s) {
  if (!b.n_seqs) return;
  if (c.hd == 128)
    f16 ? kvq8_read_t<128, __half>(c, b, k, v, ld, s) : kvq8_read_t<128, float>(c, b, k, v, ld, s);
  else
    f16 ? kvq8_read_t<64, __half>(c, b, k, v, ld, s) : kvq8_read_t<64, float>(c, b, k, v, ld, s);
}

uint64_t kvq8_attend_work(const KvQ8Dev& c, const KvQ8Batch& b) {
  (void)c;
  (void)b;
  return 16;
}

template <int HD, typename T>
static void kvq8_attend_t(const KvQ8Attend& a, cudaStream_t s) {
  launch_pdl(k_kvq8_attend<HD, T>, dim3(a.b.max_new, a.c.nkv * a.c.group, a.b.n_seqs), dim3(KQ_AT_THREADS), 0, s, a.c,
             a.b, static_cast<const T*>(a.q), a.ldq, static_cast<T*>(a.out), a.ldo, a.window, a.sinks, a.scale);
}

void launch_kvq8_attend(const KvQ8Attend& a, cudaStream_t s) {
  if (!a.b.n_seqs) return;
  if (a.c.hd == 128)
    a.f16 ? kvq8_attend_t<128, __half>(a, s) : kvq8_attend_t<128, float>(a, s);
  else
    a.f16 ? kvq8_attend_t<64, __half>(a, s) : kvq8_attend_t<64, float>(a, s);
}
