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
//
// What a kernel reads, the kernel before it may still be writing while this one
// is resident and waits (programmatic dependent launch).  So nothing here goes
// through the read-only path (ld.global.nc, which the compiler may also take for
// const __restrict__ pointers): that is for memory that stays the same for a
// kernel's whole life.
constexpr uint32_t KQ_PAGE = 64;   // positions of a page
constexpr uint32_t KQ_BLOCK = 16;  // positions that share a scale
constexpr uint32_t KQ_NB = KQ_PAGE / KQ_BLOCK;

// Byte offset inside a block of key (tok, dim).
template <int HD>
__device__ __forceinline__ uint32_t kq_koff(uint32_t tok, uint32_t dim) {
  return (tok >> 3) * 8 * HD + (dim >> 6) * 512 + (tok & 7) * 64 + (dim & 63);
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
  } else if (len == 0) {
    n = 0;  // an idle slot of a batch of fixed size
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

// Physical page of sequence i's page j as the table has it, and checked: -1
// (status) when it is none.
__device__ __forceinline__ int64_t kq_entry(const KvQ8Batch& b, uint32_t i, uint32_t j) {
  const int64_t at = (int64_t)i * b.max_pages + j;
  return b.pages ? (int64_t)b.pages[at] : at;
}
__device__ __forceinline__ int32_t kq_checked(const KvQ8Dev& c, int64_t p) {
  if (p < 0 || p >= c.n_pages) {
    atomicOr(c.status, KQ_BAD_PAGE);
    return -1;
  }
  return (int32_t)p;
}
__device__ __forceinline__ int32_t kq_page(const KvQ8Dev& c, const KvQ8Batch& b, uint32_t i, uint32_t j) {
  return kq_checked(c, kq_entry(b, i, j));
}

__device__ __forceinline__ float kq_ld(const float* p) { return *p; }
__device__ __forceinline__ float kq_ld(const __half* p) { return __half2float(*p); }
__device__ __forceinline__ void kq_st(float* p, float v) { *p = v; }
__device__ __forceinline__ void kq_st(__half* p, float v) { *p = __float2half_rn(v); }

// code + 128 of x at scale s (code 0 for an empty scale): round(x / s).
__device__ __forceinline__ uint32_t kq_code(float x, float s) {
  return 128 + (s > 0.f ? __float2int_rn(fminf(fmaxf(__fdiv_rn(x, s), -127.f), 127.f)) : 0);
}
// The same for n values, in the low bytes of w, without a division for each: with
// inv = RN(1 / s) and lo the rest of the inverse, q = RN(x inv + x lo) is within
// an ulp of x / s, so that RN(q + r inv) with the remainder r = x - s q, which
// is exact, is the correctly rounded quotient (Markstein's theorem).  Adding 1.5
// * 2^23 rounds it to an integer.  Scales whose remainders would lose bits are
// left to the division, in a loop: it seldom runs, and code that seldom runs has
// to be fetched first.
template <int N>
__device__ __forceinline__ void kq_codes(const float* x, float s, uint32_t* w) {
  constexpr float magic = 12582912.f + 128.f;
  if (s >= 7.8886090522101181e-31f && s <= 1.2676506002282294e30f) {  // 2^-100, 2^100
    const float inv = __frcp_rn(s), lo = __fmul_rn(__fmaf_rn(-s, inv, 1.f), inv);
#pragma unroll
    for (int i = 0; i < N; i++) {
      const float q = __fmaf_rn(x[i], inv, __fmul_rn(x[i], lo));
      w[i] = __float_as_uint(__fadd_rn(__fmaf_rn(__fmaf_rn(-s, q, x[i]), inv, q), magic));
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; i++) w[i] = 128;
    if (s > 0.f) {
      float z[N];
#pragma unroll
      for (int i = 0; i < N; i++) z[i] = x[i];
#pragma unroll 1
      for (int i = 0; i < N; i++) z[i] = __uint_as_float(kq_code(z[i], s));
#pragma unroll
      for (int i = 0; i < N; i++) w[i] = __float_as_uint(z[i]);
    }
  }
}
// The low bytes of four words.
__device__ __forceinline__ uint32_t kq_bytes(const uint32_t* w) {
  return __byte_perm(__byte_perm(w[0], w[1], 0x0040), __byte_perm(w[2], w[3], 0x0040), 0x5410);
}
// code + 128 of an older byte under a scale that grew by 1 / ratio
__device__ __forceinline__ uint32_t kq_recode(uint32_t byte, float ratio) {
  return 128 + __float2int_rn(__fmul_rn((float)((int)byte - 128), ratio));
}

__device__ __forceinline__ void kq_cp16(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}

// a * b + c of two pairs in one instruction, each rounded by itself.
__device__ __forceinline__ float2 kq_fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n .reg .b64 x, y, z;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n mov.b64 z, {%6, %7};\n"
      " fma.rn.f32x2 x, x, y, z;\n mov.b64 {%0, %1}, x;\n}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 kq_add2(float2 a, float2 b) {
  float2 d;
  asm("{\n .reg .b64 x, y;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n"
      " add.rn.f32x2 x, x, y;\n mov.b64 {%0, %1}, x;\n}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}

// N consecutive, aligned elements at p.
template <int N>
__device__ __forceinline__ void kq_ldn(const float* p, float* x) {
#pragma unroll
  for (int i = 0; i < N; i += 4) {
    if constexpr (N >= 4) {
      const float4 v = *reinterpret_cast<const float4*>(p + i);
      x[i] = v.x, x[i + 1] = v.y, x[i + 2] = v.z, x[i + 3] = v.w;
    } else {
      const float2 v = *reinterpret_cast<const float2*>(p);
      x[0] = v.x, x[1] = v.y;
    }
  }
}
template <int N>
__device__ __forceinline__ void kq_ldn(const __half* p, float* x) {
  uint32_t w[N / 2];
  if constexpr (N >= 8) {
#pragma unroll
    for (int i = 0; i < N / 8; i++) {
      const uint4 v = *reinterpret_cast<const uint4*>(p + 8 * i);
      w[4 * i] = v.x, w[4 * i + 1] = v.y, w[4 * i + 2] = v.z, w[4 * i + 3] = v.w;
    }
  } else if constexpr (N == 4) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    w[0] = v.x, w[1] = v.y;
  } else {
    w[0] = *reinterpret_cast<const uint32_t*>(p);
  }
#pragma unroll
  for (int i = 0; i < N / 2; i++) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    x[2 * i] = f.x, x[2 * i + 1] = f.y;
  }
}

// ---------------------------------------------------------------------------
// Append.  Grid (CTAs of a sequence, n_seqs).  An item is one block of one head;
// a CTA takes every gridDim.x-th of its sequence, its first half keys, its
// second half values, a thread two 16-byte pieces (a key thread's are the two
// halves of its rotated pairs).  Scale: the largest magnitude of the call's
// values / 127, and at least the block's older scale when positions before this
// call's are kept; those take the codes of the larger scale.  Bound by the bytes
// of k and v: the rows and rotation factors of the next two items are on their
// way to shared memory (cp.async, whole rows) while one is quantized.  Measured:
// 8192 positions of 8 heads of 128 in f32 (88 MB) 20.4 us (4.3 TB/s; 18.6 with
// the codes' arithmetic left out; loads straight to registers, a CTA an item,
// 23.3), 64 sequences of one position and 4 heads 4.8 us.  Rows of shared memory
// are 16 bytes apart in banks for the values' four positions a thread; the
// factors' pieces are permuted instead, since they are read 32 floats a thread.
// ---------------------------------------------------------------------------
template <int HD, typename T>
struct KqApStage {
  static constexpr uint32_t N = 16 / sizeof(T);        // elements of a piece
  static constexpr uint32_t CH = HD / N, RC = HD / 4;  // pieces of a row, of a position's factors
  uint4 k[KQ_BLOCK][CH + 1], v[KQ_BLOCK][CH + 1], rope[KQ_BLOCK][RC];
  // factor piece i of position tok
  __device__ __forceinline__ uint4& factors(uint32_t tok, uint32_t i) {
    return rope[tok][i ^ (i >> 3 & (HD / 32 - 1)) ^ (tok * (HD / 32) & 7)];
  }
};

constexpr uint32_t KQ_AP_STAGES = 2;
template <int HD>
constexpr uint32_t kq_ap_ctas() {
  return 512 / HD;  // CTAs per SM
}

template <int HD, typename T>
__global__ void __launch_bounds__(HD, kq_ap_ctas<HD>())
    k_kvq8_append(KvQ8Dev c, KvQ8Batch b, const T* k, const T* v, uint64_t ld, bool late) {
  using Stage = KqApStage<HD, T>;
  constexpr uint32_t CH = Stage::CH, RC = Stage::RC, N = Stage::N;
  extern __shared__ uint4 kq_dyn[];
  Stage* stages = reinterpret_cast<Stage*>(kq_dyn);
  __shared__ uint32_t s_top[2][HD / 32];
  if (!late) pdl_trigger();
  pdl_wait();
  if (late) pdl_trigger();  // what comes next may read what this kernel's predecessors wrote before it waits
  const KqSeq s = kq_seq(b, blockIdx.y, c.status);
  if (s.n_new == 0) return;
  if (c.rope && s.len > (int64_t)c.n_rope) {
    if (threadIdx.x == 0) atomicOr(c.status, KQ_BAD_POS);
    return;
  }
  constexpr uint32_t U = HD / 2, half = HD / 2;  // threads of a side
  const int32_t p0 = s.len - s.n_new, last = (s.len - 1) / (int32_t)KQ_BLOCK;
  struct Item {
    int32_t blk;
    uint32_t h;
  };
  const uint32_t dblk = gridDim.x / c.nkv, dh = gridDim.x % c.nkv;
  const auto after = [&](const Item& i) {
    const bool carry = i.h + dh >= c.nkv;
    return Item{i.blk + (int32_t)(dblk + carry), i.h + dh - (carry ? c.nkv : 0)};
  };
  const auto issue = [&](const Item& i, Stage& st) {
    if (i.blk <= last) {
      const int32_t base = i.blk * (int32_t)KQ_BLOCK;
      const int32_t a = max(p0 - base, 0), e = min(s.len - base, (int32_t)KQ_BLOCK);
      const int32_t y0 = threadIdx.x / CH, r0 = threadIdx.x / RC;
      // elements from this head's (position base, 0), which is in the buffer for positions [a, e) only
      const int64_t from =
          ((int64_t)s.row0 + base - p0 + y0) * (int64_t)ld + (int64_t)(i.h * HD + threadIdx.x % CH * N);
#pragma unroll
      for (uint32_t n = 0; n < KQ_BLOCK * CH / HD; n++) {
        const int32_t y = y0 + n * (HD / CH);
        if (y >= a && y < e) {
          const int64_t at = from + (int64_t)(n * (HD / CH)) * (int64_t)ld;
          kq_cp16(&st.k[y][threadIdx.x % CH], k + at);
          kq_cp16(&st.v[y][threadIdx.x % CH], v + at);
        }
      }
      if (c.rope) {
        const auto* f = c.rope + (int64_t)(base + r0) * half + threadIdx.x % RC * 2;
#pragma unroll
        for (uint32_t n = 0; n < KQ_BLOCK * RC / HD; n++) {
          const int32_t y = r0 + n * (HD / RC);
          if (y >= a && y < e) kq_cp16(&st.factors(y, threadIdx.x % RC), f + n * (HD / RC) * half);
        }
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  const uint32_t side = threadIdx.x / U, u = threadIdx.x % U;
  // keys: position tok, dims d .. d + 15 and half + d ..; values: positions 2t, 2t + 1, 8 + 2t, 9 + 2t of dims
  // 32 q + 8 i + g and HD / 2 + that
  const uint32_t tok = u / (HD / 32), d = u % (HD / 32) * 16, g = u >> 2 & 7, t = u & 3, q = u >> 5;
  const auto entry_of = [&](const Item& i) { return i.blk <= last ? kq_entry(b, blockIdx.y, i.blk / KQ_NB) : 0; };
  Item now{p0 / (int32_t)KQ_BLOCK + (int32_t)(blockIdx.x / c.nkv), blockIdx.x % c.nkv}, next = after(now);
  int64_t entry = entry_of(now);
  issue(now, stages[0]);
  issue(next, stages[1]);
  uint32_t turn = 0;
#pragma unroll 1
  for (; now.blk <= last; turn ^= 1) {
    const int32_t blk = now.blk, base = blk * (int32_t)KQ_BLOCK;
    const int32_t a = max(p0 - base, 0), e = min(s.len - base, (int32_t)KQ_BLOCK);  // new positions [a, e)
    const int32_t page = kq_checked(c, entry);
    const uint64_t at = ((uint64_t)max(page, 0) * c.nkv + now.h) * 2 + side;
    uint8_t* codes = c.codes + at * KQ_PAGE * HD + blk % KQ_NB * KQ_BLOCK * HD;
    float* sc = c.scales + at * KQ_NB + blk % KQ_NB;
    const bool old = a > 0 && page >= 0;  // positions before the call's are kept
    const float before = old ? *sc : 0.f;
    // this thread's pieces: keys in (tile of 8 positions, 64 dims), values in (tile of 32 dims)
    uint8_t* dst = codes + (side ? q * 512 + g * 64 + t * 16 : kq_koff<HD>(tok, d));
    const uint32_t step = side ? HD / 64 * 512 : kq_koff<HD>(0, half);
    uint4 kept[2];
    if (old) kept[0] = *reinterpret_cast<const uint4*>(dst), kept[1] = *reinterpret_cast<const uint4*>(dst + step);
    asm volatile("cp.async.wait_group %0;" ::"n"(KQ_AP_STAGES - 1) : "memory");
    __syncthreads();
    Stage& st = stages[turn];
    float x[32];
#pragma unroll
    for (int i = 0; i < 32; i++) x[i] = 0.f;
    if (side == 0) {
      if ((int32_t)tok >= a && (int32_t)tok < e) {
#pragma unroll
        for (uint32_t i = 0; i < 16 / N; i++) {
          kq_ldn<N>(reinterpret_cast<const T*>(&st.k[tok][d / N + i]), x + i * N);
          kq_ldn<N>(reinterpret_cast<const T*>(&st.k[tok][CH / 2 + d / N + i]), x + 16 + i * N);
        }
        if (c.rope) {
#pragma unroll
          for (uint32_t i = 0; i < 8; i++) {
            const uint4 w = st.factors(tok, d / 2 + i);
            const float f[4] = {__uint_as_float(w.x), __uint_as_float(w.y), __uint_as_float(w.z), __uint_as_float(w.w)};
#pragma unroll
            for (uint32_t n = 0; n < 2; n++) {
              const float m = x[2 * i + n], o = x[16 + 2 * i + n];
              x[2 * i + n] = __fsub_rn(__fmul_rn(m, f[2 * n]), __fmul_rn(o, f[2 * n + 1]));
              x[16 + 2 * i + n] = __fadd_rn(__fmul_rn(m, f[2 * n + 1]), __fmul_rn(o, f[2 * n]));
            }
          }
        }
      }
    } else {
#pragma unroll
      for (int32_t j = 0; j < 4; j++) {
        const int32_t y = (j >> 1) * 8 + 2 * t + (j & 1);
        if (y >= a && y < e) {
          const T* p = reinterpret_cast<const T*>(st.v[y]) + 32 * q + g;
#pragma unroll
          for (uint32_t i = 0; i < 8; i++) x[4 * i + j] = kq_ld(p + (i >> 2) * half + (i & 3) * 8);
        }
      }
    }
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < 32; i += 2) asm("max.NaN.abs.f32 %0, %0, %1, %2;" : "+f"(top) : "f"(x[i]), "f"(x[i + 1]));
    if (!(top <= 3.402823466e38f)) {
      if (page >= 0) atomicOr(c.status, KQ_NOT_FINITE);
      top = INFINITY;
    }
    // largest magnitude of the side; non-negative floats order like their bits, and a side with a value that is not
    // finite ends with infinity
    const uint32_t bits = __reduce_max_sync(0xffffffffu, __float_as_uint(top));
    if ((threadIdx.x & 31) == 0) s_top[turn][threadIdx.x >> 5] = bits;
    __syncthreads();  // the stage's rows are read, too
    now = next;
    next = after(next);
    issue(next, st);
    entry = entry_of(now);
    if (page < 0) continue;
    top = __uint_as_float(s_top[turn][side * (HD / 64)]);
    if (HD == 128) top = fmaxf(top, __uint_as_float(s_top[turn][side * 2 + 1]));
    float scale = __fdiv_rn(top, 127.f);
    if (a > 0 && !(scale > before)) scale = before;
    if (top == INFINITY) scale = __int_as_float(0x7fffffff);  // no number, not a wrong one
    const bool grew = a > 0 && scale > before;
    if (u == 0) *sc = scale;
    uint32_t w[32];
    kq_codes<32>(x, scale, w);
#pragma unroll
    for (int i = 0; i < 8; i++) w[i] = kq_bytes(w + 4 * i);
    if (a > 0) {
      const float ratio = __fdiv_rn(before, scale);
#pragma unroll
      for (int i = 0; i < 8; i++) {
        const uint32_t o = reinterpret_cast<const uint32_t*>(kept)[i];
#pragma unroll
        for (int32_t n = 0; n < 4; n++) {
          if ((side ? (n >> 1) * 8 + 2 * (int32_t)t + (n & 1) : (int32_t)tok) >= a) continue;
          const uint32_t byte = o >> (8 * n) & 255;
          w[i] = (w[i] & ~(255u << (8 * n))) | (grew ? kq_recode(byte, ratio) : byte) << (8 * n);
        }
      }
    }
    if (side == 0 && (int32_t)tok >= e) continue;
    *reinterpret_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
    *reinterpret_cast<uint4*>(dst + step) = make_uint4(w[4], w[5], w[6], w[7]);
  }
}

// ---------------------------------------------------------------------------
// Read-back: the rows a batch names as values.  Grid (blocks a sequence can
// touch, nkv, n_seqs): a CTA takes one block of one head; the pieces pass
// through shared memory, since a value piece holds four positions of four dims.
// Bound by the bytes: 8192 positions of 8 heads of 128 to f16 (51 MB) 11.3 us.
// ---------------------------------------------------------------------------
__device__ __forceinline__ void kq_st4(float* p, const float* x) {
  *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
}
__device__ __forceinline__ uint32_t kq_pack(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ void kq_st4(__half* p, const float* x) {
  *reinterpret_cast<uint2*>(p) = make_uint2(kq_pack(x[0], x[1]), kq_pack(x[2], x[3]));
}

template <int HD, typename T>
__global__ void __launch_bounds__(HD) k_kvq8_read(KvQ8Dev c, KvQ8Batch b, T* __restrict__ k, T* __restrict__ v,
                                                  uint64_t ld) {
  pdl_trigger();
  pdl_wait();
  const KqSeq s = kq_seq(b, blockIdx.z, c.status);
  const int32_t p0 = s.len - s.n_new;
  const int32_t blk = p0 / (int32_t)KQ_BLOCK + (int32_t)blockIdx.x, base = blk * (int32_t)KQ_BLOCK;
  if (s.n_new == 0 || base >= s.len) return;
  const int32_t page = kq_page(c, b, blockIdx.z, blk / KQ_NB);
  if (page < 0) return;
  const uint32_t h = blockIdx.y, u = threadIdx.x;
  const int32_t a = max(p0 - base, 0), e = min(s.len - base, (int32_t)KQ_BLOCK);
  __shared__ __align__(16) uint8_t tile[2][KQ_BLOCK][HD + 16];
  const uint64_t at = ((uint64_t)page * c.nkv + h) * 2;
  const uint8_t* codes = c.codes + at * KQ_PAGE * HD + blk % KQ_NB * KQ_BLOCK * HD;
  const uint4 kp = *reinterpret_cast<const uint4*>(codes + u * 16);
  const uint4 vp = *reinterpret_cast<const uint4*>(codes + KQ_PAGE * HD + u * 16);
  const float sc[2] = {c.scales[at * KQ_NB + blk % KQ_NB], c.scales[(at + 1) * KQ_NB + blk % KQ_NB]};
  const uint32_t g = u >> 2 & 7, t = u & 3, r = u >> 5;  // piece (g, t) of tile r
  *reinterpret_cast<uint4*>(&tile[0][r / (HD / 64) * 8 + g][r % (HD / 64) * 64 + t * 16]) = kp;
  const uint32_t w[4] = {vp.x, vp.y, vp.z, vp.w};
#pragma unroll
  for (int i = 0; i < 4; i++)
#pragma unroll
    for (int n = 0; n < 4; n++) tile[1][(n >> 1) * 8 + 2 * t + (n & 1)][r * 32 + 8 * i + g] = (uint8_t)(w[i] >> (8 * n));
  __syncthreads();
  // four dims a thread
#pragma unroll
  for (uint32_t x = u; x < 2 * KQ_BLOCK * HD / 4; x += HD) {
    const uint32_t side = x / (KQ_BLOCK * HD / 4), tok = x / (HD / 4) % KQ_BLOCK, d = x % (HD / 4) * 4;
    T* out = side ? v : k;
    if (!out || (int32_t)tok < a || (int32_t)tok >= e) continue;
    const uint32_t bytes = *reinterpret_cast<const uint32_t*>(&tile[side][tok][d]);
    float y[4];
#pragma unroll
    for (int n = 0; n < 4; n++) y[n] = __fmul_rn((float)((int)(bytes >> (8 * n) & 255) - 128), sc[side]);
    kq_st4(out + (uint64_t)(s.row0 + base + (int32_t)tok - p0) * ld + (uint64_t)h * HD + d, y);
  }
}

// ---------------------------------------------------------------------------
// Attention of few rows over long caches (k_kvq8_split + k_kvq8_merge).
//
// A segment is one KV head of one sequence for one group of 8 rows (row = (new
// token, query head of the KV head)).  It costs its pages plus KQ_SEG: loading
// the rows and writing the result take about as long.  All segments of the
// call, sequence by sequence, are cut into equal runs of that cost, one per
// CTA, so that ragged batches load the SMs evenly; a run may hold several
// segments, and a segment may span several runs: it is then written as partial
// results that k_kvq8_merge joins.  Where no sequence has more than
// KQ_WHOLE_PAGES pages every segment is a CTA of its own (k_kvq8_whole):
// nothing to plan and nothing to join.
//
// The cache bytes bound the kernel, so everything else has to fit under them.
// A CTA walks its pages two at a time, a warp taking 32 positions (two blocks)
// of one.  Codes become fp16 exactly (0x6400 | byte is 1024 + byte: one byte
// permute and one subtraction for two of them) and both products run on
// mma.m16n8k16: its 16 rows are the 8 query rows twice, as the high and the low
// part of an 11 + 11 bit split, so that the products keep f32's precision at no
// further cost.  The block's scales stay outside: the keys' multiplies the
// score, the values' the probability before its split.  The tensor cores'
// additions truncate, which over a long run would shrink the sums (2.6e-6 after
// 148 of them), so a warp's 32 positions are summed from zero and then added
// to the running sums in f32.
//
// Softmax: with scores x_t (base 2) and value scales v_t the running maximum m
// is taken over x_t + log v_t, the logarithm rounded down to an integer.  The
// weights w_t = 2^(x_t + log v_t - m) that multiply the codes, once the rest of
// v_t is multiplied in, are then at most 2, whatever the scales, and l = sum w_t
// 2^-log v_t is the denominator.  Its terms are found from the weights, not from
// 2^(x_t - m): with scales near the end of f32's range that is no normal number.
// m follows its maximum only when it falls behind by 2^8 (fp16 holds the weights
// up to there), so that the sums are seldom rescaled.  Scales under 2^-96 count as
// that in m, so that l stays finite.
//
// Measured with the merge: 16 sequences of 32768 positions, 8 KV heads of 128,
// 64 query heads (1.08 GB) 193 us, 5.6 TB/s (230 us where calls follow each
// other for seconds: the power limit); 48 ragged ones of up to 8192, 4 KV heads
// (208 MB) 53 us, of which about 5 pass before the first page has come and 3 in
// the merge.  Multiplies and sums in pairs took the last 2 %.  16 rows a segment,
// or more runs than the SMs hold at once, are not faster.
// ---------------------------------------------------------------------------
constexpr int KQ_SP_THREADS = 128;
constexpr uint32_t KQ_SP_STAGES = 2;     // tiles of a warp in shared memory
constexpr uint32_t KQ_SP_CTAS = 3;       // CTAs per SM
constexpr uint32_t KQ_SP_POS = 32;       // positions of a page that a warp takes
constexpr float KQ_LAG = 8.f;            // m is at most this far behind (base 2)
constexpr uint32_t KQ_SEG = 2;           // a segment's cost besides its pages, in pages
constexpr uint32_t KQ_WHOLE_PAGES = 4;
constexpr float KQ_MIN_SCALE = 1.2621774483536189e-29f;  // 2^-96

template <int HD>
struct KqSplitSmem {
  struct Stage {
    uint8_t k[KQ_SP_POS * HD], v[KQ_SP_POS * HD];
    float ks[2], vs[2];  // the two blocks' scales
  };
  union {
    Stage ring[KQ_SP_THREADS / 32][KQ_SP_STAGES];
    float acc[KQ_SP_THREADS / 32][8][HD + 8];  // the warps' sums at a segment's end
  };
  __half qh[8][HD], ql[8][HD];
  float rowf[8];
  uint32_t rowpos[8];
  float m[KQ_SP_THREADS / 32][8], l[KQ_SP_THREADS / 32][8];
  uint64_t scan[KQ_SP_THREADS / 32];
};

// The pages of a sequence that any of its new positions sees: virtual page v
// is page v below n_sink, lo + v - n_sink from there on; n pages in all.
struct KqSpan {
  uint32_t n_sink, lo, n;
  __device__ __forceinline__ uint32_t page(uint32_t v) const { return v < n_sink ? v : lo + v - n_sink; }
};
__device__ __forceinline__ KqSpan kq_span(uint32_t pmin, uint32_t pmax, uint32_t window, uint32_t sinks) {
  KqSpan r{0, 0, 0};
  if (window && pmin >= window) {
    r.lo = (pmin - window + 1) / KQ_PAGE;
    r.n_sink = min(sinks / KQ_PAGE + (sinks % KQ_PAGE != 0), r.lo);
  }
  r.n = r.n_sink + pmax / KQ_PAGE - r.lo + 1;
  return r;
}

// What the split form needs to know of a sequence.
struct KqPlan {
  KqSeq s;
  KqSpan span;
  uint32_t groups;  // row groups of one KV head
  __device__ __forceinline__ uint64_t cost(uint32_t nkv) const { return (uint64_t)groups * (span.n + KQ_SEG) * nkv; }
};
__device__ __forceinline__ KqPlan kq_plan(const KvQ8Dev& c, const KvQ8Batch& b, uint32_t i, uint32_t window,
                                          uint32_t sinks) {
  KqPlan p;
  p.s = kq_seq(b, i, c.status);
  if (p.s.n_new && c.rope && p.s.len > (int64_t)c.n_rope) {
    atomicOr(c.status, KQ_BAD_POS);
    p.s.n_new = 0;
  }
  p.groups = ((uint32_t)p.s.n_new * c.group + 7) / 8;
  p.span = KqSpan{0, 0, 0};
  if (p.s.n_new) p.span = kq_span(p.s.len - p.s.n_new, p.s.len - 1, window, sinks);
  return p;
}

__device__ __forceinline__ void kq_mma(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Four bytes (code + 128) as fp16 codes, exactly.
__device__ __forceinline__ void kq_halves(uint32_t w, uint32_t* h) {
  const __half2 off = __half2half2(__ushort_as_half(0x6480));  // 1024 + 128
  const uint32_t a = __byte_perm(w, 0x64646464u, 0x4140), b = __byte_perm(w, 0x64646464u, 0x4342);
  const __half2 x = __hsub2(*reinterpret_cast<const __half2*>(&a), off);
  const __half2 y = __hsub2(*reinterpret_cast<const __half2*>(&b), off);
  h[0] = *reinterpret_cast<const uint32_t*>(&x);
  h[1] = *reinterpret_cast<const uint32_t*>(&y);
}
// High and low parts of two values: hi = rn(x), lo = rn((x - hi) * 2^11).
__device__ __forceinline__ void kq_split2(float a, float b, uint32_t* hi, uint32_t* lo) {
  const __half2 h = __floats2half2_rn(a, b);
  const float2 f = __half22float2(h);
  *hi = *reinterpret_cast<const uint32_t*>(&h);
  const float2 r = kq_fma2(f, make_float2(-2048.f, -2048.f), make_float2(a * 2048.f, b * 2048.f));
  *lo = kq_pack(r.x, r.y);
}
__device__ __forceinline__ void kq_cp8(void* dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ float kq_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Length of a run: even, so that a run's pages come in pairs.
__device__ __forceinline__ uint64_t kq_per(uint64_t total, uint32_t runs) {
  return (total + 2ull * runs - 1) / (2ull * runs) * 2;
}

// Partial results: one slot per run end.  A slot holds the 8 rows' sums of
// codes, then their m, then their l.
template <int HD>
__host__ __device__ constexpr uint32_t kq_slot_floats() {
  return 8 * HD + 16;
}

template <int HD, typename T>
struct KqSplitArgs {
  KvQ8Dev c;
  KvQ8Batch b;
  const T* q;
  T* out;
  uint64_t ldq, ldo;
  uint32_t window, sinks;
  float scale;          // softmax scale * log2(e)
  XRun* runs;           // the result as run records too (every segment then goes through the merge), or null
  uint32_t run0;
  uint64_t* prefix;     // [n_seqs + 1] cost before each sequence (written by CTA 0)
  float* slots;         // [2 * gridDim.x]; k_kvq8_rows: the parts' results, kr_part_floats each
  uint32_t parts;       // k_kvq8_rows: CTAs of the same rows
  uint32_t after;       // k_kvq8_split: the predecessor is an append (late) of the batch's rows
};

// Rows of one segment: 16 threads a row, each N pairs.  get() starts the
// loads; put() rotates, scales the row by a power of two to a largest
// magnitude in [2^13, 2^14) and leaves its two parts in shared memory.  rowf
// undoes the power and holds the softmax scale; rowpos is the row's position
// (rows that are none are zeros at position phi; nothing of them is written).
template <int HD, typename T>
struct KqRows {
  static constexpr uint32_t half = HD / 2, N = half / 16;
  float x[2 * N], f[2 * N];
  bool live;
  uint32_t pos;
  __device__ __forceinline__ void get(const KqSplitArgs<HD, T>& a, const KqSeq& s, uint32_t kvh, uint32_t grp) {
    const uint32_t rr = grp * 8 + (threadIdx.x >> 4), j = rr / a.c.group, d = (threadIdx.x & 15) * N;
    live = j < (uint32_t)s.n_new;
    pos = s.len - s.n_new + j;
#pragma unroll
    for (uint32_t i = 0; i < 2 * N; i++) x[i] = 0.f, f[i] = i % 2 ? 0.f : 1.f;
    if (live) {
      const T* p = a.q + (uint64_t)(s.row0 + j) * a.ldq + (uint64_t)(kvh * a.c.group + rr % a.c.group) * HD + d;
      kq_ldn<N>(p, x);
      kq_ldn<N>(p + half, x + N);
      if (a.c.rope) {
        const float* r = reinterpret_cast<const float*>(a.c.rope + (uint64_t)pos * half + d);
        kq_ldn<N>(r, f);
        kq_ldn<N>(r + N, f + N);
      }
    }
  }
  __device__ __forceinline__ void put(const KqSplitArgs<HD, T>& a, KqSplitSmem<HD>& sm, uint32_t phi) {
    const uint32_t r = threadIdx.x >> 4, l16 = threadIdx.x & 15;
    float top = 0.f;
#pragma unroll
    for (uint32_t i = 0; i < N; i++) {
      const float u = x[i], w = x[N + i];
      if (a.c.rope) {
        x[i] = __fsub_rn(__fmul_rn(u, f[2 * i]), __fmul_rn(w, f[2 * i + 1]));
        x[N + i] = __fadd_rn(__fmul_rn(u, f[2 * i + 1]), __fmul_rn(w, f[2 * i]));
      }
      top = fmaxf(top, fmaxf(fabsf(x[i]), fabsf(x[N + i])));
    }
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    int e = (int)((__float_as_uint(top) >> 23) & 255) - 127;
    e = max(e, -100);
    const float up = __uint_as_float((uint32_t)(127 + 13 - e) << 23);  // e <= 128: the exponent stays positive
#pragma unroll
    for (uint32_t k = 0; k < 2; k++)
#pragma unroll
      for (uint32_t i = 0; i < N; i += 2) {
        uint32_t hi, lo;
        kq_split2(x[k * N + i] * up, x[k * N + i + 1] * up, &hi, &lo);
        *reinterpret_cast<uint32_t*>(&sm.qh[r][k * half + l16 * N + i]) = hi;
        *reinterpret_cast<uint32_t*>(&sm.ql[r][k * half + l16 * N + i]) = lo;
      }
    if (l16 == 0) {
      sm.rowf[r] = a.scale * __uint_as_float((uint32_t)(127 - 13 + e) << 23);
      sm.rowpos[r] = live ? pos : phi;
    }
  }
};

// A block's value scale v as rest * 2^log, inv = 2^-log; log from -96 (v below
// that: rest takes it, and 0) to 122.  For a v that is no number log is some number
// and rest is v.
struct KqScale {
  float log, inv, rest;
  __device__ __forceinline__ explicit KqScale(float v) {
    const uint32_t e = __float_as_uint(fminf(fmaxf(v, KQ_MIN_SCALE), 5.316911983139664e36f)) >> 23;  // 31 .. 249
    log = (float)((int)e - 127);
    inv = __uint_as_float((254 - e) << 23);
    rest = v * inv;
  }
};

// Pages v0 .. v0 + nv - 1 of a segment.  The result goes to out where these
// are all of its pages, else to the slot.  Called by the whole CTA.
template <int HD, typename T>
__device__ __forceinline__ void kq_segment(const KqSplitArgs<HD, T>& a, KqSplitSmem<HD>& sm, const KqPlan& p,
                                           uint32_t seq, uint32_t kvh, uint32_t grp, uint32_t v0, uint32_t nv,
                                           float* slot) {
    constexpr uint32_t KJ = HD / 64, NQ = HD / 32;
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    const uint32_t j0 = grp * 8 / a.c.group, j1 = min((grp * 8 + 7) / a.c.group, (uint32_t)p.s.n_new - 1);
    const uint32_t plo = p.s.len - p.s.n_new + j0, phi = p.s.len - p.s.n_new + j1;  // the group's positions
    KqRows<HD, T> rows;
    rows.get(a, p.s, kvh, grp);

    // the warp's tiles: pages v0 + 2 i + warp / 2, positions 32 (warp % 2) ..
    const uint32_t side = warp >> 1, sub = warp & 1;
    const uint32_t nt = (nv - min(nv, side) + 1) / 2;
    // pages of the next 32 of them, one per lane, and of the 32 after those
    auto page_of = [&](uint32_t i) {
      return max(kq_page(a.c, a.b, seq, p.span.page(v0 + min(2 * i + side, nv - 1))), 0);
    };
    int32_t pid = page_of(lane), pid_next = nt > 32 ? page_of(32 + lane) : 0;
    uint32_t issued = 0;
    auto tile_pos = [&](uint32_t i) { return p.span.page(v0 + 2 * i + side) * KQ_PAGE + sub * KQ_SP_POS; };
    // whether none of the group's rows sees any of the tile
    auto dead = [&](uint32_t pos) {
      return pos > phi ||
             (a.window && pos + KQ_SP_POS <= plo && plo - (pos + KQ_SP_POS - 1) >= a.window && pos >= a.sinks);
    };
    auto issue = [&]() {
      const uint32_t i = issued++;
      if (i < nt) {
        if (i && i % 32 == 0) {
          pid = pid_next;
          pid_next = i + 32 < nt ? page_of(i + 32 + lane) : 0;
        }
        const int32_t page = __shfl_sync(0xffffffffu, pid, i % 32);
        if (!dead(tile_pos(i))) {
          auto& st = sm.ring[warp][i % KQ_SP_STAGES];
          const uint64_t at = ((uint64_t)page * a.c.nkv + kvh) * 2;
          const uint8_t* src = a.c.codes + at * KQ_PAGE * HD + sub * KQ_SP_POS * HD + lane * 16;
#pragma unroll
          for (uint32_t x = 0; x < KQ_SP_POS * HD / 512; x++) {
            kq_cp16(st.k + x * 512 + lane * 16, src + x * 512);
            kq_cp16(st.v + x * 512 + lane * 16, src + KQ_PAGE * HD + x * 512);
          }
          if (lane < 2) kq_cp8(lane ? st.vs : st.ks, a.c.scales + (at + lane) * KQ_NB + sub * 2);
        }
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    for (uint32_t i = 0; i + 1 < KQ_SP_STAGES; i++) issue();

    rows.put(a, sm, phi);
    __syncthreads();
    uint32_t qh[KJ][8], ql[KJ][8];  // row g, dims 64j + 16t .. + 15
#pragma unroll
    for (uint32_t j = 0; j < KJ; j++)
#pragma unroll
      for (uint32_t i = 0; i < 8; i++) {
        qh[j][i] = *reinterpret_cast<const uint32_t*>(&sm.qh[g][j * 64 + t * 16 + 2 * i]);
        ql[j][i] = *reinterpret_cast<const uint32_t*>(&sm.ql[g][j * 64 + t * 16 + 2 * i]);
      }
    const float rowf = sm.rowf[g];
    const uint32_t rowpos = sm.rowpos[g];
    float m = -INFINITY, l = 0.f, o[HD / 8][2];
#pragma unroll
    for (int n = 0; n < HD / 8; n++) o[n][0] = o[n][1] = 0.f;

    for (uint32_t i = 0; i < nt; i++) {
      __syncwarp();  // every lane is done with the stage refilled next
      issue();
      asm volatile("cp.async.wait_group %0;" ::"n"(KQ_SP_STAGES - 1) : "memory");
      __syncwarp();  // every lane's copies of tile i have landed
      const uint32_t pos = tile_pos(i);
      if (dead(pos)) continue;
      auto& st = sm.ring[warp][i % KQ_SP_STAGES];
      float x[8];  // scores: block k / 4, positions 8 (k / 2 % 2) + 2t + k % 2 of it
#pragma unroll
      for (uint32_t n = 0; n < 4; n++) {
        float acc[4] = {};
#pragma unroll
        for (uint32_t j = 0; j < KJ; j++) {
          const uint4 kw = *reinterpret_cast<const uint4*>(st.k + n * 8 * HD + j * 512 + lane * 16);
          const uint32_t word[4] = {kw.x, kw.y, kw.z, kw.w};
#pragma unroll
          for (uint32_t y = 0; y < 4; y++) {
            uint32_t h[2];
            kq_halves(word[y], h);
            const uint32_t qa[4] = {qh[j][2 * y], ql[j][2 * y], qh[j][2 * y + 1], ql[j][2 * y + 1]};
            kq_mma(acc, qa, h[0], h[1]);
          }
        }
        const float f = st.ks[n >> 1] * rowf;
        x[2 * n] = fmaf(acc[2], 1.f / 2048.f, acc[0]) * f;
        x[2 * n + 1] = fmaf(acc[3], 1.f / 2048.f, acc[1]) * f;
      }
      uint32_t hidden = 0;
      if (pos + KQ_SP_POS - 1 > plo ||
          (a.window && pos + KQ_SP_POS > a.sinks && phi - pos >= a.window)) {  // some row does not see all of it
#pragma unroll
        for (int k = 0; k < 8; k++) {
          const uint32_t at = pos + (k >> 1) * 8 + 2 * t + (k & 1);
          const bool seen = at <= rowpos && (!a.window || rowpos - at < a.window || at < a.sinks);
          if (!seen) {
            x[k] = -INFINITY;
            hidden |= 1u << k;
          }
        }
      }
      // each block's scale as (1 .. 2) times a power of two
      const KqScale va(st.vs[0]), vb(st.vs[1]);
      float top = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])) + va.log,
                        fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])) + vb.log);
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      if (__any_sync(0xffffffffu, top > m + KQ_LAG)) {
        const float mn = fmaxf(m, top), f = mn == m ? 1.f : kq_exp2(m - mn);
        m = mn;
        l *= f;
#pragma unroll
        for (int n = 0; n < HD / 8; n++) o[n][0] *= f, o[n][1] *= f;
      }
      const float sub_m = m == -INFINITY ? 0.f : m, ca = va.log - sub_m, cb = vb.log - sub_m;
      float wv[8];
#pragma unroll
      for (int k = 0; k < 8; k++) wv[k] = kq_exp2(x[k] + (k < 4 ? ca : cb));
      l = fmaf((wv[0] + wv[1]) + (wv[2] + wv[3]), va.inv, l);
      l = fmaf((wv[4] + wv[5]) + (wv[6] + wv[7]), vb.inv, l);
#pragma unroll
      for (int k = 0; k < 8; k++) wv[k] *= k < 4 ? va.rest : vb.rest;
      if (hidden) {  // 0, whatever the scale of a block without positions of the sequence
#pragma unroll
        for (int k = 0; k < 8; k++)
          if (hidden >> k & 1) wv[k] = 0.f;
      }
      uint32_t pa[2][4];
#pragma unroll
      for (int k = 0; k < 4; k++) kq_split2(wv[2 * k], wv[2 * k + 1], &pa[k >> 1][2 * (k & 1)], &pa[k >> 1][2 * (k & 1) + 1]);
#pragma unroll
      for (uint32_t n = 0; n < NQ; n++) {
        const uint4 wa = *reinterpret_cast<const uint4*>(st.v + n * 512 + lane * 16);
        const uint4 wb = *reinterpret_cast<const uint4*>(st.v + KQ_BLOCK * HD + n * 512 + lane * 16);
        const uint32_t word[8] = {wa.x, wa.y, wa.z, wa.w, wb.x, wb.y, wb.z, wb.w};
#pragma unroll
        for (uint32_t k = 0; k < 4; k++) {
          float d[4] = {};
          uint32_t h[2];
          kq_halves(word[k], h);
          kq_mma(d, pa[0], h[0], h[1]);
          kq_halves(word[4 + k], h);
          kq_mma(d, pa[1], h[0], h[1]);
          const float2 sum = kq_fma2(make_float2(d[2], d[3]), make_float2(1.f / 2048.f, 1.f / 2048.f),
                                     make_float2(d[0], d[1]));
          const float2 y = kq_add2(make_float2(o[n * 4 + k][0], o[n * 4 + k][1]), sum);
          o[n * 4 + k][0] = y.x, o[n * 4 + k][1] = y.y;
        }
      }
    }
    l += __shfl_xor_sync(0xffffffffu, l, 1);
    l += __shfl_xor_sync(0xffffffffu, l, 2);
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();  // the ring is free
    if (t == 0) {
      sm.m[warp][g] = m;
      sm.l[warp][g] = l;
    }
#pragma unroll
    for (int n = 0; n < HD / 8; n++)
      *reinterpret_cast<float2*>(&sm.acc[warp][g][n * 8 + 2 * t]) = make_float2(o[n][0], o[n][1]);
    __syncthreads();
    const bool whole = nv == p.span.n && !a.runs;
    // a row is HD / 4 lanes, four dims each
    constexpr uint32_t L = HD / 4, RPP = KQ_SP_THREADS / L;  // lanes per row, rows per pass
#pragma unroll
    for (uint32_t r0 = 0; r0 < 8; r0 += RPP) {
      const uint32_t r = r0 + tid / L, d = tid % L * 4;
      const float top = fmaxf(fmaxf(sm.m[0][r], sm.m[1][r]), fmaxf(sm.m[2][r], sm.m[3][r]));
      float num[4] = {}, den = 0.f;
#pragma unroll
      for (int y = 0; y < KQ_SP_THREADS / 32; y++) {
        const float f = sm.m[y][r] == -INFINITY ? 0.f : kq_exp2(sm.m[y][r] - top);
        const float4 v = *reinterpret_cast<const float4*>(&sm.acc[y][r][d]);
        num[0] = fmaf(f, v.x, num[0]);
        num[1] = fmaf(f, v.y, num[1]);
        num[2] = fmaf(f, v.z, num[2]);
        num[3] = fmaf(f, v.w, num[3]);
        den = fmaf(f, sm.l[y][r], den);
      }
      if (whole) {
        const uint32_t rr = grp * 8 + r, j = rr / a.c.group;
        if (j < (uint32_t)p.s.n_new) {
#pragma unroll
          for (int i = 0; i < 4; i++) num[i] = den == 0.f ? 0.f : __fdiv_rn(num[i], den);
          kq_st4(a.out + (uint64_t)(p.s.row0 + j) * a.ldo + (uint64_t)(kvh * a.c.group + rr % a.c.group) * HD + d, num);
        }
      } else {
        kq_st4(slot + r * HD + d, num);
        if (d == 0) {
          slot[8 * HD + r] = top;
          slot[8 * HD + 8 + r] = den;
        }
      }
    }
}

template <int HD, typename T>
__global__ void __launch_bounds__(KQ_SP_THREADS, KQ_SP_CTAS) k_kvq8_split(const __grid_constant__ KqSplitArgs<HD, T> a) {
  extern __shared__ __align__(128) uint8_t smem_raw[];
  KqSplitSmem<HD>& sm = *reinterpret_cast<KqSplitSmem<HD>*>(smem_raw);
  const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  // Behind an append of the same rows only the CTAs that read the pages it wrote wait for it: those that go up to a
  // sequence's end (one new row, so the last page alone).
  if (!a.after) pdl_wait();
  pdl_trigger();  // after the wait: what the merge reads of the inputs is final when it starts
  // this CTA's run [w0, w1) of the call's cost and the sequence it starts in
  uint64_t total = 0, mine = 0;  // mine: the cost of sequence tid
  for (uint32_t i0 = 0; i0 < a.b.n_seqs; i0 += KQ_SP_THREADS) {
    const uint32_t i = i0 + tid;
    uint64_t n = i < a.b.n_seqs ? kq_plan(a.c, a.b, i, a.window, a.sinks).cost(a.c.nkv) : 0;
    if (i0 == 0) mine = n;
    for (int o = 16; o > 0; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
    if (lane == 0) sm.scan[warp] = n;
    __syncthreads();
    for (int w = 0; w < KQ_SP_THREADS / 32; w++) total += sm.scan[w];
    __syncthreads();
  }
  const uint64_t per = kq_per(total, gridDim.x);
  const uint64_t w0 = min(per * blockIdx.x, total), w1 = min(w0 + per, total);
  uint64_t before = 0, off = 0;
  uint32_t seq = 0;
  if (a.b.n_seqs > 1 || blockIdx.x == 0) {
    __shared__ uint32_t s_seq;
    __shared__ uint64_t s_off;
    for (uint32_t i0 = 0; i0 < a.b.n_seqs; i0 += KQ_SP_THREADS) {
      const uint32_t i = i0 + tid;
      const uint64_t n = i0 == 0              ? mine
                         : i < a.b.n_seqs ? kq_plan(a.c, a.b, i, a.window, a.sinks).cost(a.c.nkv)
                                          : 0;
      uint64_t inc = n;
      for (int o = 1; o < 32; o <<= 1) {
        const uint64_t x = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= (uint32_t)o) inc += x;
      }
      if (lane == 31) sm.scan[warp] = inc;
      __syncthreads();
      uint64_t base = before;
      for (uint32_t w = 0; w < KQ_SP_THREADS / 32; w++) {
        if (w < warp) base += sm.scan[w];
        before += sm.scan[w];
      }
      if (blockIdx.x == 0 && i < a.b.n_seqs) a.prefix[i] = base + inc - n;
      if (n && w0 >= base + inc - n && w0 < base + inc) {
        s_seq = i;
        s_off = w0 - (base + inc - n);
      }
      __syncthreads();
    }
    if (blockIdx.x == 0 && tid == 0) a.prefix[a.b.n_seqs] = total;
    if (w0 < w1) {
      seq = s_seq;
      off = s_off;
    }
  } else {
    off = w0;
  }
  if (w0 >= w1) return;

  KqPlan p = kq_plan(a.c, a.b, seq, a.window, a.sinks);
  for (uint64_t w = w0; w < w1;) {
    while (off >= p.cost(a.c.nkv)) {
      off -= p.cost(a.c.nkv);
      p = kq_plan(a.c, a.b, ++seq, a.window, a.sinks);  // w < total: a later sequence has segments
    }
    const uint32_t len = p.span.n + KQ_SEG, seg = (uint32_t)(off / len), u0 = (uint32_t)(off % len);
    const uint32_t u1 = (uint32_t)min((uint64_t)len, u0 + (w1 - w));
    const uint32_t v0 = max(u0, KQ_SEG) - KQ_SEG, v1 = max(u1, KQ_SEG) - KQ_SEG;
    if (v1 > v0) {
      if (a.after && v1 == p.span.n) pdl_wait();
      // a run has at most two pieces that are not whole segments: its first and its last
      kq_segment<HD, T>(a, sm, p, seq, seg / p.groups, seg % p.groups, v0, v1 - v0,
                        a.slots + (2ull * blockIdx.x + (w != w0)) * kq_slot_floats<HD>());
      __syncthreads();  // shared memory is reused by the next segment
    }
    w += u1 - u0;
    off += u1 - u0;
  }
}

// Every segment a CTA: grid (nkv * most row groups, n_seqs).
template <int HD, typename T>
__global__ void __launch_bounds__(KQ_SP_THREADS, KQ_SP_CTAS) k_kvq8_whole(const __grid_constant__ KqSplitArgs<HD, T> a) {
  extern __shared__ __align__(128) uint8_t smem_raw[];
  KqSplitSmem<HD>& sm = *reinterpret_cast<KqSplitSmem<HD>*>(smem_raw);
  pdl_trigger();
  pdl_wait();
  const KqPlan p = kq_plan(a.c, a.b, blockIdx.y, a.window, a.sinks);
  const uint32_t kvh = blockIdx.x % a.c.nkv, grp = blockIdx.x / a.c.nkv;
  if (grp < p.groups) kq_segment<HD, T>(a, sm, p, blockIdx.y, kvh, grp, 0, p.span.n, nullptr);
}

// Join the pieces of a segment that spans several runs.  Grid (rows of a KV
// head, nkv, n_seqs); four warps take every fourth piece, a lane HD / 32 dims.
constexpr int KQ_MG_THREADS = 128;
constexpr uint32_t KQ_MG_PIECES = 1024;  // runs of a call at most

template <int HD, typename T>
__global__ void __launch_bounds__(KQ_MG_THREADS) k_kvq8_merge(const __grid_constant__ KqSplitArgs<HD, T> a,
                                                              uint32_t runs) {
  const KqPlan p = kq_plan(a.c, a.b, blockIdx.z, a.window, a.sinks);  // inputs: final (see k_kvq8_split)
  const uint32_t rr = blockIdx.x, kvh = blockIdx.y, grp = rr / 8, r = rr % 8, j = rr / a.c.group;
  pdl_wait();
  if (j >= (uint32_t)p.s.n_new) return;
  const uint64_t per = kq_per(a.prefix[a.b.n_seqs], runs);
  const uint64_t s0 = a.prefix[blockIdx.z] + (uint64_t)(kvh * p.groups + grp) * (p.span.n + KQ_SEG);
  const uint64_t s1 = s0 + p.span.n + KQ_SEG;
  const uint32_t i0 = (uint32_t)((s0 + KQ_SEG) / per), n = (uint32_t)((s1 - 1) / per) - i0 + 1;
  if (n == 1 && !a.runs) return;  // written by the run itself
  __shared__ float wt[KQ_MG_PIECES];
  __shared__ float red[KQ_MG_THREADS / 32][HD], rden[KQ_MG_THREADS / 32], rtop[KQ_MG_THREADS / 32];
  const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  auto slot = [&](uint32_t i) {  // run i0 + i: its first piece unless the segment starts inside it
    return a.slots + (2ull * (i0 + i) + ((uint64_t)(i0 + i) * per < s0)) * kq_slot_floats<HD>();
  };
  float top = -INFINITY;
  for (uint32_t i = tid; i < n; i += KQ_MG_THREADS) {
    const float m = slot(i)[8 * HD + r];
    wt[i] = m;
    top = fmaxf(top, m);
  }
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (lane == 0) rtop[warp] = top;
  __syncthreads();
  top = fmaxf(fmaxf(rtop[0], rtop[1]), fmaxf(rtop[2], rtop[3]));
  float den = 0.f;
  for (uint32_t i = tid; i < n; i += KQ_MG_THREADS) {
    const float f = wt[i] == -INFINITY ? 0.f : kq_exp2(wt[i] - top);
    wt[i] = f;
    den = fmaf(f, slot(i)[8 * HD + 8 + r], den);
  }
  for (int o = 16; o > 0; o >>= 1) den += __shfl_xor_sync(0xffffffffu, den, o);
  if (lane == 0) rden[warp] = den;
  __syncthreads();
  constexpr int DPL = HD / 32;
  float acc[DPL] = {};
#pragma unroll 8
  for (uint32_t i = warp; i < n; i += KQ_MG_THREADS / 32) {
    const float* x = slot(i) + r * HD + lane * DPL;
#pragma unroll
    for (int d = 0; d < DPL; d++) acc[d] = fmaf(wt[i], x[d], acc[d]);
  }
#pragma unroll
  for (int d = 0; d < DPL; d++) red[warp][lane * DPL + d] = acc[d];
  __syncthreads();
  const uint32_t head = kvh * a.c.group + rr % a.c.group;
  if (tid < HD) {
    const float num = (red[0][tid] + red[1][tid]) + (red[2][tid] + red[3][tid]);
    den = (rden[0] + rden[1]) + (rden[2] + rden[3]);
    const float y = den == 0.f ? 0.f : __fdiv_rn(num, den);
    kq_st(a.out + (uint64_t)(p.s.row0 + j) * a.ldo + (uint64_t)head * HD + tid, y);
    wt[tid] = y;
  }
  if (a.runs) {  // one row: the input of the o_proj GEMV
    __syncthreads();
    if (tid < HD) values_to_runs(wt, HD, nullptr, a.runs, a.run0 + head * (HD / 16), tid, HD);
  }
}

// ---------------------------------------------------------------------------
// Attention of many rows (k_kvq8_rows): prompts, and pieces of them, on the
// fifth-generation tensor cores.
//
// A CTA takes 128 rows (row = (new token, query head of the KV head)) and walks
// the pages they see, two pages (128 positions) a step:
//   warps 0-3    a thread a row, even steps: scores from tensor memory, softmax,
//   and 4-7      weights back; odd steps
//   warps 8-11   turn the next step's values into an fp16 operand in shared
//                memory (UMMA K-major without swizzle, [dim][position]), then,
//                a thread a row, add the step's O from tensor memory to the
//                row's sums in registers
//   warps 12-14  turn the keys into their operand ([position][dim])
//   warp 15      one thread issues S = Q K^T, then O = P V (tcgen05.mma, M = 128)
//
// The products keep f32's precision as in k_kvq8_split: codes are exact in
// fp16, and Q and P are two fp16 parts each (Q's rows scaled to 2^13, P's
// weights by 2^13, so that the low part needs no scale of its own), multiplied
// one after the other into the same accumulator, the low part first, while
// what the tensor cores' additions cut off is small.  Over a long run that
// still adds up (3.8e-5 after 250 pages where O stayed in tensor memory):
// hence the sums in registers, and hence one CTA an SM.  Two pages a step: a
// product of 128 positions reads its 128 rows once instead of twice, which
// bounded it (1200 cycles for the scores of one page).  The two warpgroups of
// the softmax take turns, so that one's exponentials run under the other's
// maximum, conversion and waits; the running maximum goes from one to the
// other as soon as a step's is known.  Scores have three buffers in tensor
// memory, so that neither waits for the other's products, and a step's P takes
// the place of its S: of 32 positions, 16 columns for the high and 16 for the
// low parts.  P's positions go in the order of the value bytes (2t, 2t + 1, 8 +
// 2t, 9 + 2t for t = 0..3 of a block), which makes its pairs neighbours and the
// conversion of the values a plain copy.
//
// Where a call has fewer CTAs than the GPU has SMs, the steps of a CTA's rows
// are cut into `parts` of about equal length, a CTA each, whose results
// k_kvq8_join joins.
//
// Measured: 2048 rows of 28 heads behind 100 positions, 4 KV heads of 128, f32,
// 105 us (33 GFLOP, done twice for the two parts: 0.62 PFLOP/s; 104 with the keys
// through the read-only path, which is not theirs to take).  A step takes
// about 3800 cycles, 1300 of them the products': the softmax's and the
// conversions' instructions bound it (multiplies and sums in pairs gave 2 %).  A
// CTA's start and end take 27K of its 60K cycles on average: 10K until the rows
// are operands, 7K for the first step alone, 5K for the result.
// ---------------------------------------------------------------------------
constexpr uint32_t KR_M = 128;
constexpr uint32_t KR_THREADS = 512;
constexpr uint32_t KR_CONV = 3;            // warps that convert keys
constexpr uint32_t KR_POS = 2 * KQ_PAGE;   // positions of a step
constexpr float KR_LOGP = 13.f;            // the weights are scaled by 2^13
// registers: 128 a thread at launch, 512 for the four warpgroups together
constexpr int KR_REG_ACC = 200, KR_REG_OTHER = 104;
static_assert(3 * KR_REG_OTHER + KR_REG_ACC <= 512, "register shares");
constexpr uint32_t KR_NS = 3;              // scores in tensor memory
enum : uint32_t { KR_S = 0, KR_O = KR_NS * KR_POS };  // tensor memory: S 3 x 128 columns, O HD

template <int HD>
struct KrSmem {
  __half qh[KR_M * HD], ql[KR_M * HD], k[2][KR_POS * HD], v[2][KR_POS * HD];
  float rowf[KR_M], l[2][KR_M], last[2][KR_M], m[2][KR_M], alpha[4][KR_M];
  uint32_t rowpos[KR_M];
  uint64_t k_full[2], v_full[2], s_full[KR_NS], m_full[2], a_full[4], p_full[KR_NS], o_full, o_free, l_full, q_full, fin;
  uint32_t tmem;
};

template <uint32_t N>
__host__ __device__ constexpr uint32_t kr_idesc() {  // f16 x f16 -> f32, M = 128
  return (1u << 4) | ((N >> 3) << 17) | ((KR_M >> 4) << 24);
}
__device__ __forceinline__ void kr_mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, {%5, %5, %5, %5}, p;\n}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(acc), "r"(0u)
      : "memory");
}
__device__ __forceinline__ void kr_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, {%5, %5, %5, %5}, p;\n}\n" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(acc), "r"(0u)
      : "memory");
}
__device__ __forceinline__ void kr_ld16(uint32_t t, float* v) {
  uint32_t* r = reinterpret_cast<uint32_t*>(v);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, "
      "[%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(t)
      : "memory");
}
__device__ __forceinline__ void kr_ld32(uint32_t t, float* v) {
  uint32_t* r = reinterpret_cast<uint32_t*>(v);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, "
      "[%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(t)
      : "memory");
}
__device__ __forceinline__ void kr_st8(uint32_t t, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(t), "r"(r[0]),
               "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
// Wait for the loads; the registers go through it, so that nothing that uses
// them comes before it.
__device__ __forceinline__ void kr_wait_ld(float* v) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]),
                 "+f"(v[8]), "+f"(v[9]), "+f"(v[10]), "+f"(v[11]), "+f"(v[12]), "+f"(v[13]), "+f"(v[14]), "+f"(v[15])
               :
               : "memory");
}
__device__ __forceinline__ void kr_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

template <int N>
__device__ __forceinline__ void kr_regs_inc() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void kr_regs_dec() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

// Bits n of positions base .. base + 31 with lo <= base + n < hi.
__device__ __forceinline__ uint32_t kr_bits(uint32_t base, uint32_t lo, uint32_t hi) {
  const uint32_t a = lo > base ? min(lo - base, 32u) : 0u, b = hi > base ? min(hi - base, 32u) : 0u;
  const uint32_t below_b = b >= 32 ? 0xffffffffu : (1u << b) - 1, below_a = a >= 32 ? 0xffffffffu : (1u << a) - 1;
  return below_b & ~below_a;
}

// A part's result: the rows' sums, maxima and denominators.
template <int HD>
__host__ __device__ constexpr uint32_t kr_part_floats() {
  return KR_M * HD + 2 * KR_M;
}

// Page numbers of 32 pages, one per lane, and of the 32 after them.
struct KrPages {
  uint32_t cur, next;
  template <class F>
  __device__ __forceinline__ KrPages(F&& page_of, uint32_t lane) : cur(page_of(lane)), next(page_of(32 + lane)) {}
  // before the first use of page n, an even number
  template <class F>
  __device__ __forceinline__ void move(F&& page_of, uint32_t lane, uint32_t n) {
    if (n % 32 == 0) {
      cur = next;
      next = page_of(n + 32 + lane);
    }
  }
  __device__ __forceinline__ uint32_t at(uint32_t n) const { return __shfl_sync(0xffffffffu, cur, n % 32); }
};

// One row and 16 positions (a block) of a step.  f and lv are the block's score
// factor and the log2 of its value scale, bits the positions that the row sees
// (MASK).
template <bool MASK>
__device__ __forceinline__ float kr_top(const float* s, float f, float lv, uint32_t bits) {
  float x[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
  for (int k = 0; k < 16; k++)
    if (!MASK || (bits >> k & 1)) x[k & 3] = fmaxf(x[k & 3], s[k]);
  const float top = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
  return MASK && top == -INFINITY ? top : fmaf(top, f, lv);
}
// Weights to tensor memory at t, the high parts, and t + 16, the low ones.
__device__ __forceinline__ void kr_put(const float* x, uint32_t t) {
  uint32_t hi[8], lo[8];
#pragma unroll
  for (int c = 0; c < 8; c++) {  // pair c of the value order: positions 8 (c % 2) + 2 (c / 2), + 1
    const float a = x[8 * (c & 1) + (c & ~1)], z = x[8 * (c & 1) + (c & ~1) + 1];
    const __half2 h = __floats2half2_rn(a, z);
    const float2 g = __half22float2(h);
    hi[c] = *reinterpret_cast<const uint32_t*>(&h);
    const float2 r = kq_fma2(g, make_float2(-1.f, -1.f), make_float2(a, z));
    lo[c] = kq_pack(r.x, r.y);
  }
  kr_st8(t, hi);
  kr_st8(t + 16, lo);
}
// The block's weights 2^(f s - m) v 2^KR_LOGP: c = log2 v + KR_LOGP - m puts the
// scales into the exponent.  Returns their sum, which divided by v is the
// denominator's share, with the same 2^KR_LOGP as the sums have.
__device__ __forceinline__ float kr_weights(float* x, float f, float c) {
  float2 sum[2] = {};
#pragma unroll
  for (int k = 0; k < 16; k += 2) {
    const float2 e = kq_fma2(make_float2(x[k], x[k + 1]), make_float2(f, f), make_float2(c, c));
    x[k] = kq_exp2(e.x);
    x[k + 1] = kq_exp2(e.y);
    sum[k / 2 & 1] = kq_add2(sum[k / 2 & 1], make_float2(x[k], x[k + 1]));
  }
  return (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
}
// The same with positions that the row does not see, and for any scale: v is the
// block's, c goes by the larger of it and KQ_MIN_SCALE.
__device__ __forceinline__ float kr_weights_masked(float* x, float f, float c, float v, uint32_t bits) {
  const float less = v >= KQ_MIN_SCALE ? 1.f : v * (1.f / KQ_MIN_SCALE);  // a NaN stays one
  float sum = 0.f;
#pragma unroll
  for (int k = 0; k < 16; k++) {
    const bool seen = bits >> k & 1;
    const float w = kq_exp2(fmaf(x[k], f, c));
    sum += seen ? w : 0.f;
    x[k] = seen ? w * less : 0.f;  // 0 whatever the scale of a block not written yet
  }
  return sum;
}
template <int HD, typename T>
__global__ void __launch_bounds__(KR_THREADS, 1) k_kvq8_rows(const __grid_constant__ KqSplitArgs<HD, T> a) {
  extern __shared__ __align__(128) uint8_t smem_raw[];
  KrSmem<HD>& sm = *reinterpret_cast<KrSmem<HD>*>(smem_raw);
  constexpr uint32_t half = HD / 2, KJ = HD / 64;
  const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, kvh = blockIdx.y, seq = blockIdx.z;
  pdl_trigger();
  pdl_wait();
  const KqSeq s = kq_plan(a.c, a.b, seq, 0, 0).s;
  const uint32_t nrows = (uint32_t)s.n_new * a.c.group, tiles = (nrows + KR_M - 1) / KR_M;
  const uint32_t part = blockIdx.x % a.parts, tile = tiles - 1 - blockIdx.x / a.parts;  // the longest first
  if (blockIdx.x / a.parts >= tiles) return;
  const uint32_t r0 = tile * KR_M;
  const uint32_t p0 = s.len - s.n_new;
  const uint32_t plo = p0 + r0 / a.c.group, phi = p0 + min(r0 + KR_M - 1, nrows - 1) / a.c.group;
  const KqSpan span = kq_span(plo, phi, a.window, a.sinks);
  const uint32_t all = (span.n + 1) / 2, step0 = (uint32_t)((uint64_t)all * part / a.parts);
  const uint32_t steps = (uint32_t)((uint64_t)all * (part + 1) / a.parts) - step0;  // of this CTA
  float* slot = a.slots + (((uint64_t)(seq * a.c.nkv + kvh) * (gridDim.x / a.parts) + tile) * a.parts + part) *
                              kr_part_floats<HD>();
  if (steps == 0) {  // only where there are parts
    if (tid < KR_M) {
      slot[KR_M * HD + tid] = -INFINITY;
      slot[KR_M * HD + KR_M + tid] = 0.f;
    }
    return;
  }
  // page i of this CTA's steps; one past the last is the last again
  auto page_of = [&](uint32_t i) {
    return (uint32_t)max(kq_page(a.c, a.b, seq, span.page(min(2 * step0 + i, span.n - 1))), 0);
  };

  if (tid == 0) {
    for (int i = 0; i < 2; i++) {
      mbar_init(&sm.k_full[i], KR_CONV);
      mbar_init(&sm.v_full[i], 4);
      mbar_init(&sm.m_full[i], KR_M);
    }
    for (uint32_t i = 0; i < KR_NS; i++) {
      mbar_init(&sm.s_full[i], 1);
      mbar_init(&sm.p_full[i], KR_M);
    }
    for (int i = 0; i < 4; i++) mbar_init(&sm.a_full[i], KR_M);
    mbar_init(&sm.o_full, 1);
    mbar_init(&sm.o_free, KR_M);
    mbar_init(&sm.l_full, 2 * KR_M);
    mbar_init(&sm.q_full, 256);
    mbar_init(&sm.fin, 1);
    fence_barrier_init();
  }
  if (warp == 15) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&sm.tmem))
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tm = sm.tmem;
  bool ok = true;

  // With n buffers, step i uses buffer i % n, for the (i / n)th time: a wait for
  // step i's use is a wait for parity (i / n) % 2.  No barrier may get a whole
  // use ahead of a thread that still waits for the one before; beside each wait
  // stands what the next use needs from that thread.  A wait that runs out does
  // so by each lane's own clock: where a warp goes on together, its lanes agree
  // (__all_sync) before what needs them all.
  auto wait = [&](auto& bar, uint32_t i) {
    constexpr uint32_t n = sizeof(bar) / sizeof(uint64_t);
    return mbar_wait(reinterpret_cast<uint64_t*>(&bar) + i % n, (i / n) & 1);
  };

  if (warp >= 12) kr_regs_dec<KR_REG_OTHER>();
  if (warp == 15) {
    if (lane == 0) {
      auto scores = [&](uint32_t i) {
#pragma unroll 1
        for (uint32_t part = 0; part < 2; part++)
#pragma unroll
          for (uint32_t ks = 0; ks < HD / 16; ks++)
            kr_mma_ss(tm + KR_S + i % KR_NS * KR_POS,
                      umma_desc((part ? sm.qh : sm.ql) + ks * 2 * (KR_M / 8) * 64, (KR_M / 8) * 128, 128),
                      umma_desc(sm.k[i & 1] + ks * 2 * (KR_POS / 8) * 64, (KR_POS / 8) * 128, 128),
                      kr_idesc<KR_POS>(), part || ks);
        umma_commit(&sm.s_full[i % KR_NS]);
      };
      ok = mbar_wait(&sm.q_full, 0);
      for (uint32_t i = 0; i < min(2u, steps) && ok; i++) {
        ok = wait(sm.k_full, i);
        if (ok) scores(i);
      }
      for (uint32_t i = 0; i < steps && ok; i++) {
        // the scores of step i + 2 replace the weights of step i - 1 (what follows is issued by this thread)
        ok = i == 0 || wait(sm.o_full, i - 1);
        if (i + 2 < steps) {
          ok = ok && wait(sm.k_full, i + 2);  // next: keys of i + 4, after S of i + 2
          tc_fence_after();
          if (ok) scores(i + 2);
        }
        // next: values of i + 2, after O of i; weights of i + 3, after its S; O of step i read, after it is made
        ok = ok && wait(sm.v_full, i) && wait(sm.p_full, i) && (i == 0 || wait(sm.o_free, i - 1));
        tc_fence_after();
        if (!ok) break;
#pragma unroll 1
        for (uint32_t part = 0; part < 2; part++)
#pragma unroll
          for (uint32_t ks = 0; ks < KR_POS / 16; ks++)
            kr_mma_ts(tm + KR_O, tm + KR_S + i % KR_NS * KR_POS + ks / 2 * 32 + (part ? 0 : 16) + ks % 2 * 8,
                      umma_desc(sm.v[i & 1] + ks * 2 * (HD / 8) * 64, (HD / 8) * 128, 128), kr_idesc<HD>(),
                      part || ks);
        umma_commit(&sm.o_full);
      }
      umma_commit(&sm.fin);  // everything issued, whether or not a wait ran out
      ok = mbar_wait(&sm.fin, 0) && ok;
    }
    __syncwarp();
  } else if (warp >= 12) {
    const uint32_t cw = warp - 12, g = lane & 7;
    // a page's keys are 8 KJ tiles of 8 positions x 64 dims; the lane takes dims 16 (lane / 8) .. of position lane % 8.
    // A step's tiles are taken in turn by the warps, and loaded a step ahead.
    constexpr uint32_t NT = 16 * KJ, X = (NT + KR_CONV - 1) / KR_CONV;
    uint4 w[X];
    auto load = [&](uint32_t pa, uint32_t pb) {
      const uint8_t* src = a.c.codes + (uint64_t)kvh * 2 * KQ_PAGE * HD + g * 64 + (lane >> 3) * 16;
      const uint64_t stride = (uint64_t)a.c.nkv * 2 * KQ_PAGE * HD;
#pragma unroll
      for (uint32_t x = 0; x < X; x++) {
        const uint32_t tile = cw + KR_CONV * x;
        if (tile < NT)
          w[x] = *reinterpret_cast<const uint4*>(src + (tile < NT / 2 ? pa : pb) * stride + tile % (NT / 2) * 512);
      }
    };
    KrPages ids(page_of, lane);
    load(ids.at(0), ids.at(1));
    for (uint32_t i = 0; i < steps; i++) {
      ids.move(page_of, lane, 2 * i + 2);
      const uint32_t pa = ids.at(2 * i + 2), pb = ids.at(2 * i + 3);
      // S of step i - 2 has read the keys; next: S of i + 1, after its keys
      ok = __all_sync(0xffffffffu, i < 2 || wait(sm.s_full, i - 2));
      if (!ok) break;
      __half* dst = sm.k[i & 1] + g * 8;
#pragma unroll
      for (uint32_t x = 0; x < X; x++) {
        const uint32_t tile = cw + KR_CONV * x, kc = (tile % KJ * 4 + (lane >> 3)) * 2;
        if (tile >= NT) continue;
        uint32_t h[8];
        kq_halves(w[x].x, h);
        kq_halves(w[x].y, h + 2);
        kq_halves(w[x].z, h + 4);
        kq_halves(w[x].w, h + 6);
        __half* at = dst + (kc * (KR_POS / 8) + tile / KJ) * 64;
        *reinterpret_cast<uint4*>(at) = make_uint4(h[0], h[1], h[2], h[3]);
        *reinterpret_cast<uint4*>(at + (KR_POS / 8) * 64) = make_uint4(h[4], h[5], h[6], h[7]);
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.k_full[i & 1]);
      load(pa, pb);
    }
  } else if (warp >= 8) {
    kr_regs_inc<KR_REG_ACC>();
    const uint32_t row = tid & 127, lanes = ((warp & 3) * 32) << 16, cw = warp - 8, g = lane & 7;
    // a page's values are 8 KJ tiles of 16 positions x 32 dims, taken in pairs; the lane takes pieces t = 2 tp, 2 tp + 1
    // (tp = lane / 8 % 2) of dims 8 c + lane % 8 of the pair's tile lane / 16
    constexpr uint32_t X = KJ;  // pairs of a page for one of four warps
    uint4 w[2][2 * X];
    auto load = [&](uint32_t page, uint4* v) {
      const uint8_t* src = a.c.codes + (((uint64_t)page * a.c.nkv + kvh) * 2 + 1) * KQ_PAGE * HD + (lane >> 4) * 512 +
                           g * 64 + (lane >> 3 & 1) * 32;
#pragma unroll
      for (uint32_t x = 0; x < X; x++) {
        v[2 * x] = *reinterpret_cast<const uint4*>(src + (cw + 4 * x) * 1024);
        v[2 * x + 1] = *reinterpret_cast<const uint4*>(src + (cw + 4 * x) * 1024 + 16);
      }
    };
    KrPages ids(page_of, lane);
    auto values = [&](uint32_t i) {  // the operand of step i; the codes of step i + 1 start to load
#pragma unroll
      for (uint32_t page = 0; page < 2; page++)
#pragma unroll
        for (uint32_t x = 0; x < X; x++) {
          const uint32_t tile = 2 * (cw + 4 * x) + (lane >> 4), q = tile % (HD / 32);
          const uint32_t kc = page * 8 + tile / (HD / 32) * 2 + (lane >> 3 & 1);
          const uint4 va = w[page][2 * x], vb = w[page][2 * x + 1];
          const uint32_t u[4] = {va.x, va.y, va.z, va.w}, z[4] = {vb.x, vb.y, vb.z, vb.w};
#pragma unroll
          for (uint32_t c = 0; c < 4; c++) {
            uint32_t h[4];
            kq_halves(u[c], h);
            kq_halves(z[c], h + 2);
            *reinterpret_cast<uint4*>(sm.v[i & 1] + (kc * (HD / 8) + q * 4 + c) * 64 + g * 8) =
                make_uint4(h[0], h[1], h[2], h[3]);
          }
        }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.v_full[i & 1]);
      ids.move(page_of, lane, 2 * i + 2);
      load(ids.at(2 * i + 2), w[0]);
      load(ids.at(2 * i + 3), w[1]);
    };
    load(ids.at(0), w[0]);
    load(ids.at(1), w[1]);
    // the rows first: both share the issue slots, and the values are not needed before the first weights (105.4 ->
    // 104.2 us for 2048 rows)
    ok = __all_sync(0xffffffffu, mbar_wait(&sm.q_full, 0));
    values(0);
    float acc[HD];
#pragma unroll
    for (int d = 0; d < HD; d++) acc[d] = 0.f;
    for (uint32_t i = 0; i < steps && ok; i++) {
      if (i + 1 < steps) values(i + 1);  // O of step i - 1, the operand's last reader, is done: it has been added
      // next: alpha of i + 4, after S of i + 4, after O of i + 1, after O of i has been read; O of i + 1, after that too
      ok = __all_sync(0xffffffffu, wait(sm.a_full, i) && wait(sm.o_full, i));
      if (!ok) break;
      tc_fence_after();
      const float alpha = sm.alpha[i & 3][row];
#pragma unroll
      for (int d = 0; d < HD; d += 16) {
        float o[16];
        kr_ld16(tm + lanes + KR_O + d, o);
        kr_wait_ld(o);
#pragma unroll
        for (int k = 0; k < 16; k++) acc[d + k] = fmaf(acc[d + k], alpha, o[k]);
      }
      tc_fence_before();
      mbar_arrive(&sm.o_free);
    }
    ok = __all_sync(0xffffffffu, ok && mbar_wait(&sm.l_full, 0));
    // The result goes out through shared memory (the operands': every product is done), a warp a row at a time.  Each
    // warpgroup's denominator goes by the maximum of its own last step, the sums by that of the last.
    if (ok) {
      const float m0 = sm.last[0][row], m1 = sm.last[1][row], top = fmaxf(m0, m1);
      // without a maximum l is 0, or a NaN: maxima pass over scores that are no numbers
      const float l = (m0 == -INFINITY ? sm.l[0][row] : sm.l[0][row] * kq_exp2(m0 - top)) +
                      (m1 == -INFINITY ? sm.l[1][row] : sm.l[1][row] * kq_exp2(m1 - top));
      float inv = l == 0.f ? 0.f : __fdiv_rn(1.f, l);  // 2^KR_LOGP is in the sums and in l
      if (a.parts > 1) {
        inv = 1.f;
        slot[KR_M * HD + row] = top;
        slot[KR_M * HD + KR_M + row] = l;
      }
      constexpr uint32_t ST = HD + 4;  // floats of a row: rows start in different banks
      static_assert(KR_M * ST * 4 <= sizeof(sm.k) + sizeof(sm.v), "room for the result");
      float* tile = reinterpret_cast<float*>(&sm.k[0][0]) + (warp & 3) * 32 * ST;  // this warp's 32 rows
#pragma unroll
      for (int d = 0; d < HD; d += 4) {
#pragma unroll
        for (int k = 0; k < 4; k++) acc[d + k] = l == 0.f ? 0.f : acc[d + k] * inv;
        kq_st4(tile + lane * ST + d, acc + d);
      }
      __syncwarp();
      constexpr uint32_t L = HD / 4, RP = 32 / L;  // lanes of a row, rows at a time
      const uint32_t mine = r0 + row, j = mine / a.c.group;
      const uint64_t off = (uint64_t)(s.row0 + j) * a.ldo + (uint64_t)(kvh * a.c.group + mine - j * a.c.group) * HD;
      const uint32_t first = (warp & 3) * 32, live = nrows > r0 + first ? min(nrows - r0 - first, 32u) : 0;
#pragma unroll 4
      for (uint32_t r = 0; r < 32; r += RP) {
        const uint32_t at = r + lane / L, d = lane % L * 4;
        const uint64_t to = __shfl_sync(0xffffffffu, off, at);
        float v[4];
        kq_ldn<4>(tile + at * ST + d, v);
        if (at >= live) continue;
        if (a.parts > 1)
          kq_st4(slot + (first + at) * HD + d, v);
        else
          kq_st4(a.out + to + d, v);
      }
    }
  } else {
    kr_regs_dec<KR_REG_OTHER>();
    // The rows, rotated, scaled to 2^13 and split.  A warp takes eight rows, a lane 8 dims of one at a time (and the 8
    // they are paired with): eight lanes then store one core matrix.
    {
      constexpr uint32_t CH = half / 32;
#pragma unroll 1
      for (uint32_t rg = warp; rg < KR_M / 8; rg += 8) {
        const uint32_t r = rg * 8 + (lane & 7), rr = r0 + r, j = rr / a.c.group;
        const T* p = a.q + (uint64_t)(s.row0 + j) * a.ldq + (uint64_t)(kvh * a.c.group + rr - j * a.c.group) * HD;
        const float* cs = reinterpret_cast<const float*>(a.c.rope + (uint64_t)(p0 + j) * half);
        float x[CH][16], f[CH][16], top = 0.f;
#pragma unroll
        for (uint32_t ch = 0; ch < CH; ch++) {
          const uint32_t d = (lane >> 3) * 8 + ch * 32;
#pragma unroll
          for (uint32_t i = 0; i < 16; i++) x[ch][i] = 0.f, f[ch][i] = i % 2 ? 0.f : 1.f;
          if (rr < nrows) {
            kq_ldn<8>(p + d, x[ch]);
            kq_ldn<8>(p + half + d, x[ch] + 8);
            if (a.c.rope) kq_ldn<16>(cs + 2 * d, f[ch]);
          }
        }
#pragma unroll
        for (uint32_t ch = 0; ch < CH; ch++)
#pragma unroll
          for (uint32_t i = 0; i < 8; i++) {
            const float u = x[ch][i], w = x[ch][8 + i];
            if (a.c.rope) {
              x[ch][i] = __fsub_rn(__fmul_rn(u, f[ch][2 * i]), __fmul_rn(w, f[ch][2 * i + 1]));
              x[ch][8 + i] = __fadd_rn(__fmul_rn(u, f[ch][2 * i + 1]), __fmul_rn(w, f[ch][2 * i]));
            }
            top = fmaxf(top, fmaxf(fabsf(x[ch][i]), fabsf(x[ch][8 + i])));
          }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
        const int e = max((int)((__float_as_uint(top) >> 23) & 255) - 127, -100);
        // a negative softmax scale turns the row, so that factors are not negative
        const float up = copysignf(__uint_as_float((uint32_t)(127 + 13 - e) << 23), a.scale);
#pragma unroll
        for (uint32_t ch = 0; ch < CH; ch++)
#pragma unroll
          for (uint32_t k = 0; k < 2; k++) {
            const uint32_t kc = (lane >> 3) + ch * 4 + k * (half / 8), at = (kc * (KR_M / 8) + rg) * 64 + (lane & 7) * 8;
            uint32_t hi[4], lo[4];
#pragma unroll
            for (uint32_t i = 0; i < 4; i++) {
              const float u = x[ch][8 * k + 2 * i] * up, w = x[ch][8 * k + 2 * i + 1] * up;
              const __half2 h = __floats2half2_rn(u, w);
              const float2 g = __half22float2(h);
              hi[i] = *reinterpret_cast<const uint32_t*>(&h);
              lo[i] = kq_pack(u - g.x, w - g.y);
            }
            *reinterpret_cast<uint4*>(&sm.qh[at]) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
            *reinterpret_cast<uint4*>(&sm.ql[at]) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
          }
        if (lane < 8) {
          sm.rowf[r] = fabsf(a.scale) * __uint_as_float((uint32_t)(127 - 13 + e) << 23);
          sm.rowpos[r] = rr < nrows ? p0 + j : phi;  // a row that is none: zeros, not written
        }
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      mbar_arrive(&sm.q_full);
    }
    ok = __all_sync(0xffffffffu, mbar_wait(&sm.q_full, 0));
    const uint32_t row = tid & 127, wg = warp >> 2, lanes = ((warp & 3) * 32) << 16, side = lane >> 2 & 1;
    const float rowf = sm.rowf[row];
    const uint32_t rowpos = sm.rowpos[row];
    float m = -INFINITY, l = 0.f;
    // a step's scales, one block a lane (lanes 0-7 and their likes), loaded two steps ahead
    auto scales = [&](uint32_t page, float* ks, float* vs) {
      const float* p = a.c.scales + ((uint64_t)page * a.c.nkv + kvh) * 2 * KQ_NB + (lane & 3);
      *ks = p[0];
      *vs = p[KQ_NB];
    };
    float ks_next, vs_next;
    scales(page_of(2 * wg + side), &ks_next, &vs_next);
    uint32_t next = page_of(2 * wg + 4 + side);
    for (uint32_t i = wg; i < steps && ok; i += 2) {
      const float ks = ks_next, vs = vs_next, lv = __log2f(fmaxf(vs, KQ_MIN_SCALE));
      scales(next, &ks_next, &vs_next);
      next = page_of(2 * i + 8 + side);
      ok = __all_sync(0xffffffffu, wait(sm.s_full, i));  // next: S of i + 3, after O of i, after this step's weights
      if (!ok) break;
      tc_fence_after();
      const uint32_t t = tm + lanes + KR_S + i % KR_NS * KR_POS;
      const uint32_t at = 2 * (step0 + i);
      const bool none = at + 1 >= span.n;  // the last step has one page
      const uint32_t pos[2] = {span.page(at) * KQ_PAGE, span.page(at + 1) * KQ_PAGE};
      bool masked = none;
#pragma unroll
      for (int k = 0; k < 2; k++)
        masked = masked || pos[k] + KQ_PAGE - 1 > plo ||
                 (a.window && pos[k] + KQ_PAGE > a.sinks && phi - min(pos[k], phi) >= a.window);
      // the positions 32 j .. of the step that the row sees
      auto vis = [&](uint32_t j) {
        const uint32_t base = (j < 2 ? pos[0] : pos[1]) + 32 * (j & 1), end = rowpos + 1;
        uint32_t bits = kr_bits(base, a.window && end > a.window ? end - a.window : 0, end);
        if (a.window) bits |= kr_bits(base, 0, min(a.sinks, end));
        return none && j >= 2 ? 0u : bits;
      };
      float top = -INFINITY;
#pragma unroll 1
      for (uint32_t j = 0; j < 4; j++) {
        const float f0 = __shfl_sync(0xffffffffu, ks, 2 * j) * rowf, f1 = __shfl_sync(0xffffffffu, ks, 2 * j + 1) * rowf;
        const float a0 = __shfl_sync(0xffffffffu, lv, 2 * j), a1 = __shfl_sync(0xffffffffu, lv, 2 * j + 1);
        float x[32];
        kr_ld32(t + 32 * j, x);
        kr_wait_ld(x);
        kr_wait_ld(x + 16);
        if (masked) {
          const uint32_t bits = vis(j);
          top = fmaxf(top, fmaxf(kr_top<true>(x, f0, a0, bits), kr_top<true>(x + 16, f1, a1, bits >> 16)));
        } else {
          top = fmaxf(top, fmaxf(kr_top<false>(x, f0, a0, 0), kr_top<false>(x + 16, f1, a1, 0)));
        }
      }
      float before = -INFINITY;
      if (i) {  // next: the maximum of i + 1, after this step's
        ok = __all_sync(0xffffffffu, wait(sm.m_full, i - 1));
        if (!ok) break;
        before = sm.m[(i - 1) & 1][row];
      }
      const float mn = fmaxf(before, top), sub = mn == -INFINITY ? 0.f : mn;
      sm.m[i & 1][row] = mn;
      mbar_arrive(&sm.m_full[i & 1]);
      sm.alpha[i & 3][row] = mn == before ? 1.f : kq_exp2(before - mn);  // step i - 4's has been read: O of i - 3 is made
      mbar_arrive(&sm.a_full[i & 3]);
      l = mn == m ? l : l * kq_exp2(m - mn);
      m = mn;
#pragma unroll 1
      for (uint32_t j = 0; j < 4; j++) {
        const float f0 = __shfl_sync(0xffffffffu, ks, 2 * j) * rowf, f1 = __shfl_sync(0xffffffffu, ks, 2 * j + 1) * rowf;
        const float v0 = __shfl_sync(0xffffffffu, vs, 2 * j), v1 = __shfl_sync(0xffffffffu, vs, 2 * j + 1);
        const float a0 = __shfl_sync(0xffffffffu, lv, 2 * j), a1 = __shfl_sync(0xffffffffu, lv, 2 * j + 1);
        float x[32];
        kr_ld32(t + 32 * j, x);
        kr_wait_ld(x);
        kr_wait_ld(x + 16);
        const float lp = KR_LOGP - sub;
        if (!masked && v0 >= KQ_MIN_SCALE && v1 >= KQ_MIN_SCALE) {  // else the scales may be no numbers
          l = fmaf(kr_weights(x, f0, a0 + lp), __fdividef(1.f, v0), l);
          l = fmaf(kr_weights(x + 16, f1, a1 + lp), __fdividef(1.f, v1), l);
        } else {
          const uint32_t bits = masked ? vis(j) : 0xffffffffu;
          l = fmaf(kr_weights_masked(x, f0, a0 + lp, v0, bits), __fdividef(1.f, fmaxf(v0, KQ_MIN_SCALE)), l);
          l = fmaf(kr_weights_masked(x + 16, f1, a1 + lp, v1, bits >> 16), __fdividef(1.f, fmaxf(v1, KQ_MIN_SCALE)), l);
        }
        kr_put(x, t + 32 * j);
        kr_put(x + 16, t + 32 * j + 8);
      }
      kr_wait_st();
      tc_fence_before();
      mbar_arrive(&sm.p_full[i % KR_NS]);
    }
    sm.l[wg][row] = l;
    sm.last[wg][row] = m;
    mbar_arrive(&sm.l_full);
  }
  if (!ok && lane == 0) atomicOr(a.c.status, KQ_TIMEOUT);
  tc_fence_before();
  __syncthreads();
  if (warp == 15) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tm) : "memory");
}

// Join the parts of k_kvq8_rows: a warp a row, a lane HD / 32 dims.  Grid (rows
// of a KV head / 4, nkv, n_seqs).
constexpr int KR_JOIN_THREADS = 128;

template <int HD, typename T>
__global__ void __launch_bounds__(KR_JOIN_THREADS) k_kvq8_join(const __grid_constant__ KqSplitArgs<HD, T> a,
                                                               uint32_t tiles) {
  pdl_trigger();
  pdl_wait();
  const KqSeq s = kq_plan(a.c, a.b, blockIdx.z, 0, 0).s;
  const uint32_t rr = blockIdx.x * (KR_JOIN_THREADS / 32) + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  const uint32_t kvh = blockIdx.y, j = rr / a.c.group, row = rr % KR_M;
  if (j >= (uint32_t)s.n_new) return;
  const float* slot = a.slots + ((uint64_t)(blockIdx.z * a.c.nkv + kvh) * tiles + rr / KR_M) * a.parts *
                                    kr_part_floats<HD>();
  float top = -INFINITY;
  for (uint32_t i = 0; i < a.parts; i++) top = fmaxf(top, slot[(uint64_t)i * kr_part_floats<HD>() + KR_M * HD + row]);
  constexpr int DPL = HD / 32;
  float acc[DPL] = {}, den = 0.f;
#pragma unroll 4
  for (uint32_t i = 0; i < a.parts; i++) {
    const float* p = slot + (uint64_t)i * kr_part_floats<HD>();
    const float m = p[KR_M * HD + row], l = p[KR_M * HD + KR_M + row];
    if (m == -INFINITY) {  // its sums may not be there; l is 0 where the row saw nothing, else a NaN
      den += l;
      continue;
    }
    const float f = kq_exp2(m - top);
    float x[DPL];
    kq_ldn<DPL>(p + row * HD + lane * DPL, x);
    den = fmaf(f, l, den);
#pragma unroll
    for (int d = 0; d < DPL; d++) acc[d] = fmaf(f, x[d], acc[d]);
  }
  T* out = a.out + (uint64_t)(s.row0 + j) * a.ldo + (uint64_t)(kvh * a.c.group + rr % a.c.group) * HD + lane * DPL;
#pragma unroll
  for (int d = 0; d < DPL; d++) kq_st(out + d, den == 0.f ? 0.f : __fdiv_rn(acc[d], den));
}

// ---------------------------------------------------------------------------
// Launches
// ---------------------------------------------------------------------------
// Runs f once for each device (a kernel's attributes hold per device); devices
// past the 64 bits run it every time.
template <class F>
static void kvq8_once(std::atomic<uint64_t>& ready, F&& f) {
  int dev = 0;
  CK(cudaGetDevice(&dev));
  const uint64_t bit = dev < 64 ? 1ull << dev : 0;
  if (ready.load(std::memory_order_acquire) & bit) return;
  f();
  ready.fetch_or(bit, std::memory_order_release);
}

// Blocks that max_new consecutive positions can touch.
static uint32_t kvq8_blocks(const KvQ8Batch& b) { return (b.max_new + 2 * KQ_BLOCK - 2) / KQ_BLOCK; }

template <int HD, typename T>
static void kvq8_append_t(const KvQ8Dev& c, const KvQ8Batch& b, const void* k, const void* v, uint64_t ld, bool late,
                          cudaStream_t s) {
  using Stages = KqApStage<HD, T>[KQ_AP_STAGES];
  static std::atomic<uint64_t> ready{0};
  kvq8_once(ready, [&] {
    CK(cudaFuncSetAttribute(k_kvq8_append<HD, T>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(Stages)));
  });
  // one sequence: every SM filled once, a CTA taking as many items as that leaves it (8192 positions of 8 heads 20.4 us;
  // an item a CTA 23.0).  Several may be shorter than max_new: an item a CTA keeps the SMs even (ragged prompts 7 us;
  // cut like one sequence 10), which two equal ones of 8192 pay for (41 us)
  const uint64_t items = (uint64_t)kvq8_blocks(b) * c.nkv, slots = (uint64_t)num_sms() * kq_ap_ctas<HD>();
  const uint64_t per = b.n_seqs > 1 ? 1 : (items + slots - 1) / slots;
  launch_pdl(k_kvq8_append<HD, T>, dim3((unsigned)((items + per - 1) / per), b.n_seqs), dim3(HD), sizeof(Stages), s, c,
             b, static_cast<const T*>(k), static_cast<const T*>(v), ld, late);
}

void launch_kvq8_append(const KvQ8Dev& c, const KvQ8Batch& b, bool f16, const void* k, const void* v, uint64_t ld,
                        cudaStream_t s, bool late) {
  if (!b.n_seqs) return;
  if (c.hd == 128)
    f16 ? kvq8_append_t<128, __half>(c, b, k, v, ld, late, s) : kvq8_append_t<128, float>(c, b, k, v, ld, late, s);
  else
    f16 ? kvq8_append_t<64, __half>(c, b, k, v, ld, late, s) : kvq8_append_t<64, float>(c, b, k, v, ld, late, s);
}

template <int HD, typename T>
static void kvq8_read_t(const KvQ8Dev& c, const KvQ8Batch& b, void* k, void* v, uint64_t ld, cudaStream_t s) {
  launch_pdl(k_kvq8_read<HD, T>, dim3(kvq8_blocks(b), c.nkv, b.n_seqs), dim3(HD), 0, s, c, b, static_cast<T*>(k),
             static_cast<T*>(v), ld);
}

void launch_kvq8_read(const KvQ8Dev& c, const KvQ8Batch& b, bool f16, void* k, void* v, uint64_t ld, cudaStream_t s) {
  if (!b.n_seqs) return;
  if (c.hd == 128)
    f16 ? kvq8_read_t<128, __half>(c, b, k, v, ld, s) : kvq8_read_t<128, float>(c, b, k, v, ld, s);
  else
    f16 ? kvq8_read_t<64, __half>(c, b, k, v, ld, s) : kvq8_read_t<64, float>(c, b, k, v, ld, s);
}

// Runs of the split form: every SM filled, never more than there can be tiles.
static uint32_t kvq8_runs(const KvQ8Dev& c, const KvQ8Batch& b) {
  const uint64_t most = (uint64_t)b.n_seqs * c.nkv * (((uint64_t)b.max_new * c.group + 7) / 8) * (b.max_pages + KQ_SEG);
  return (uint32_t)std::min<uint64_t>({most, (uint64_t)num_sms() * KQ_SP_CTAS, KQ_MG_PIECES});
}
static uint64_t kvq8_prefix_bytes(const KvQ8Batch& b) { return ((uint64_t)b.n_seqs + 1) * 8 + 15 & ~15ull; }

// CTAs of the same rows: enough to fill the SMs, each with two steps (four
// pages) or more of the longest sequence there can be.
static uint32_t kvq8_tiles(const KvQ8Dev& c, const KvQ8Batch& b) {
  return (uint32_t)(((uint64_t)b.max_new * c.group + KR_M - 1) / KR_M);
}
static uint32_t kvq8_parts(const KvQ8Dev& c, const KvQ8Batch& b) {
  const uint64_t ctas = (uint64_t)kvq8_tiles(c, b) * c.nkv * b.n_seqs;
  return (uint32_t)std::max<uint64_t>(1, std::min<uint64_t>((uint64_t)num_sms() / ctas, b.max_pages / 4));
}

// Whether the call's rows go to k_kvq8_rows or to the split form, by the time
// that each takes for the longest sequence there can be: a step of two pages of
// 128 rows (fewer cost the same) takes k_kvq8_rows 2 us an SM, a page of 8 rows
// the split form 2.8 ns with all SMs at work; starting and joining takes 17 and
// 7.  Measured (us, split / rows): 1 sequence, 20 rows x 7 heads on 1000
// positions 13.8 / 21.4, 100 rows on 2000 46 / 28, 512 rows on 3000 288 / 71;
// 12 x 6 rows x 5 heads on up to 3000 37 / 63, all on 3000 68 / 60.  The lengths
// are on the device, so the table's width stands for them: a wide one with short
// sequences goes to k_kvq8_rows (20 rows on 20 positions, 512 pages: 27 us, with
// one page 8).
static bool kvq8_by_rows(const KvQ8Dev& c, const KvQ8Batch& b) {
  const double pages = b.max_pages, groups = (double)b.n_seqs * c.nkv * (((uint64_t)b.max_new * c.group + 7) / 8);
  const double waves = std::ceil((double)kvq8_tiles(c, b) * c.nkv * b.n_seqs / num_sms());
  return 17.0 + pages * waves / kvq8_parts(c, b) < 7.0 + 0.0028 * groups * pages;
}

static uint64_t kvq8_part_bytes(const KvQ8Dev& c) { return (uint64_t)(KR_M * c.hd + 2 * KR_M) * 4; }
static uint64_t kvq8_split_bytes(const KvQ8Dev& c, uint64_t runs) { return 2 * runs * (8 * c.hd + 16) * 4; }

uint64_t kvq8_attend_work(const KvQ8Dev& c, const KvQ8Batch& b) {
  if (!b.n_seqs) return 16;
  if (!kvq8_by_rows(c, b)) return kvq8_prefix_bytes(b) + kvq8_split_bytes(c, kvq8_runs(c, b));
  const uint64_t parts = kvq8_parts(c, b);
  return parts == 1 ? 16 : (uint64_t)kvq8_tiles(c, b) * c.nkv * b.n_seqs * parts * kvq8_part_bytes(c);
}

uint64_t kvq8_attend_work_most(const KvQ8Dev& c, uint32_t n_seqs) {
  KvQ8Batch b{};
  b.n_seqs = n_seqs;
  // parts are made only where they and the rows' tiles fit the SMs
  return std::max(kvq8_prefix_bytes(b) + kvq8_split_bytes(c, KQ_MG_PIECES), num_sms() * kvq8_part_bytes(c));
}

template <int HD, typename T>
static void kvq8_attend_t(const KvQ8Attend& a, cudaStream_t s) {
  const size_t smem = sizeof(KqSplitSmem<HD>);
  static std::atomic<uint64_t> ready{0};
  kvq8_once(ready, [&] {
    CK(cudaFuncSetAttribute(k_kvq8_split<HD, T>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    CK(cudaFuncSetAttribute(k_kvq8_whole<HD, T>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    CK(cudaFuncSetAttribute(k_kvq8_rows<HD, T>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(KrSmem<HD>)));
  });
  const uint32_t runs = kvq8_runs(a.c, a.b);
  KqSplitArgs<HD, T> k{a.c,
                       a.b,
                       static_cast<const T*>(a.q),
                       static_cast<T*>(a.out),
                       a.ldq,
                       a.ldo,
                       a.window,
                       a.sinks,
                       a.scale * 1.44269504088896341f,
                       static_cast<XRun*>(a.runs),
                       a.run0,
                       static_cast<uint64_t*>(a.work),
                       reinterpret_cast<float*>(static_cast<uint8_t*>(a.work) + kvq8_prefix_bytes(a.b)),
                       1,
                       a.after_append};
  if (!a.runs && kvq8_by_rows(a.c, a.b)) {
    const uint32_t tiles = kvq8_tiles(a.c, a.b);
    k.parts = kvq8_parts(a.c, a.b);
    k.slots = static_cast<float*>(a.work);
    launch_pdl(k_kvq8_rows<HD, T>, dim3(tiles * k.parts, a.c.nkv, a.b.n_seqs), dim3(KR_THREADS), sizeof(KrSmem<HD>), s,
               k);
    if (k.parts > 1)
      launch_pdl(k_kvq8_join<HD, T>, dim3((a.b.max_new * a.c.group + 3) / 4, a.c.nkv, a.b.n_seqs),
                 dim3(KR_JOIN_THREADS), 0, s, k, tiles);
    return;
  }
  if (!a.runs && a.b.max_pages <= KQ_WHOLE_PAGES) {
    const uint64_t groups = ((uint64_t)a.b.max_new * a.c.group + 7) / 8;
    launch_pdl(k_kvq8_whole<HD, T>, dim3((unsigned)(a.c.nkv * groups), a.b.n_seqs), dim3(KQ_SP_THREADS), smem, s, k);
    return;
  }
  launch_pdl(k_kvq8_split<HD, T>, dim3(runs), dim3(KQ_SP_THREADS), smem, s, k);
  launch_pdl(k_kvq8_merge<HD, T>, dim3(a.b.max_new * a.c.group, a.c.nkv, a.b.n_seqs), dim3(KQ_MG_THREADS), 0, s, k,
             runs);
}

void launch_kvq8_attend(const KvQ8Attend& a, cudaStream_t s) {
  if (!a.b.n_seqs) return;
  if (a.runs && a.b.n_seqs * a.b.max_new != 1) fail(FZ_EINVAL, "run records are made for one row");
  // With records every segment goes through the merge, and a run has two slots: as many runs as segments, so that none
  // holds more than two of them (a run is then at most a page longer than a segment).
  if (a.runs && a.c.nkv * ((a.c.group + 7) / 8) > kvq8_runs(a.c, a.b))
    fail(FZ_EINVAL, "%u KV heads in a step on an 8-bit cache, the limit is %u", a.c.nkv, kvq8_runs(a.c, a.b));
  if (a.c.hd == 128)
    a.f16 ? kvq8_attend_t<128, __half>(a, s) : kvq8_attend_t<128, float>(a, s);
  else
    a.f16 ? kvq8_attend_t<64, __half>(a, s) : kvq8_attend_t<64, float>(a, s);
}
