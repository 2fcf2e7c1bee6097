// fz_kvq8_*: the 8-bit paged KV cache on the caller's device buffers.  Checks
// of arguments, the choice of the device and the reports of the status word; the
// operators' kernels are in kvq8.cuh.

#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>

#include "fz_internal.h"
#include "kernels.h"

using namespace fz;

static_assert(FZ_KVQ8_PAGE == 64 && FZ_KVQ8_BLOCK == 16, "the kernels' page");

namespace {

void ck(cudaError_t e, const char* what) {
  if (e != cudaSuccess) {
    cudaGetLastError();  // not left for the next call to find
    fail(FZ_ECUDA, "%s failed: %s", what, cudaGetErrorString(e));
  }
}

// The device that owns p is current while this lives.
struct OnDeviceOf {
  int before = 0, dev = 0;
  explicit OnDeviceOf(const void* p) {
    cudaPointerAttributes a{};
    ck(cudaPointerGetAttributes(&a, p), "cudaPointerGetAttributes");
    need(a.type == cudaMemoryTypeDevice || a.type == cudaMemoryTypeManaged, "codes is not device memory");
    ck(cudaGetDevice(&before), "cudaGetDevice");
    dev = a.device;
    if (dev != before) ck(cudaSetDevice(dev), "cudaSetDevice");
  }
  ~OnDeviceOf() {
    if (dev != before) cudaSetDevice(before);
  }
  OnDeviceOf(const OnDeviceOf&) = delete;
  OnDeviceOf& operator=(const OnDeviceOf&) = delete;
};

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
bool aligned4(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3) == 0; }

KvQ8Dev device_view(const fz_kvq8* kv) {
  need(kv != nullptr, "null cache");
  need(kv->codes && kv->scales && kv->status, "null cache buffer");
  need(aligned16(kv->codes) && aligned16(kv->scales), "codes and scales must be 16-byte aligned");
  need(aligned4(kv->status), "the status word must be 4-byte aligned");
  need(kv->head_dim == 64 || kv->head_dim == 128, "head_dim %u unsupported (64 or 128)", kv->head_dim);
  need(kv->n_kv_heads > 0 && kv->n_kv_heads <= 65535, "%u KV heads unsupported", kv->n_kv_heads);
  need(kv->n_heads > 0 && kv->n_heads <= 65535 && kv->n_heads % kv->n_kv_heads == 0,
       "%u heads not divisible by %u kv heads", kv->n_heads, kv->n_kv_heads);
  need(kv->n_pages > 0 && kv->n_pages <= 0x7fffffffu, "%u pages unsupported", kv->n_pages);
  need(kv->rope ? kv->n_rope > 0 && kv->n_rope <= 0x7fffffffu : kv->n_rope == 0,
       "rotation table and its %u positions do not match", kv->n_rope);
  need(aligned16(kv->rope), "the rotation table must be 16-byte aligned");
  return KvQ8Dev{static_cast<uint8_t*>(kv->codes),
                 kv->scales,
                 reinterpret_cast<const float2*>(kv->rope),
                 kv->status,
                 kv->n_pages,
                 kv->n_rope,
                 kv->n_kv_heads,
                 kv->n_heads / kv->n_kv_heads,
                 kv->head_dim};
}

KvQ8Batch device_view(const fz_kvq8_seqs* s) {
  need(s != nullptr, "null sequences");
  need(s->n_seqs <= 65535, "%u sequences in one call, the limit is 65535", s->n_seqs);
  if (s->n_seqs) {
    need(s->pages && s->lens, "null page table or lengths");
    need(aligned4(s->pages) && aligned4(s->lens) && aligned4(s->starts),
         "page table, lengths and row starts must be 4-byte aligned");
    need(s->max_pages > 0 && s->max_pages <= 0x7fffffffu / FZ_KVQ8_PAGE, "%u pages per sequence unsupported",
         s->max_pages);
    need(s->max_new > 0 && s->max_new <= s->max_pages * FZ_KVQ8_PAGE, "%u new positions do not fit %u pages",
         s->max_new, s->max_pages);
    need(s->n_rows <= 0x7fffffffu, "%u rows unsupported", s->n_rows);
    need(s->starts || s->n_rows >= (uint64_t)s->n_seqs * s->max_new, "%u rows for %u sequences of %u", s->n_rows,
         s->n_seqs, s->max_new);
  }
  // no sequence has more rows than there are
  return KvQ8Batch{s->pages, s->lens, s->starts, s->n_seqs, s->max_pages, std::min(s->max_new, s->n_rows), s->n_rows, 0};
}

// Rows of `heads` heads at p, ld elements apart; true for f16.
bool check_rows(const char* what, uint32_t dtype, const void* p, uint64_t ld, uint32_t heads, uint32_t hd) {
  need(dtype == FZ_F32 || dtype == FZ_F16, "%s: type %u unsupported (FZ_F32 or FZ_F16)", what, dtype);
  need(p != nullptr, "%s: null argument", what);
  need(aligned16(p) && ld % (dtype == FZ_F32 ? 4 : 8) == 0, "%s: rows must start on 16-byte boundaries", what);
  need(ld >= (uint64_t)heads * hd && ld <= 0x7fffffffu, "%s: row stride %llu for %u heads of %u", what,
       (unsigned long long)ld, heads, hd);
  return dtype == FZ_F16;
}

__global__ void k_take_bits(uint32_t* word, uint32_t* found) { *found = atomicExch(word, 0u); }

// Reads the word and clears it in one step: a bit that a call on another stream
// sets meanwhile is read here or stays for the next time.
uint32_t take_bits(uint32_t* word, cudaStream_t s) {
  struct Scratch {
    void* p = nullptr;
    cudaStream_t s;
    ~Scratch() {
      if (p) cudaFreeAsync(p, s);
    }
  } found{nullptr, s};
  uint32_t bits = 0;
  ck(cudaMallocAsync(&found.p, 4, s), "cudaMallocAsync");
  k_take_bits<<<1, 1, 0, s>>>(word, static_cast<uint32_t*>(found.p));
  ck(cudaGetLastError(), "k_take_bits");
  ck(cudaMemcpyAsync(&bits, found.p, 4, cudaMemcpyDeviceToHost, s), "cudaMemcpyAsync");
  ck(cudaStreamSynchronize(s), "cudaStreamSynchronize");
  return bits;
}

}  // namespace

extern "C" {

int fz_kvq8_append_dev(const fz_kvq8* kv, const fz_kvq8_seqs* s, uint32_t dtype, const void* k, const void* v,
                       uint64_t ld, void* stream) {
  return guard([&] {
    const KvQ8Dev c = device_view(kv);
    const KvQ8Batch b = device_view(s);
    if (!b.n_seqs || !b.n_rows) return;
    const bool f16 = check_rows("k", dtype, k, ld, c.nkv, c.hd);
    check_rows("v", dtype, v, ld, c.nkv, c.hd);
    OnDeviceOf on(kv->codes);
    launch_kvq8_append(c, b, f16, k, v, ld, static_cast<cudaStream_t>(stream));
  });
}

int fz_kvq8_read_dev(const fz_kvq8* kv, const fz_kvq8_seqs* s, uint32_t dtype, void* k, void* v, uint64_t ld,
                     void* stream) {
  return guard([&] {
    const KvQ8Dev c = device_view(kv);
    const KvQ8Batch b = device_view(s);
    if (!b.n_seqs || !b.n_rows || !(k || v)) return;
    const bool f16 = check_rows("k", dtype, k ? k : v, ld, c.nkv, c.hd);
    check_rows("v", dtype, v ? v : k, ld, c.nkv, c.hd);
    OnDeviceOf on(kv->codes);
    launch_kvq8_read(c, b, f16, k, v, ld, static_cast<cudaStream_t>(stream));
  });
}

int fz_kvq8_attend_work(const fz_kvq8* kv, const fz_kvq8_seqs* s, uint64_t* bytes) {
  return guard([&] {
    need(bytes != nullptr, "null argument");
    const KvQ8Batch b = device_view(s);
    const KvQ8Dev c = device_view(kv);
    *bytes = b.n_seqs && b.n_rows ? kvq8_attend_work(c, b) : 16;
  });
}

int fz_kvq8_attend_dev(const fz_kvq8* kv, const fz_kvq8_seqs* s, uint32_t dtype, const void* q, uint64_t ldq,
                       void* out, uint64_t ldo, uint32_t window, uint32_t sinks, float scale, void* work,
                       uint64_t work_bytes, void* stream) {
  return guard([&] {
    KvQ8Attend a{};
    a.c = device_view(kv);
    a.b = device_view(s);
    need(std::isfinite(scale), "scale is not finite");
    if (!a.b.n_seqs || !a.b.n_rows) return;
    need((uint64_t)a.b.n_rows * kv->n_heads <= 0x7fffffffu, "%u rows of %u heads in one call", a.b.n_rows, kv->n_heads);
    a.f16 = check_rows("q", dtype, q, ldq, kv->n_heads, a.c.hd);
    check_rows("out", dtype, out, ldo, kv->n_heads, a.c.hd);
    need(q != out, "out must not overlap q");
    const uint64_t want = kvq8_attend_work(a.c, a.b);
    need(work && aligned16(work) && work_bytes >= want, "work: %llu bytes (16-byte aligned) needed, %llu given",
         (unsigned long long)want, (unsigned long long)(work ? work_bytes : 0));
    a.q = q;
    a.out = out;
    a.ldq = ldq;
    a.ldo = ldo;
    a.window = window;
    a.sinks = sinks;
    a.scale = scale == 0.f ? 1.f / sqrtf((float)a.c.hd) : scale;
    a.work = work;
    OnDeviceOf on(kv->codes);
    launch_kvq8_attend(a, static_cast<cudaStream_t>(stream));
  });
}

int fz_kvq8_status(const fz_kvq8* kv, void* stream) {
  return guard([&] {
    const KvQ8Dev c = device_view(kv);
    OnDeviceOf on(kv->codes);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    uint32_t bits = 0;
    ck(cudaMemcpyAsync(&bits, c.status, 4, cudaMemcpyDeviceToHost, s), "cudaMemcpyAsync");
    ck(cudaStreamSynchronize(s), "cudaStreamSynchronize");
    if (!bits) return;
    bits = take_bits(c.status, s);
    if (!bits) return;  // another report has them
    if (bits & KQ_TIMEOUT) fail(FZ_ETIMEOUT, "8-bit KV cache: a bounded device wait ran out");
    fail(FZ_EINVAL, "8-bit KV cache:%s%s%s%s", bits & KQ_BAD_LEN ? " lengths or rows out of range;" : "",
         bits & KQ_BAD_PAGE ? " page number out of range;" : "",
         bits & KQ_BAD_POS ? " position beyond the rotation table;" : "",
         bits & KQ_NOT_FINITE ? " keys or values that are not finite;" : "");
  });
}

}  // extern "C"
