// ops.cu -- C ABI of the operators around the MatMul node (include/momiru_ops.h):
// validation, kernel choice, TMA descriptors and workspaces at bind, and a run
// that enqueues the steps bind laid down. Follows the bind / run / quiesce split
// of momiru_gemm.cu, whose error message and f32 products it shares.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <chrono>
#include <cstdarg>
#include <cstdint>
#include <cstdio>
#include <cstring>
#include <functional>
#include <initializer_list>
#include <memory>
#include <mutex>
#include <new>
#include <string>
#include <thread>
#include <vector>

#include "../../include/momiru_ops.h"
#include "experts.cuh"
#include "launch.cuh"
#include "linear_launch.h"
#include "row_ops.cuh"

namespace mmr {
// momiru_gemm.cu
int32_t set_last_error(int32_t code, const char* message);
cudaError_t bind_zero(void* p, size_t bytes);
void gemm_set_chunk(mmr_gemm_handle* h, int k);
int32_t gemm_enqueue(mmr_gemm_handle* h, cudaStream_t s);
int32_t gemm_read_error(mmr_gemm_handle* h, uint64_t timeout_ns);
}

struct mmr_op_handle {
  int device = 0;
  int sms = 148;
  cudaStream_t stream = nullptr, last_stream = nullptr;
  struct Step {
    std::string what;
    std::function<int32_t(cudaStream_t)> launch;
  };
  std::vector<Step> steps;
  std::string plan;
  std::vector<void*> workspaces;
  std::vector<mmr_gemm_handle*> products;  // f32 products of the MatMul node
  int* d_err = nullptr;                    // device error word (256 bytes)
  int* h_err = nullptr;                    // pinned copy
  cudaEvent_t done = nullptr, err_ev = nullptr;
  bool ran = false;       // `done` was recorded (a run outside stream capture)
  bool launched = false;
  std::mutex run_mu;      // one run's wait, launches and record at a time; guards the two flags and last_stream
  std::mutex quiesce_mu;  // the pinned error word and its event
};

namespace {

using mmr::EpiMat;
using Handle = mmr_op_handle;
constexpr uint64_t kWaitNs = 2000000000ull;

int32_t fail(int32_t code, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof buf, fmt, ap);
  va_end(ap);
  return mmr::set_last_error(code, buf);
}

// Nothing throws across the C boundary.
template <typename F>
int32_t guarded(F&& f) {
  try {
    return f();
  } catch (const std::bad_alloc&) {
    return mmr::set_last_error(MMR_ERR_CUDA, "out of host memory");
  } catch (...) {
    return mmr::set_last_error(MMR_ERR_INVALID_ARGUMENT, "unexpected exception");
  }
}

struct DeviceGuard {
  int prev = -1;  // to be restored; -1 where the device was current already
  bool ok = false;
  explicit DeviceGuard(int dev) {
    int now = -1;
    if (cudaGetDevice(&now) != cudaSuccess) return;
    ok = now == dev || cudaSetDevice(dev) == cudaSuccess;
    if (ok && now != dev) prev = now;
  }
  ~DeviceGuard() {
    if (prev >= 0) cudaSetDevice(prev);
  }
};

#define MMR_TRY(expr)                    \
  do {                                   \
    if (int32_t rc_ = (expr)) return rc_; \
  } while (0)
#define MMR_CUDA(expr)                                                                          \
  do {                                                                                          \
    cudaError_t e_ = (expr);                                                                    \
    if (e_ != cudaSuccess) return fail(MMR_ERR_CUDA, "%s: %s", #expr, cudaGetErrorString(e_)); \
  } while (0)

// ---------------------------------------------------------------- tensors --
// Absent: rank 0 and no address. A scalar, or a negative rank, is present and refused.
bool present(const mmr_tensor& t) { return t.view.rank != 0 || t.view.address != 0; }

int elem_size(int dtype) { return dtype == MMR_DTYPE_BF16 || dtype == MMR_DTYPE_F16 ? 2 : 4; }

constexpr unsigned kF32 = 1u << MMR_DTYPE_F32, kBf16 = 1u << MMR_DTYPE_BF16, kF16 = 1u << MMR_DTYPE_F16,
                   kI32 = 1u << MMR_DTYPE_I32;
constexpr unsigned kHalf = kBf16 | kF16, kFloat = kHalf | kF32;

const char* dtype_name(int d) {
  switch (d) {
    case MMR_DTYPE_F32: return "f32";
    case MMR_DTYPE_BF16: return "bf16";
    case MMR_DTYPE_F16: return "f16";
    case MMR_DTYPE_I32: return "i32";
    default: return "unknown";
  }
}

// One checked operand: shape, bounds and the byte range it touches.
struct Ref {
  const char* name = "";
  uint64_t base = 0;  // address of element [0, .., 0]
  int rank = 0, es = 4, dtype = 0;
  int64_t d[3] = {1, 1, 1}, s[3] = {0, 0, 0};
  uint64_t lo = 0, hi = 0;  // [lo, hi) in bytes; empty when some extent is 0
  uint64_t address = 0;
  bool on = false;
};

// Reads `t` as a rank-`rank` operand of one of `dtypes`; axes are right-aligned
// in Ref (a matrix is d[1] x d[2], a vector d[2]).
int32_t read_tensor(const mmr_tensor& t, const char* name, int device, int rank, unsigned dtypes, Ref* r) {
  const mmr_view& v = t.view;
  r->name = name;
  if (!present(t)) return fail(MMR_ERR_INVALID_ARGUMENT, "%s: missing", name);
  if (t.dtype < 0 || t.dtype > MMR_DTYPE_I32 || !(dtypes >> t.dtype & 1u))
    return fail(MMR_ERR_INVALID_ARGUMENT, "%s: element type %s is not taken here", name, dtype_name(t.dtype));
  if (v.rank != rank) return fail(MMR_ERR_INVALID_SHAPE, "%s: rank %d, expected %d", name, v.rank, rank);
  r->rank = rank;
  r->dtype = t.dtype;
  r->es = elem_size(t.dtype);
  r->address = v.address;
  r->on = true;
  // 128 bits: an extent below 2^31 times a stride of up to 2^40 passes 64
  __int128 lo = 0, hi = 0;
  bool empty = false;
  for (int i = 0; i < rank; ++i) {
    if (v.dims[i] < 0) return fail(MMR_ERR_INVALID_SHAPE, "%s: negative extent on axis %d", name, i);
    if (v.dims[i] > (int64_t(1) << 31) - 1024)
      return fail(MMR_ERR_INVALID_SHAPE, "%s: extent %lld on axis %d exceeds 2^31 - 1024", name, (long long)v.dims[i], i);
    if (v.strides[i] > (int64_t(1) << 40) || v.strides[i] < -(int64_t(1) << 40))
      return fail(MMR_ERR_UNSUPPORTED_LAYOUT, "%s: stride on axis %d beyond 2^40 elements", name, i);
    r->d[3 - rank + i] = v.dims[i];
    r->s[3 - rank + i] = v.strides[i];
    if (v.dims[i] == 0) {
      empty = true;
      continue;
    }
    const __int128 reach = __int128(v.dims[i] - 1) * v.strides[i];
    (reach < 0 ? lo : hi) += reach;
  }
  if (v.base_offset_bytes % r->es || v.address % r->es)
    return fail(MMR_ERR_UNSUPPORTED_LAYOUT, "%s: address or offset is not aligned to its %d-byte elements", name, r->es);
  if (v.device_ordinal != device)
    return fail(MMR_ERR_UNSUPPORTED_DEVICE, "%s: device ordinal %d differs from the operator's %d", name,
                v.device_ordinal, device);
  r->base = v.address + v.base_offset_bytes;
  r->lo = r->hi = r->base;
  if (!empty) {
    if (v.address == 0) return fail(MMR_ERR_INVALID_ARGUMENT, "%s: null address", name);
    if (v.base_offset_bytes / r->es + lo < 0)
      return fail(MMR_ERR_OUT_OF_BOUNDS, "%s: a negative stride reaches before the buffer", name);
    const __int128 need = v.base_offset_bytes + (hi + 1) * r->es;
    if (need > v.bytes || need > UINT64_MAX - v.address)
      return fail(MMR_ERR_OUT_OF_BOUNDS, "%s: view needs %.0f bytes but the buffer has %llu", name, double(need),
                  (unsigned long long)v.bytes);
    r->lo = r->base + uint64_t(lo * r->es);
    r->hi = r->base + uint64_t((hi + 1) * r->es);
  }
  return MMR_OK;
}

int32_t want_dims(const Ref& r, std::initializer_list<int64_t> dims) {
  int i = 3 - int(dims.size());
  for (int64_t want : dims) {
    if (r.d[i] != want)
      return fail(MMR_ERR_INVALID_SHAPE, "%s: extent %lld on axis %d, expected %lld", r.name, (long long)r.d[i],
                  i - (3 - r.rank), (long long)want);
    ++i;
  }
  return MMR_OK;
}

int32_t same_dtype(const Ref& r, int dtype) {
  if (r.dtype != dtype)
    return fail(MMR_ERR_INVALID_ARGUMENT, "%s: element type %s where the other operands have %s", r.name,
                dtype_name(r.dtype), dtype_name(dtype));
  return MMR_OK;
}

// Whether two operands may share bytes. Two matrices that are column blocks of
// one row pitch interleave without meeting, which their byte ranges cannot tell.
bool overlap(const Ref& x, const Ref& y) {
  if (x.lo == x.hi || y.lo == y.hi || x.lo >= y.hi || y.lo >= x.hi) return false;
  if (x.rank == 2 && y.rank == 2 && x.es == y.es && x.s[2] == 1 && y.s[2] == 1 && x.s[1] == y.s[1] && x.s[1] > 0) {
    const int64_t ld = x.s[1], gap = (int64_t(y.base) - int64_t(x.base)) / x.es;
    const int64_t off = (gap % ld + ld) % ld;  // y's first column counted from x's
    if (off >= x.d[2] && off + y.d[2] <= ld) return false;
  }
  return true;
}
bool same_view(const Ref& x, const Ref& y) {
  return x.base == y.base && x.rank == y.rank && memcmp(x.d, y.d, sizeof x.d) == 0 && memcmp(x.s, y.s, sizeof x.s) == 0;
}

// An output's elements must be distinct: sorted by stride, each axis steps past
// the whole extent of the finer ones.
int32_t check_output(const Ref& o) {
  if (o.lo == o.hi) return MMR_OK;
  std::vector<std::pair<int64_t, int64_t>> ax;
  for (int i = 0; i < 3; ++i)
    if (o.d[i] > 1) ax.emplace_back(o.s[i] < 0 ? -o.s[i] : o.s[i], o.d[i]);
  std::sort(ax.begin(), ax.end());
  __int128 span = 1;
  for (const auto& [stride, extent] : ax) {
    if (stride < span) return fail(MMR_ERR_UNSAFE_ALIASING, "%s: the output's own elements overlap", o.name);
    span += __int128(stride) * (extent - 1);
  }
  return MMR_OK;
}

int32_t check_aliasing(std::initializer_list<const Ref*> outs, std::initializer_list<const Ref*> ins,
                       const Ref* in_place = nullptr) {
  for (const Ref* o : outs) {
    if (!o->on) continue;
    MMR_TRY(check_output(*o));
    for (const Ref* i : ins)
      if (i->on && overlap(*o, *i) && !(i == in_place && o == *outs.begin() && same_view(*o, *i)))
        return fail(MMR_ERR_UNSAFE_ALIASING, "%s overlaps %s", o->name, i->name);
    for (const Ref* q : outs)
      if (q != o && q->on && overlap(*o, *q)) return fail(MMR_ERR_UNSAFE_ALIASING, "%s overlaps %s", o->name, q->name);
  }
  return MMR_OK;
}

// ----------------------------------------------------------------- device --
int32_t check_device(int device, std::initializer_list<const Ref*> refs, int* sms) {
  int ndev = 0;
  if (cudaGetDeviceCount(&ndev) != cudaSuccess || ndev == 0) {
    cudaGetLastError();
    return fail(MMR_ERR_UNSUPPORTED_DEVICE, "no CUDA device is visible");
  }
  if (device < 0 || device >= ndev)
    return fail(MMR_ERR_UNSUPPORTED_DEVICE, "device ordinal %d outside 0..%d", device, ndev - 1);
  int major = 0, minor = 0;
  MMR_CUDA(cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, device));
  MMR_CUDA(cudaDeviceGetAttribute(&minor, cudaDevAttrComputeCapabilityMinor, device));
  MMR_CUDA(cudaDeviceGetAttribute(sms, cudaDevAttrMultiProcessorCount, device));
  if (major != 10 || minor != 0)
    return fail(MMR_ERR_UNSUPPORTED_DEVICE, "device %d is sm_%d%d; this library is built for sm_100a", device, major,
                minor);
  for (const Ref* r : refs) {
    if (!r->on || r->lo == r->hi) continue;
    cudaPointerAttributes pa;
    if (cudaPointerGetAttributes(&pa, reinterpret_cast<void*>(r->address)) != cudaSuccess) {
      cudaGetLastError();
      return fail(MMR_ERR_UNSUPPORTED_DEVICE, "%s: its address is not known to CUDA", r->name);
    }
    if ((pa.type != cudaMemoryTypeDevice && pa.type != cudaMemoryTypeManaged) || pa.device != device)
      return fail(MMR_ERR_UNSUPPORTED_DEVICE, "%s: not memory of device %d", r->name, device);
  }
  return MMR_OK;
}

struct Destroy {
  void operator()(Handle* h) const { mmr_op_destroy(h); }
};
using Owned = std::unique_ptr<Handle, Destroy>;

int32_t new_handle(int device, int sms, void* stream, Owned* out) {
  Owned h(new Handle());
  h->device = device;
  h->sms = sms;
  h->stream = reinterpret_cast<cudaStream_t>(stream);
  MMR_CUDA(cudaMalloc(&h->d_err, 256));
  MMR_CUDA(mmr::bind_zero(h->d_err, 256));
  MMR_CUDA(cudaHostAlloc(&h->h_err, sizeof(int), cudaHostAllocDefault));
  *h->h_err = 0;
  MMR_CUDA(cudaEventCreateWithFlags(&h->done, cudaEventDisableTiming));
  MMR_CUDA(cudaEventCreateWithFlags(&h->err_ev, cudaEventDisableTiming));
  *out = std::move(h);
  return MMR_OK;
}

// `bytes` in 128 bits: an operand broadcast over its axes (strides of 0) may be
// larger to pack than 64 bits can say.
int32_t workspace(Handle* h, __int128 bytes, void** out) {
  if (bytes > (int64_t(1) << 48)) return fail(MMR_ERR_INVALID_SHAPE, "a workspace of %.3g bytes", double(bytes));
  void* p = nullptr;
  const cudaError_t e = cudaMalloc(&p, size_t(std::max<__int128>(bytes, 256)));
  if (e != cudaSuccess) {
    cudaGetLastError();
    return fail(MMR_ERR_CUDA, "allocating a workspace of %lld bytes: %s", (long long)bytes, cudaGetErrorString(e));
  }
  h->workspaces.push_back(p);
  *out = p;
  return MMR_OK;
}

// Records a launch; `fn` returns the cudaError_t of the enqueue.
template <typename F>
void add_step(Handle* h, const char* fmt, F fn, long long a = 0, long long b = 0, long long c = 0) {
  char buf[192];
  snprintf(buf, sizeof buf, fmt, a, b, c);
  std::string what = buf;
  h->plan += what + "\n";
  h->steps.push_back({what, [fn, what](cudaStream_t s) -> int32_t {
                        const cudaError_t e = fn(s);
                        return e == cudaSuccess ? MMR_OK : fail(MMR_ERR_CUDA, "%s: %s", what.c_str(), cudaGetErrorString(e));
                      }});
}

// ------------------------------------------------------------ tensor maps --
typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiledFn encode_fn() {
  static EncodeTiledFn fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &ptr, 12000, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeTiledFn>(ptr);
  });
  return fn;
}

// A 16-bit product operand as TMA reads it: `mn` rows or columns by `k`.
struct Operand {
  uint64_t base = 0;
  int64_t mn = 0, k = 0, batch = 1;
  int64_t s_mn = 0, s_k = 0, s_b = 0;
  bool mn_major = false;
};

// 128-byte swizzled boxes: K-major 64 k x `rows` of mn, MN-major 64 mn x 64 k.
int32_t encode16(CUtensorMap* tm, const Operand& o, int dtype, int rows, const char* name) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return fail(MMR_ERR_CUDA, "cuTensorMapEncodeTiled is unavailable");
  const uint64_t inner = o.mn_major ? o.mn : o.k, outer = o.mn_major ? o.k : o.mn;
  uint64_t pitch = uint64_t(o.mn_major ? o.s_k : o.s_mn) * 2;
  if (outer <= 1) pitch = (inner * 2 + 15) & ~uint64_t(15);
  uint64_t bpitch = uint64_t(o.s_b) * 2;
  if (o.batch <= 1) bpitch = pitch * outer;
  cuuint64_t dims[3] = {inner, outer, uint64_t(o.batch)};
  cuuint64_t strides[2] = {pitch, bpitch};
  cuuint32_t box[3] = {64, cuuint32_t(o.mn_major ? 64 : rows), 1};
  cuuint32_t estr[3] = {1, 1, 1};
  const CUresult r =
      fn(tm, dtype == MMR_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
         reinterpret_cast<void*>(o.base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return fail(MMR_ERR_UNSUPPORTED_LAYOUT, "%s: cuTensorMapEncodeTiled failed (%d): dims {%llu,%llu,%llu}", name, int(r),
                (unsigned long long)inner, (unsigned long long)outer, (unsigned long long)o.batch);
  return MMR_OK;
}

bool tma_pitch(uint64_t base, int64_t pitch, int64_t extent, int64_t s_b, int64_t batch, int64_t inner) {
  if (base % 16) return false;
  if (extent > 1 && (pitch <= 0 || pitch % 8 || pitch < inner || pitch >= (int64_t(1) << 38))) return false;
  return batch <= 1 || (s_b > 0 && s_b % 8 == 0 && s_b < (int64_t(1) << 38));
}

// Makes `o` readable by TMA: as it lies where it can, else packed by each run
// into rows of a 16-byte pitch (entered in `packs`). `major`: 0 any, 1 K-major
// only, 2 MN-major only.
int32_t admit(Handle* h, Operand* o, int major, const char* name, mmr::PackList* packs) {
  if (o->mn == 0 || o->k == 0 || o->batch == 0) return MMR_OK;  // nothing is loaded
  if (major != 2 && (o->s_k == 1 || o->k == 1) && tma_pitch(o->base, o->s_mn, o->mn, o->s_b, o->batch, o->k)) {
    o->mn_major = false;
    return MMR_OK;
  }
  if (major != 1 && (o->s_mn == 1 || o->mn == 1) && tma_pitch(o->base, o->s_k, o->k, o->s_b, o->batch, o->mn)) {
    o->mn_major = true;
    return MMR_OK;
  }
  const int64_t as_mn = std::abs(o->s_mn), as_k = std::abs(o->s_k);
  const bool mn_major = major == 2 || (major == 0 && as_mn < as_k);
  mmr::PackParams q;
  q.src = reinterpret_cast<const void*>(o->base);
  q.s_b = o->s_b;
  q.rows = int(mn_major ? o->k : o->mn);
  q.cols = int(mn_major ? o->mn : o->k);
  q.s_r = mn_major ? o->s_k : o->s_mn;
  q.s_c = mn_major ? o->s_mn : o->s_k;
  q.pitch = (q.cols + 7) / 8 * 8;
  q.rows_out = q.rows;
  if (o->batch > 65535) return fail(MMR_ERR_UNSUPPORTED_LAYOUT, "%s: more than 65535 matrices to pack", name);
  const int64_t per = int64_t(q.rows) * q.pitch;
  q.batch = int(o->batch);
  MMR_TRY(workspace(h, __int128(per) * o->batch * 2, &q.dst));
  packs->p[packs->n++] = q;
  o->base = reinterpret_cast<uint64_t>(q.dst);
  o->mn_major = mn_major;
  (mn_major ? o->s_k : o->s_mn) = q.pitch;
  (mn_major ? o->s_mn : o->s_k) = 1;
  o->s_b = per;
  return MMR_OK;
}

// One launch for all operands of a product that have to be packed.
void add_packs(Handle* h, const mmr::PackList& packs, int elem_bytes = 2) {
  if (packs.n == 0) return;
  int64_t tiles = 1, batch = 1;
  for (int i = 0; i < packs.n; ++i) {
    tiles = std::max(tiles, int64_t((packs.p[i].rows_out + 31) / 32) * ((packs.p[i].pitch + 31) / 32));
    batch = std::max<int64_t>(batch, packs.p[i].batch);
  }
  const dim3 grid(unsigned(std::min<int64_t>(tiles, 8 * h->sms)), unsigned(packs.n), unsigned(batch));
  add_step(h, "mmr_pack_kernel grid %lld x %lld x %lld", [packs, grid, elem_bytes](cudaStream_t s) {
    return mmr::launch_kernel(
        elem_bytes == 2 ? mmr::mmr_pack_kernel<unsigned short> : mmr::mmr_pack_kernel<unsigned int>, grid, dim3(256), 0, s,
        dim3(1, 1, 1), packs);
  }, grid.x, grid.y, grid.z);
}

// Never read by TMA: a valid descriptor for a product without any k-blocks.
void no_operand(Handle* h, Operand* o) {
  o->base = reinterpret_cast<uint64_t>(h->d_err);
  o->mn = o->batch = 1;
  o->k = o->s_mn = 64;
  o->s_k = 1;
  o->mn_major = false;
}

EpiMat epi_mat(const Ref& r) {
  EpiMat m;
  if (!r.on) return m;
  m.p = reinterpret_cast<void*>(r.base);
  m.bs = r.s[0];
  m.ld = r.s[1];
  m.cs = r.s[2];
  const int per = 16 / r.es;
  m.vec = (r.s[2] == 1 || r.d[2] == 1) && r.base % 16 == 0 && (r.s[1] % per == 0 || r.d[1] == 1) &&
          (r.s[0] % per == 0 || r.d[0] == 1);
  if (r.d[2] == 1) m.vec = 0;
  return m;
}

// --------------------------------------------------------------- products --
struct Groups {  // ragged rows or contraction
  int experts = 0;
  const int *offsets = nullptr, *counts = nullptr;
  int64_t rows = 0, assignments = 0;
};

// ---- which kernel, and how the strip kernel divides its work: the least of the
// times estimated (us) for `mats` weight matrices of n columns and k_blocks, each
// met by `rows` rows (expert products: the mean). Both estimates were fitted to
// products of 1 to 1024 rows with N and K of 512 to 11008 and are within about
// 2 us of what was measured there.
//
// Strip: 5.5 for launch, first bytes and last store; then the longer of the
// weights' way from memory (6.4 TB/s, 5.3 with one CTA an SM) and the k-blocks of the SM with the most CTAs (its
// MMAs bound one at 0.235 up to 64 rows and 0.21 at 128, where another CTA hides
// its latencies; alone 0.25 and 0.33); 3 for every further wave of CTAs; the join
// of K slices and the epilogue by rows. A narrower strip than 128 columns only lost:
// an MMA costs its ~100 cycles however few rows of it are used.
//
// Pairs: 6.5, and the longer of the weights' way (at three quarters of memory's
// rate) and the rounds: per k-block 0.3 for every full round of tiles, 0.34 for a
// partial one, 0.234 where that is cut into half tiles.
//
// 128 x 4096 x 4096 takes 13.1 us as 128-row strips in 4 slices, 16.4 in 2 and
// 21.6 on pairs; 128 x 11008 x 4096 32 us on strips, 28.5 on pairs; 1024 rows
// over 32 experts of 2048 x 1024 29.5 us on strips, 39.3 on pairs.
struct StripShape {
  int mt = 16, split = 1, stages = 3;
  double us = 0;
};

StripShape strip_shape(int sms, int64_t mats, double rows, bool ragged, int64_t n, int k_blocks) {
  StripShape best;
  const int64_t strips = (n + mmr::LS_COLS - 1) / mmr::LS_COLS;
  for (int mt = 16; mt <= 128; mt *= 2) {
    const int64_t units = mats * (ragged ? int64_t(rows / mt) + 1 : (int64_t(rows) + mt - 1) / mt) * strips;
    for (int split = 1; split <= mmr::LS_MAX_SPLIT && split <= std::max(k_blocks, 1); split *= 2) {
      // three CTAs an SM (the registers allow no more) where each has three stages
      int share = 3, stages = 0;
      for (;; --share) {
        const int budget = 232448 / share - (share > 1 ? 2048 : 0);
        stages = mmr::LS_MAX_STAGES;
        while (stages > 1 && mmr::strip_smem_bytes(mt, stages, split) > budget) --stages;
        if (stages >= 3 || share == 1) break;
      }
      const int64_t ctas = units * split;
      // clusters of one CTA an SM do not fill the GPU, whose parts have no whole
      // number of clusters of SMs: what does not fit runs as a second wave
      if (share == 1 && ctas > sms * (split == 8 ? 11 : split == 4 ? 14 : split == 2 ? 15 : 16) / 16 && split > 1) continue;
      const int64_t deep = (ctas + sms - 1) / sms, waves = (ctas + sms * share - 1) / (sms * share);
      const int64_t blocks = (k_blocks + split - 1) / split;
      const double stream = double(deep * blocks) * (mt <= 64 ? (deep > 1 ? 0.235 : 0.25) : deep > 1 ? 0.21 : 0.33);
      const double memory = double(mats) * double(n) * k_blocks * 128 / (deep > 1 ? 6.4e6 : 5.3e6);
      const double us = 5.5 + std::max(stream, memory) + 3.0 * double(waves - 1) +
                        (split > 1 ? 0.5 + 0.012 * mt : 0.02 * mt);
      if (best.us == 0 || us < best.us - 0.05) best = {mt, split, stages, us};
    }
    if (!ragged && mt >= rows) break;
  }
  return best;
}

double pair_us(int sms, int64_t mats, double rows, bool ragged, int64_t n, int k_blocks) {
  const int64_t pairs = sms / 2;
  const int64_t tiles = mats * (ragged ? int64_t(rows / 256) + 1 : (int64_t(rows) + 255) / 256) * ((n + 255) / 256);
  const int64_t rem = tiles % pairs;
  const double rounds = k_blocks * (0.3 * double(tiles / pairs) + (rem == 0 ? 0.0 : 2 * rem <= pairs ? 0.234 : 0.34));
  return 6.5 + std::max(rounds, double(mats) * double(n) * k_blocks * 128 / 4.9e6);
}

int round16(int64_t v) { return int((v + 15) / 16 * 16); }

int32_t check_tiles(int64_t tiles) {
  return tiles > (int64_t(1) << 30) ? fail(MMR_ERR_INVALID_SHAPE, "more than 2^30 output tiles") : int32_t(MMR_OK);
}

// out[m, n] = epilogue(A[m, k] B[k, n]) in 16-bit operands; a.mn = m, b.mn = n.
// With `g`, the experts' products over ragged rows (b batched).
int32_t add_product(Handle* h, int dtype, Operand a, Operand b, mmr::EpiParams epi, const Groups* g) {
  const bool bf16 = dtype == MMR_DTYPE_BF16;
  const int64_t m = a.mn, n = b.mn, k = a.k;
  epi.n = int(n);
  if (m == 0 || n == 0) return MMR_OK;
  const int k_blocks = int((k + 63) / 64);
  const int64_t mats = g ? std::min<int64_t>(g->experts, g->assignments) : 1;
  const double rows = g ? double(g->assignments) / double(mats) : double(m);
  const StripShape shape = strip_shape(h->sms, mats, rows, g != nullptr, n, k_blocks);
  const bool strip = rows <= 1024 && shape.us < pair_us(h->sms, mats, rows, g != nullptr, n, k_blocks);
  mmr::PackList packs;
  MMR_TRY(admit(h, &a, strip || g ? 1 : 0, "lhs", &packs));
  MMR_TRY(admit(h, &b, 0, "rhs", &packs));
  add_packs(h, packs);
  if (k == 0) {
    no_operand(h, &a);
    no_operand(h, &b);
  }
  CUtensorMap ta, tb;
  if (strip) {
    mmr::StripParams p;
    p.m = int(m);
    p.n = int(n);
    p.k_blocks = k_blocks;
    p.mt = g ? shape.mt : std::min(shape.mt, round16(m));
    p.strips = int((n + mmr::LS_COLS - 1) / mmr::LS_COLS);
    p.m_units = g ? int(std::min<int64_t>(g->experts, g->assignments) + g->assignments / p.mt)
                  : int((m + p.mt - 1) / p.mt);
    if (g) {
      p.experts = g->experts;
      p.offsets = g->offsets;
      p.counts = g->counts;
      p.rows = g->rows;
    }
    p.split = shape.split;
    p.stages = shape.stages;
    p.tmem_cols = 32;
    while (p.tmem_cols < uint32_t(p.mt)) p.tmem_cols *= 2;
    p.epi = epi;
    p.err = h->d_err;
    p.timeout_ns = kWaitNs;
    MMR_TRY(encode16(&tb, b, dtype, mmr::LS_COLS, "rhs"));
    MMR_TRY(encode16(&ta, a, dtype, p.mt, "lhs"));
    const int64_t grid = int64_t(p.strips) * p.m_units * p.split;
    if (grid > (int64_t(1) << 31) - 1) return fail(MMR_ERR_INVALID_SHAPE, "more than 2^31 units of work");
    const int smem = mmr::strip_smem_bytes(p.mt, p.stages, p.split);
    const bool w_mn = b.mn_major;
    MMR_CUDA(mmr::strip_prepare(bf16, w_mn));
    add_step(h, "mmr_linear_strip_kernel grid %lld, split %lld, rows %lld", [=](cudaStream_t s) {
      return mmr::strip_launch(bf16, w_mn, int(grid), smem, s, tb, ta, p);
    }, grid, p.split, p.mt);
    return MMR_OK;
  }
  mmr::PairParams p;
  mmr::PairShape sh;
  sh.bf16 = bf16;
  sh.rag = g ? 1 : 0;
  sh.a_mn = a.mn_major;
  sh.b_mn = b.mn_major;
  p.m = int(m);
  p.n = int(n);
  p.tiles_m = int((m + 255) / 256);
  p.tile_rows = mmr::lp_tile_rows(p.m, p.tiles_m);
  p.tiles_n = int((n + 255) / 256);
  p.k_blocks = k_blocks;
  int64_t tiles = int64_t(p.tiles_m) * p.tiles_n;
  if (g) {
    p.experts = g->experts;
    p.offsets = g->offsets;
    p.counts = g->counts;
    p.rows = g->rows;
    tiles = (std::min<int64_t>(g->experts, g->assignments) + g->assignments / 256) * p.tiles_n;  // at most
  }
  MMR_TRY(check_tiles(tiles));
  p.tiles_total = int(tiles);
  p.epi = epi;
  p.err = h->d_err;
  p.timeout_ns = kWaitNs;
  MMR_TRY(encode16(&ta, a, dtype, 64, "lhs"));
  MMR_TRY(encode16(&tb, b, dtype, 128, "rhs"));
  sh.grid = 2 * int(std::min<int64_t>(h->sms / 2, std::max<int64_t>(2 * tiles, 1)));
  MMR_CUDA(mmr::pair_prepare(sh));
  add_step(h, "mmr_linear_pair_kernel grid %lld, tiles %lld, k-blocks %lld", [=](cudaStream_t s) {
    return mmr::pair_launch(sh, s, ta, tb, p);
  }, sh.grid, tiles, k_blocks);
  return MMR_OK;
}

// out[e] (m x n) = A_e^T B_e over the rows of each expert's segment.
int32_t add_segment_product(Handle* h, int dtype, Operand a, Operand b, const EpiMat& out, const Groups& g) {
  const bool bf16 = dtype == MMR_DTYPE_BF16;
  mmr::PairParams p;
  p.m = int(a.mn);
  p.n = int(b.mn);
  if (p.m == 0 || p.n == 0 || g.experts == 0) return MMR_OK;
  mmr::PackList packs;
  MMR_TRY(admit(h, &a, 2, "rows", &packs));
  MMR_TRY(admit(h, &b, 2, "d_out", &packs));
  add_packs(h, packs);
  if (g.rows == 0) {
    no_operand(h, &a);
    no_operand(h, &b);
  }
  mmr::PairShape sh;
  sh.bf16 = bf16;
  sh.rag = 2;
  sh.a_mn = sh.b_mn = true;
  p.tiles_m = (p.m + 255) / 256;
  p.tile_rows = mmr::lp_tile_rows(p.m, p.tiles_m);
  p.tiles_n = (p.n + 255) / 256;
  const int64_t tiles = int64_t(p.tiles_m) * p.tiles_n * g.experts;
  MMR_TRY(check_tiles(tiles));
  p.tiles_total = int(tiles);
  p.experts = g.experts;
  p.offsets = g.offsets;
  p.counts = g.counts;
  p.rows = g.rows;
  p.epi.out = out;
  p.epi.n = p.n;
  p.err = h->d_err;
  p.timeout_ns = kWaitNs;
  CUtensorMap ta, tb;
  MMR_TRY(encode16(&ta, a, dtype, 64, "rows"));
  MMR_TRY(encode16(&tb, b, dtype, 128, "d_out"));
  sh.grid = 2 * int(std::min<int64_t>(h->sms / 2, 2 * tiles));
  MMR_CUDA(mmr::pair_prepare(sh));
  add_step(h, "mmr_linear_pair_kernel (segments) grid %lld, tiles %lld", [=](cudaStream_t s) {
    return mmr::pair_launch(sh, s, ta, tb, p);
  }, sh.grid, tiles);
  return MMR_OK;
}

// Calls f with the activation as a compile-time constant.
template <typename F>
auto pick_act(int act, F&& f) {
  switch (act) {
    case MMR_ACT_RELU: return f(std::integral_constant<int, MMR_ACT_RELU>());
    case MMR_ACT_RELU6: return f(std::integral_constant<int, MMR_ACT_RELU6>());
    case MMR_ACT_GELU_ERF: return f(std::integral_constant<int, MMR_ACT_GELU_ERF>());
    case MMR_ACT_GELU_TANH: return f(std::integral_constant<int, MMR_ACT_GELU_TANH>());
    case MMR_ACT_SILU: return f(std::integral_constant<int, MMR_ACT_SILU>());
    default: return f(std::integral_constant<int, MMR_ACT_NONE>());
  }
}

// d_pre (and d_bias) from d_out and pre. Fills `d_pre` with the view that the
// products read: d_out itself without an activation, else a workspace.
int32_t add_act_grad(Handle* h, int act, const Ref& d_out, const Ref& pre, const Ref& d_bias, Ref* d_pre,
                     const Groups* g, const int* sources) {
  const int64_t rows = d_out.d[1], n = d_out.d[2];
  *d_pre = d_out;
  const bool through = act != MMR_ACT_NONE;
  if (n == 0 || (!through && !d_bias.on)) return MMR_OK;
  mmr::ActGradParams p;
  p.d_out = epi_mat(d_out);
  p.rows = rows;
  p.n = int(n);
  p.act = act;
  p.sources = sources;
  const int64_t chunks = (rows + mmr::AG_ROWS - 1) / mmr::AG_ROWS;
  if (through) {
    p.pre = epi_mat(pre);
    d_pre->s[2] = 1;
    d_pre->s[1] = (n + 7) / 8 * 8;
    void* w = nullptr;
    MMR_TRY(workspace(h, __int128(rows) * d_pre->s[1] * d_out.es, &w));
    d_pre->base = reinterpret_cast<uint64_t>(w);
    d_pre->name = "d_pre";
    p.d_pre = epi_mat(*d_pre);
  }
  if (d_bias.on) {
    void* w = nullptr;
    MMR_TRY(workspace(h, __int128(chunks) * n * 4, &w));
    p.partial = static_cast<float*>(w);
  }
  const int dt = d_out.dtype;
  const bool vec = n % 8 == 0 && p.d_out.vec && (!through || p.pre.vec);
  const dim3 grid(unsigned((n + mmr::AG_COLS - 1) / mmr::AG_COLS), unsigned(std::min<int64_t>(std::max<int64_t>(chunks, 1), 65535)));
  if (rows > 0)
    add_step(h, "mmr_act_grad_kernel grid %lld x %lld", [=](cudaStream_t s) {
      using K = void (*)(const mmr::ActGradParams);
      const K k = pick_act(p.act, [&](auto a) -> K {
        constexpr int kAct = decltype(a)::value;
        if (vec)
          return dt == MMR_DTYPE_F32    ? mmr::mmr_act_grad_kernel<float, kAct, true>
                 : dt == MMR_DTYPE_BF16 ? mmr::mmr_act_grad_kernel<__nv_bfloat16, kAct, true>
                                        : mmr::mmr_act_grad_kernel<__half, kAct, true>;
        return dt == MMR_DTYPE_F32    ? mmr::mmr_act_grad_kernel<float, kAct, false>
               : dt == MMR_DTYPE_BF16 ? mmr::mmr_act_grad_kernel<__nv_bfloat16, kAct, false>
                                      : mmr::mmr_act_grad_kernel<__half, kAct, false>;
      });
      return mmr::launch_kernel(k, grid, dim3(256), 0, s, dim3(1, 1, 1), p);
    }, grid.x, grid.y);
  if (d_bias.on) {
    mmr::ColSumParams c;
    c.partial = p.partial;
    c.out = reinterpret_cast<void*>(d_bias.base);
    c.out_bs = d_bias.s[1];
    c.out_s = d_bias.s[2];
    c.n = int(n);
    c.chunks = int(chunks);
    c.offsets = g ? g->offsets : nullptr;
    const dim3 cg(unsigned((n + 31) / 32), unsigned(g ? g->experts : 1));
    add_step(h, "mmr_col_sum_kernel grid %lld x %lld", [=](cudaStream_t s) {
      auto k = dt == MMR_DTYPE_F32    ? mmr::mmr_col_sum_kernel<float>
               : dt == MMR_DTYPE_BF16 ? mmr::mmr_col_sum_kernel<__nv_bfloat16>
                                      : mmr::mmr_col_sum_kernel<__half>;
      return mmr::launch_kernel(k, cg, dim3(256), 0, s, dim3(1, 1, 1), c);
    }, cg.x, cg.y);
  }
  return MMR_OK;
}

// ------------------------------------------------- f32 through the MatMul node --
mmr_view f32_view(uint64_t base, int64_t rows, int64_t cols, int64_t s_r, int64_t s_c, int device, uint64_t lo,
                  uint64_t hi) {
  mmr_view v{};
  v.address = lo;  // the view's own bytes: bounds were checked against its buffer
  v.bytes = hi - lo;
  v.base_offset_bytes = base - lo;
  v.rank = 2;
  v.device_ordinal = device;
  v.dims[0] = rows;
  v.dims[1] = cols;
  v.strides[0] = s_r;
  v.strides[1] = s_c;
  return v;
}
// A dense workspace matrix.
mmr_view f32_view(const void* p, int64_t rows, int64_t cols, int64_t ld, int device) {
  const uint64_t b = reinterpret_cast<uint64_t>(p);
  return f32_view(b, rows, cols, ld, 1, device, b, b + 4 * uint64_t(rows) * ld);
}
// K elements summed in tensor memory at a time. The tensor core's additions
// truncate, and the error of a product is that of one chunk: 2.1e-6 relative at
// the node's 256, 1.2e-6 at 128, 7.9e-7 at 64, 5.7e-7 at 32, for 256 / 272 / 290
// / 323 us at 2048 x 4096 x 4096. A layer's f32 sums are kept below 1e-6.
constexpr int kF32Chunk = 64;

mmr_matmul_desc f32_desc(const Handle* h, int math, const mmr_view& lhs, const mmr_view& rhs, const mmr_view& out,
                         const Ref* bias) {
  mmr_matmul_desc d{};
  d.lhs = lhs;
  d.rhs = rhs;
  d.out = out;
  d.epilogue = MMR_EPI_NONE;
  if (bias && bias->on) {
    d.epilogue = MMR_EPI_BIAS;
    d.bias.address = bias->lo;
    d.bias.bytes = bias->hi - bias->lo;
    d.bias.base_offset_bytes = bias->base - bias->lo;
    d.bias.rank = 1;
    d.bias.device_ordinal = h->device;
    d.bias.dims[0] = bias->d[2];
    d.bias.strides[0] = bias->s[2];
  }
  d.math_mode = math;
  d.family = MMR_FAMILY_AUTO;
  d.device_ordinal = h->device;
  d.stream = h->stream;
  return d;
}

int32_t add_f32_product(Handle* h, const mmr_matmul_desc& d) {
  mmr_gemm_handle* g = nullptr;
  MMR_TRY(mmr_gemm_bind(&d, &g));
  h->products.push_back(g);
  mmr::gemm_set_chunk(g, kF32Chunk);
  mmr_gemm_info info{};
  MMR_TRY(mmr_gemm_query(g, &info));
  const char* what = info.family == MMR_FAMILY_TCGEN05 ? "matmul node (f32, tcgen05)"
                     : info.family == MMR_FAMILY_GEMV  ? "matmul node (f32, gemv)"
                                                       : "matmul node (f32, simt)";
  h->plan += what;
  h->plan += "\n";
  h->steps.push_back({what, [g](cudaStream_t s) { return mmr::gemm_enqueue(g, s); }});
  return MMR_OK;
}

// An f32 matrix as a product reads it: rows x cols with element strides.
struct F32Mat {
  uint64_t base = 0;
  int64_t rows = 0, cols = 0, s_r = 0, s_c = 0;
  F32Mat t() const { return {base, cols, rows, s_c, s_r}; }
};
F32Mat f32_mat(const Ref& r) { return {r.base, r.d[1], r.d[2], r.s[1], r.s[2]}; }

// The same matrix with strides that TMA takes on axes of extent 1, whose strides
// say nothing.
F32Mat f32_plain(F32Mat o) {
  if (o.rows == 1) o.s_r = ((o.cols - 1) * std::abs(o.s_c) + 4) / 4 * 4;
  if (o.cols == 1) o.s_c = o.rows > 1 && o.s_r == 1 ? (o.rows + 3) / 4 * 4 : 1;
  return o;
}

// As TMA wants it: one axis contiguous, the other a pitch of whole 16 bytes.
bool f32_aligned(const F32Mat& o) {
  auto pitch = [](int64_t s, int64_t extent) { return s % 4 == 0 && s >= extent; };
  return o.base % 16 == 0 && ((o.s_c == 1 && pitch(o.s_r, o.cols)) || (o.s_r == 1 && pitch(o.s_c, o.rows)));
}

// A batch of `parts` views along the contraction of a (axis `cols`) or b (`rows`).
mmr_view f32_parts_view(const F32Mat& o, bool along_cols, int parts, int64_t each, int device) {
  mmr_view v{};
  const int64_t rows = along_cols ? o.rows : each, cols = along_cols ? each : o.cols;
  const int64_t step = each * (along_cols ? o.s_c : o.s_r);
  v.rank = 3;
  v.device_ordinal = device;
  v.dims[0] = parts;
  v.dims[1] = rows;
  v.dims[2] = cols;
  v.strides[0] = step;
  v.strides[1] = o.s_r;
  v.strides[2] = o.s_c;
  v.address = o.base;
  v.bytes = 4 * uint64_t((parts - 1) * step + (rows - 1) * o.s_r + (cols - 1) * o.s_c + 1);
  return v;
}

// Up to eight rows against a K-contiguous b: one launch for all (1 x 4096 x 4096
// 184 -> 15 us). False: not this kernel's case.
bool add_f32_dot(Handle* h, int math, const F32Mat& a, const F32Mat& b, int act, const mmr::ActResParams& post) {
  const int64_t m = a.rows, k = a.cols;
  if (math == MMR_MATH_EXACT || m > 8 || (b.s_r != 1 && k != 1)) return false;
  mmr::DotParams p;
  p.a = reinterpret_cast<const float*>(a.base);
  p.b = reinterpret_cast<const float*>(b.base);
  p.a_m = a.s_r;
  p.a_k = a.s_c;
  p.b_n = b.s_c;
  p.k = int(k);
  p.act = act;
  p.post = post;
  const bool vec = k % 4 == 0 && b.base % 16 == 0 && b.s_c % 4 == 0 && a.s_c == 1 && a.base % 16 == 0 &&
                   (a.s_r % 4 == 0 || m == 1);
  using K = void (*)(const mmr::DotParams);
  const K kernel = m == 1   ? (vec ? mmr::mmr_dot_kernel<1, true> : mmr::mmr_dot_kernel<1, false>)
                   : m == 2 ? (vec ? mmr::mmr_dot_kernel<2, true> : mmr::mmr_dot_kernel<2, false>)
                   : m <= 4 ? (vec ? mmr::mmr_dot_kernel<4, true> : mmr::mmr_dot_kernel<4, false>)
                            : (vec ? mmr::mmr_dot_kernel<8, true> : mmr::mmr_dot_kernel<8, false>);
  const int grid = int(std::min<int64_t>((b.cols + 7) / 8, 16 * h->sms));
  add_step(h, "mmr_dot_kernel grid %lld", [=](cudaStream_t s) {
    return mmr::launch_kernel(kernel, dim3(grid), dim3(256), 0, s, dim3(1, 1, 1), p);
  }, grid);
  return true;
}

// x = a b, bare, in f32: into `out` where that can hold it, else into a
// workspace; *x says where, in *parts K parts that the reader adds. *direct: the
// whole product lies in out. A bias that is all that follows the product may be
// given; *biased: the node's epilogue adds it.
//
// The MatMul node, whose own admission decides its kernel for these views: the
// streaming ones where they take the operands, else the tensor-core ones, with
// operands that TMA cannot read packed first, an output or a bias that would send
// the whole product to the scalar kernel left to the pass that follows, and a K
// that is long for its few tiles divided into a batch of parts. The streaming
// kernels end at a K of 8192 (16 x 500 x 8193: 1823 us and 1.6e-6 on the scalar
// kernel, 55 us and 7.8e-7 in parts). 100 x 1000 x 8000: 347 -> 43 us; packed as
// well, 500 x 77 x 5000: 732 -> 36 us. The parts'
// number is the one of least estimated time: 0.42 us a 16-wide k-block on the
// CTA-pair kernel, 0.72 on the one-CTA kernel (up to 128 rows).
int32_t add_f32_bare(Handle* h, int math, F32Mat a, F32Mat b, F32Mat out, bool out_free, const Ref* bias, EpiMat* x,
                     int* parts, bool* direct, bool* biased) {
  const int64_t m = a.rows, k = a.cols, n = b.cols;
  const int dev = h->device;
  a = f32_plain(a);
  b = f32_plain(b);
  out = f32_plain(out);
  if (n == 1) out.s_c = 1;  // its rows keep their pitch
  auto use_out = [&] {
    x->p = reinterpret_cast<void*>(out.base);
    x->ld = out.s_r;
    x->cs = out.s_c;
    x->vec = out.s_c == 1 && out.base % 16 == 0 && (out.s_r % 4 == 0 || m == 1) && n > 1;
    *parts = 1;
    *direct = true;
  };
  auto use_workspace = [&](int count) -> int32_t {
    const int64_t ld = (n + 3) / 4 * 4;
    void* w = nullptr;
    MMR_TRY(workspace(h, __int128(count) * m * ld * 4, &w));
    x->p = w;
    x->bs = m * ld;
    x->ld = ld;
    x->cs = 1;
    x->vec = 1;
    *parts = count;
    *direct = false;
    return MMR_OK;
  };
  auto plain_view = [&](const F32Mat& o) {
    // the view's own bytes, from its lowest element (bounds were checked against its buffer)
    const int64_t lo = std::min<int64_t>(0, (o.rows - 1) * o.s_r) + std::min<int64_t>(0, (o.cols - 1) * o.s_c);
    const int64_t hi = std::max<int64_t>(0, (o.rows - 1) * o.s_r) + std::max<int64_t>(0, (o.cols - 1) * o.s_c);
    return f32_view(o.base, o.rows, o.cols, o.s_r, o.s_c, dev, o.base + 4 * lo, o.base + 4 * (hi + 1));
  };
  // The family that the node takes for out = a b (+ bias); -1: none.
  auto family = [&](const F32Mat& a, const F32Mat& b, const F32Mat& out, const Ref* bias) {
    const mmr_matmul_desc d = f32_desc(h, math, plain_view(a), plain_view(b), plain_view(out), bias);
    mmr_gemm_info info{};
    return mmr_gemm_validate(&d, &info) == MMR_OK ? int(info.family) : -1;
  };
  // Row-major stand-ins at addresses that meet nothing, for a matrix still to be packed or allocated.
  const F32Mat packed_b = {uint64_t(1) << 60, k, n, (n + 3) / 4 * 4, 1}, own_out = {uint64_t(1) << 61, m, n, (n + 3) / 4 * 4, 1};
  auto node = [&](int want) -> int32_t {
    if (out_free && family(a, b, out, nullptr) == want) use_out();
    else MMR_TRY(use_workspace(1));
    *biased = *direct && bias && bias->on && family(a, b, out, bias) == want;
    return add_f32_product(h, f32_desc(h, math, plain_view(a), plain_view(b),
                                       *direct ? plain_view(out) : f32_view(x->p, m, n, x->ld, dev), *biased ? bias : nullptr));
  };
  *biased = false;
  if (k == 0) {
    MMR_TRY(use_workspace(1));
    void* w = x->p;
    const size_t bytes = size_t(m) * x->ld * 4;
    add_step(h, "zeros", [=](cudaStream_t s) { return cudaMemsetAsync(w, 0, bytes, s); });
    return MMR_OK;
  }
  if (math == MMR_MATH_EXACT) return node(MMR_FAMILY_SIMT);  // sums in the node's own order
  const bool stream = b.s_c == 1 && family(a, f32_aligned(b) ? b : packed_b, own_out, nullptr) == MMR_FAMILY_GEMV;
  int count = 1;
  if (!stream) {
    const int64_t tiles = m > 128 ? (m + 255) / 256 * ((n + 255) / 256) : (n + 255) / 256;
    const int64_t units = m > 128 ? h->sms / 2 : h->sms;
    const double t = m > 128 ? 0.42 : 0.72;
    const int64_t blocks = (k + 15) / 16;
    double best = 0;
    for (int s = 1; s <= 16 && blocks >= 4 * s; s *= 2) {
      const double us = double((tiles * s + units - 1) / units) * double((blocks + s - 1) / s) * t +
                        (s > 1 ? 2.0 + double(s) * m * n * 8 / 4e6 : 0.0) +
                        (s > 1 && k % (4 * s) ? 3.0 + double(m + n) * k * 8 / 3e6 : 0.0);
      if (s == 1 || us < best) {
        best = us;
        count = s;
      }
    }
  }
  // K of each part, and the padded K when the parts are not equal as they lie.
  const bool uneven = count > 1 && k % (4 * count) != 0;
  const int64_t each = uneven ? ((k + count - 1) / count + 15) / 16 * 16 : k / count, k_padded = uneven ? each * count : k;
  mmr::PackList packs;
  auto pack = [&](F32Mat* o, bool k_is_cols) -> int32_t {
    const bool cols_inner = stream || std::abs(o->s_c) <= std::abs(o->s_r);  // streaming: a row-major b
    mmr::PackParams q;
    q.src = reinterpret_cast<const void*>(o->base);
    q.rows = int(cols_inner ? o->rows : o->cols);
    q.cols = int(cols_inner ? o->cols : o->rows);
    q.s_r = cols_inner ? o->s_r : o->s_c;
    q.s_c = cols_inner ? o->s_c : o->s_r;
    const bool k_inner = cols_inner == k_is_cols;
    q.pitch = int(((k_inner ? k_padded : int64_t(q.cols)) + 3) / 4 * 4);
    q.rows_out = int(k_inner ? int64_t(q.rows) : k_padded);
    MMR_TRY(workspace(h, __int128(q.rows_out) * q.pitch * 4, &q.dst));
    packs.p[packs.n++] = q;
    o->base = reinterpret_cast<uint64_t>(q.dst);
    (cols_inner ? o->s_r : o->s_c) = q.pitch;
    (cols_inner ? o->s_c : o->s_r) = 1;
    (k_is_cols ? o->cols : o->rows) = k_padded;
    return MMR_OK;
  };
  if (!stream && (uneven || !f32_aligned(a))) MMR_TRY(pack(&a, true));
  if (uneven || !f32_aligned(b)) MMR_TRY(pack(&b, false));
  add_packs(h, packs, 4);
  if (count == 1) return node(stream ? MMR_FAMILY_GEMV : MMR_FAMILY_TCGEN05);
  MMR_TRY(use_workspace(count));
  mmr_view to = f32_view(x->p, m, n, x->ld, dev);
  to.rank = 3;
  to.dims[0] = count;
  to.dims[1] = m;
  to.dims[2] = n;
  to.strides[0] = x->bs;
  to.strides[1] = x->ld;
  to.strides[2] = 1;
  to.bytes = 4 * uint64_t(count) * x->bs;
  return add_f32_product(h, f32_desc(h, math, f32_parts_view(a, true, count, each, dev),
                                     f32_parts_view(b, false, count, each, dev), to, nullptr));
}

// pre = sum of x's parts + bias; out = act(pre) + residual. In EXACT mode the
// activation is the node's, bit for bit.
void add_act_res(Handle* h, int math, int act, const mmr::ActResParams& q) {
  const int grid = int(std::min<int64_t>((int64_t(q.m) * ((q.n + 127) / 128) + 7) / 8, 16 * h->sms));
  add_step(h, "mmr_act_res_kernel grid %lld, %lld parts", [=](cudaStream_t s) {
    using K = void (*)(const mmr::ActResParams);
    const K k = pick_act(act, [&](auto a) -> K {
      constexpr int kAct = decltype(a)::value;
      if constexpr (kAct != MMR_ACT_NONE)
        if (math == MMR_MATH_EXACT) return mmr::mmr_act_res_kernel<kAct, true>;
      return mmr::mmr_act_res_kernel<kAct, false>;
    });
    return mmr::launch_kernel(k, dim3(grid), dim3(256), 0, s, dim3(1, 1, 1), q);
  }, grid, q.parts);
}

int32_t check_math(int dtype, int math) {
  if (math < MMR_MATH_STRICT_FP32 || math > MMR_MATH_EXACT) return fail(MMR_ERR_INVALID_ARGUMENT, "unknown math mode %d", math);
  if (dtype != MMR_DTYPE_F32 && math != MMR_MATH_STRICT_FP32)
    return fail(MMR_ERR_UNSUPPORTED_MATH, "%s operands are multiplied exactly with f32 sums: the math mode is StrictFp32",
                dtype_name(dtype));
  return MMR_OK;
}

int32_t check_act(int act) {
  if (act < MMR_ACT_NONE || act > MMR_ACT_SILU) return fail(MMR_ERR_INVALID_ARGUMENT, "unknown activation %d", act);
  return MMR_OK;
}

// The logical matrix of a view given transposed.
void untranspose(Ref* r) {
  std::swap(r->d[1], r->d[2]);
  std::swap(r->s[1], r->s[2]);
}

Operand operand(const Ref& r, bool rows_are_mn) {
  Operand o;
  o.base = r.base;
  o.mn = rows_are_mn ? r.d[1] : r.d[2];
  o.k = rows_are_mn ? r.d[2] : r.d[1];
  o.s_mn = rows_are_mn ? r.s[1] : r.s[2];
  o.s_k = rows_are_mn ? r.s[2] : r.s[1];
  return o;
}

// out = A B with no bias, activation or residual; written along out's unit
// stride (out^T = B^T A^T where that is the row axis).
int32_t add_plain_product(Handle* h, int dtype, Operand a, Operand b, Ref out) {
  if (out.s[2] != 1 && out.s[1] == 1) {
    std::swap(a, b);
    untranspose(&out);
  }
  mmr::EpiParams epi;
  epi.out = epi_mat(out);
  return add_product(h, dtype, a, b, epi, nullptr);
}

// ----------------------------------------------------------------- linear --
int32_t linear_bind(const mmr_linear_desc* d, Handle** out) {
  if (!out) return fail(MMR_ERR_INVALID_ARGUMENT, "null output handle pointer");
  *out = nullptr;
  if (!d) return fail(MMR_ERR_INVALID_ARGUMENT, "null descriptor");
  const int dev = d->device_ordinal;
  Ref lhs, rhs, o, bias, res, pre;
  MMR_TRY(check_act(d->activation));
  MMR_TRY(read_tensor(d->lhs, "lhs", dev, 2, kFloat, &lhs));
  MMR_TRY(check_math(lhs.dtype, d->math_mode));
  MMR_TRY(read_tensor(d->rhs, "rhs", dev, 2, kFloat, &rhs));
  MMR_TRY(read_tensor(d->out, "out", dev, 2, kFloat, &o));
  if (present(d->bias)) MMR_TRY(read_tensor(d->bias, "bias", dev, 1, kFloat, &bias));
  if (present(d->residual)) MMR_TRY(read_tensor(d->residual, "residual", dev, 2, kFloat, &res));
  if (present(d->pre)) MMR_TRY(read_tensor(d->pre, "pre", dev, 2, kFloat, &pre));
  for (const Ref* r : {&rhs, &o, &bias, &res, &pre})
    if (r->on) MMR_TRY(same_dtype(*r, lhs.dtype));
  if (d->transpose_lhs) untranspose(&lhs);
  if (d->transpose_rhs) untranspose(&rhs);
  const int64_t m = lhs.d[1], k = lhs.d[2], n = rhs.d[2];
  MMR_TRY(want_dims(rhs, {k, n}));
  MMR_TRY(want_dims(o, {m, n}));
  if (bias.on) MMR_TRY(want_dims(bias, {n}));
  if (res.on) MMR_TRY(want_dims(res, {m, n}));
  if (pre.on) MMR_TRY(want_dims(pre, {m, n}));
  MMR_TRY(check_aliasing({&o, &pre}, {&lhs, &rhs, &bias, &res}, &res));
  int sms = 0;
  MMR_TRY(check_device(dev, {&lhs, &rhs, &o, &bias, &res, &pre}, &sms));
  DeviceGuard guard(dev);
  if (!guard.ok) return fail(MMR_ERR_CUDA, "cudaSetDevice(%d) failed", dev);
  Owned h;
  MMR_TRY(new_handle(dev, sms, d->stream, &h));
  if (m == 0 || n == 0) {
    *out = h.release();
    return MMR_OK;
  }
  if (lhs.dtype == MMR_DTYPE_F32) {
    // The bare product, then one pass for what follows it. The node's own
    // epilogue takes an activation as a call per element: 2048 x 4096 x 4096 with
    // bias and SiLU took 375 us in it, 256 bare.
    mmr::ActResParams q;
    const Ref& to = pre.on ? pre : o;
    const bool to_free = pre.on || !res.on || !overlap(o, res);
    const bool more = res.on || pre.on || d->activation != MMR_ACT_NONE;
    q.pre = epi_mat(pre);
    q.residual = epi_mat(res);
    q.out = epi_mat(o);
    q.bias = reinterpret_cast<const float*>(bias.on ? bias.base : 0);
    q.bias_s = bias.s[2];
    q.m = int(m);
    q.n = int(n);
    if (!add_f32_dot(h.get(), d->math_mode, f32_mat(lhs), f32_mat(rhs), d->activation, q)) {
      bool direct = false, biased = false;
      MMR_TRY(add_f32_bare(h.get(), d->math_mode, f32_mat(lhs), f32_mat(rhs), f32_mat(to), to_free,
                           more ? nullptr : &bias, &q.x, &q.parts, &direct, &biased));
      if (!direct || more || (bias.on && !biased)) add_act_res(h.get(), d->math_mode, d->activation, q);
    }
  } else {
    mmr::EpiParams epi;
    epi.out = epi_mat(o);
    epi.pre = epi_mat(pre);
    epi.residual = epi_mat(res);
    epi.bias = reinterpret_cast<const void*>(bias.on ? bias.base : 0);
    epi.bias_s = bias.s[2];
    epi.act = d->activation;
    MMR_TRY(add_product(h.get(), lhs.dtype, operand(lhs, true), operand(rhs, false), epi, nullptr));
  }
  *out = h.release();
  return MMR_OK;
}

int32_t linear_grad_bind(const mmr_linear_grad_desc* d, Handle** out) {
  if (!out) return fail(MMR_ERR_INVALID_ARGUMENT, "null output handle pointer");
  *out = nullptr;
  if (!d) return fail(MMR_ERR_INVALID_ARGUMENT, "null descriptor");
  const int dev = d->device_ordinal;
  Ref dy, lhs, rhs, pre, dl, dr, db;
  MMR_TRY(check_act(d->activation));
  MMR_TRY(read_tensor(d->d_out, "d_out", dev, 2, kFloat, &dy));
  MMR_TRY(check_math(dy.dtype, d->math_mode));
  MMR_TRY(read_tensor(d->lhs, "lhs", dev, 2, kFloat, &lhs));
  MMR_TRY(read_tensor(d->rhs, "rhs", dev, 2, kFloat, &rhs));
  if (d->activation != MMR_ACT_NONE) MMR_TRY(read_tensor(d->pre, "pre", dev, 2, kFloat, &pre));
  if (present(d->d_lhs)) MMR_TRY(read_tensor(d->d_lhs, "d_lhs", dev, 2, kFloat, &dl));
  if (present(d->d_rhs)) MMR_TRY(read_tensor(d->d_rhs, "d_rhs", dev, 2, kFloat, &dr));
  if (present(d->d_bias)) MMR_TRY(read_tensor(d->d_bias, "d_bias", dev, 1, kFloat, &db));
  if (!dl.on && !dr.on && !db.on) return fail(MMR_ERR_INVALID_ARGUMENT, "no gradient is asked for");
  for (const Ref* r : {&lhs, &rhs, &pre, &dl, &dr, &db})
    if (r->on) MMR_TRY(same_dtype(*r, dy.dtype));
  if (d->transpose_lhs) {
    untranspose(&lhs);
    untranspose(&dl);
  }
  if (d->transpose_rhs) {
    untranspose(&rhs);
    untranspose(&dr);
  }
  const int64_t m = lhs.d[1], k = lhs.d[2], n = rhs.d[2];
  MMR_TRY(want_dims(rhs, {k, n}));
  MMR_TRY(want_dims(dy, {m, n}));
  if (pre.on) MMR_TRY(want_dims(pre, {m, n}));
  if (dl.on) MMR_TRY(want_dims(dl, {m, k}));
  if (dr.on) MMR_TRY(want_dims(dr, {k, n}));
  if (db.on) MMR_TRY(want_dims(db, {n}));
  MMR_TRY(check_aliasing({&dl, &dr, &db}, {&dy, &lhs, &rhs, &pre}));
  int sms = 0;
  MMR_TRY(check_device(dev, {&dy, &lhs, &rhs, &pre, &dl, &dr, &db}, &sms));
  DeviceGuard guard(dev);
  if (!guard.ok) return fail(MMR_ERR_CUDA, "cudaSetDevice(%d) failed", dev);
  Owned h;
  MMR_TRY(new_handle(dev, sms, d->stream, &h));
  Ref dp;
  MMR_TRY(add_act_grad(h.get(), d->activation, dy, pre, db, &dp, nullptr, nullptr));
  if (dy.dtype == MMR_DTYPE_F32) {
    // out^T = B^T A^T where the gradient's unit stride is its row axis
    auto product = [&](F32Mat a, F32Mat b, const Ref& o) -> int32_t {
      if (o.lo == o.hi) return MMR_OK;
      F32Mat v = f32_mat(o);
      if (v.s_c != 1 && v.s_r == 1) {
        std::swap(a, b);
        a = a.t();
        b = b.t();
        v = v.t();
      }
      mmr::ActResParams q;
      q.out.p = reinterpret_cast<void*>(v.base);
      q.out.ld = v.s_r;
      q.out.cs = v.s_c;
      q.out.vec = v.s_c == 1 && v.base % 16 == 0 && (v.s_r % 4 == 0 || v.rows == 1) && v.cols > 1;
      q.m = int(v.rows);
      q.n = int(v.cols);
      if (add_f32_dot(h.get(), d->math_mode, a, b, MMR_ACT_NONE, q)) return MMR_OK;
      bool direct = false, biased = false;
      MMR_TRY(add_f32_bare(h.get(), d->math_mode, a, b, v, true, nullptr, &q.x, &q.parts, &direct, &biased));
      if (!direct) add_act_res(h.get(), d->math_mode, MMR_ACT_NONE, q);
      return MMR_OK;
    };
    const F32Mat dpm = f32_mat(dp);
    if (dl.on) MMR_TRY(product(dpm, f32_mat(rhs).t(), dl));
    if (dr.on) MMR_TRY(product(f32_mat(lhs).t(), dpm, dr));
  } else {
    if (dl.on) MMR_TRY(add_plain_product(h.get(), dy.dtype, operand(dp, true), operand(rhs, true), dl));
    if (dr.on) MMR_TRY(add_plain_product(h.get(), dy.dtype, operand(lhs, false), operand(dp, false), dr));
  }
  *out = h.release();
  return MMR_OK;
}

// ---------------------------------------------------------------- experts --
int32_t expert_rows(int64_t tokens, int64_t top_k, int64_t experts, int64_t align, int64_t* rows) {
  if (tokens < 0 || top_k < 1 || top_k > 1024 || experts < 1 || experts > mmr::ES_MAX_EXPERTS)
    return fail(MMR_ERR_INVALID_SHAPE, "expert layout of %lld tokens, %lld choices, %lld experts: 1..1024 choices and 1..%d experts",
                (long long)tokens, (long long)top_k, (long long)experts, mmr::ES_MAX_EXPERTS);
  if (align < 1 || align > 128 || (align & (align - 1)))
    return fail(MMR_ERR_INVALID_ARGUMENT, "row_align %lld is not a power of two up to 128", (long long)align);
  if (tokens > ((int64_t(1) << 31) - (1 << 18)) / top_k)
    return fail(MMR_ERR_INVALID_SHAPE, "more than 2^31 assignments");
  const int64_t n = tokens * top_k;
  *rows = (n + std::min(experts, n) * (align - 1)) / align * align;
  return MMR_OK;
}

struct Layout {
  Ref slots, sources, offsets, counts;
  int64_t tokens = 0, top_k = 0, experts = 0, align = 1, rows = 0;
  int* p(const Ref& r) const { return reinterpret_cast<int*>(r.base); }
  Groups groups() const {
    Groups g;
    g.experts = int(experts);
    g.offsets = p(offsets);
    g.counts = p(counts);
    g.rows = rows;
    g.assignments = tokens * top_k;
    return g;
  }
};

int32_t read_layout(const mmr_expert_layout& l, int dev, Layout* o) {
  MMR_TRY(expert_rows(l.tokens, l.top_k, l.experts, l.row_align, &o->rows));
  o->tokens = l.tokens;
  o->top_k = l.top_k;
  o->experts = l.experts;
  o->align = l.row_align;
  MMR_TRY(read_tensor(l.slots, "slots", dev, 2, kI32, &o->slots));
  MMR_TRY(read_tensor(l.sources, "sources", dev, 1, kI32, &o->sources));
  MMR_TRY(read_tensor(l.offsets, "offsets", dev, 1, kI32, &o->offsets));
  MMR_TRY(read_tensor(l.counts, "counts", dev, 1, kI32, &o->counts));
  MMR_TRY(want_dims(o->slots, {o->tokens, o->top_k}));
  MMR_TRY(want_dims(o->sources, {o->rows}));
  MMR_TRY(want_dims(o->offsets, {o->experts + 1}));
  MMR_TRY(want_dims(o->counts, {o->experts}));
  for (const Ref* r : {&o->slots, &o->sources, &o->offsets, &o->counts})
    if ((r->d[2] > 1 && r->s[2] != 1) || (r->rank == 2 && r->d[1] > 1 && r->s[1] != r->d[2]))
      return fail(MMR_ERR_UNSUPPORTED_LAYOUT, "%s: the layout's arrays are contiguous", r->name);
  return MMR_OK;
}

// The row length in vectors of the widest kind that every row allows, and that
// kind's bytes: 16, 8, 4 or (16-bit types) 2.
int32_t row_vector(std::initializer_list<const Ref*> refs, int64_t width, int* vb) {
  *vb = 16;
  for (const Ref* r : refs) {
    if (!r->on) continue;
    if (r->d[2] > 1 && r->s[2] != 1)
      return fail(MMR_ERR_UNSUPPORTED_LAYOUT, "%s: rows must have unit column stride", r->name);
    while (r->base % *vb || (r->d[1] > 1 && (r->s[1] * r->es) % *vb) || (width * r->es) % *vb) *vb /= 2;
  }
  return MMR_OK;
}

mmr::RowMat row_mat(const Ref& r) {
  mmr::RowMat m;
  if (!r.on) return m;
  m.p = reinterpret_cast<void*>(r.base);
  m.ld = r.s[1] * r.es;
  return m;
}

int32_t dispatch_bind(const mmr_dispatch_desc* d, Handle** out) {
  if (!out) return fail(MMR_ERR_INVALID_ARGUMENT, "null output handle pointer");
  *out = nullptr;
  if (!d) return fail(MMR_ERR_INVALID_ARGUMENT, "null descriptor");
  const int dev = d->device_ordinal;
  Layout l;
  Ref ids, x, rows;
  MMR_TRY(read_layout(d->layout, dev, &l));
  MMR_TRY(read_tensor(d->ids, "ids", dev, 2, kI32, &ids));
  MMR_TRY(read_tensor(d->x, "x", dev, 2, kFloat, &x));
  MMR_TRY(read_tensor(d->rows, "rows", dev, 2, kFloat, &rows));
  MMR_TRY(same_dtype(rows, x.dtype));
  const int64_t width = x.d[2];
  MMR_TRY(want_dims(ids, {l.tokens, l.top_k}));
  MMR_TRY(want_dims(x, {l.tokens, width}));
  MMR_TRY(want_dims(rows, {l.rows, width}));
  MMR_TRY(check_aliasing({&rows, &l.slots, &l.sources, &l.offsets, &l.counts}, {&ids, &x}));
  int vb = 16;
  MMR_TRY(row_vector({&x, &rows}, width, &vb));
  int sms = 0;
  MMR_TRY(check_device(dev, {&ids, &x, &rows, &l.slots, &l.sources, &l.offsets, &l.counts}, &sms));
  DeviceGuard guard(dev);
  if (!guard.ok) return fail(MMR_ERR_CUDA, "cudaSetDevice(%d) failed", dev);
  Owned h;
  MMR_TRY(new_handle(dev, sms, d->stream, &h));
  mmr::DispatchParams p;
  p.ids = reinterpret_cast<const int*>(ids.base);
  p.ids_t = ids.s[1];
  p.ids_j = ids.s[2];
  p.tokens = int(l.tokens);
  p.top_k = int(l.top_k);
  p.experts = int(l.experts);
  p.align = int(l.align);
  p.rows = l.rows;
  p.slots = l.p(l.slots);
  p.sources = l.p(l.sources);
  p.offsets = l.p(l.offsets);
  p.counts = l.p(l.counts);
  p.x = row_mat(x);
  p.out = row_mat(rows);
  p.row_vecs = int(width * x.es / vb);
  // Enough CTAs to fill the GPU twice over, a whole number of tokens each.
  p.run = int(std::max<int64_t>(1, (l.tokens + 2 * sms - 1) / (2 * sms)));
  const int64_t need = (l.tokens + p.run - 1) / p.run;
  const int grid = int(std::max<int64_t>(need, std::min<int64_t>(2 * sms, 1 + l.rows / mmr::ES_WARPS)));
  if (l.tokens * l.top_k > mmr::ES_DIRECT) {
    void* w = nullptr;
    MMR_TRY(workspace(h.get(), __int128(grid) * l.experts * 4, &w));
    p.hist = static_cast<int*>(w);
    add_step(h.get(), "mmr_expert_hist_kernel grid %lld", [=](cudaStream_t s) {
      return mmr::launch_kernel(mmr::mmr_expert_hist_kernel, dim3(grid), dim3(mmr::ES_THREADS), p.experts * 4, s,
                                dim3(1, 1, 1), p);
    }, grid);
  }
  const int smem = mmr::dispatch_smem_bytes(p.experts);
  static_assert(mmr::dispatch_smem_bytes(mmr::ES_MAX_EXPERTS) <= 48 * 1024, "more than a launch has without asking");
  auto kernel = vb == 16 ? mmr::mmr_dispatch_kernel<16> : vb == 8 ? mmr::mmr_dispatch_kernel<8>
                : vb == 4 ? mmr::mmr_dispatch_kernel<4> : mmr::mmr_dispatch_kernel<2>;
  add_step(h.get(), "mmr_dispatch_kernel grid %lld, %lld-byte vectors", [=](cudaStream_t s) {
    return mmr::launch_kernel(kernel, dim3(grid), dim3(mmr::ES_THREADS), smem, s, dim3(1, 1, 1), p);
  }, grid, vb);
  *out = h.release();
  return MMR_OK;
}

// Picks the kernel for an element type and vector width.
#define MMR_PICK(KERNEL, dt, vb, X)                                                                            \
  ((dt) == MMR_DTYPE_F32                                                                                       \
       ? ((vb) == 16 ? KERNEL<float, 16, X> : (vb) == 8 ? KERNEL<float, 8, X> : KERNEL<float, 4, X>)           \
   : (dt) == MMR_DTYPE_BF16                                                                                    \
       ? ((vb) == 16 ? KERNEL<__nv_bfloat16, 16, X> : (vb) == 8 ? KERNEL<__nv_bfloat16, 8, X>                  \
          : (vb) == 4 ? KERNEL<__nv_bfloat16, 4, X> : KERNEL<__nv_bfloat16, 2, X>)                             \
       : ((vb) == 16 ? KERNEL<__half, 16, X> : (vb) == 8 ? KERNEL<__half, 8, X> : (vb) == 4 ? KERNEL<__half, 4, X> \
                                                                                            : KERNEL<__half, 2, X>))

int32_t combine_bind(const mmr_combine_desc* d, Handle** out) {
  if (!out) return fail(MMR_ERR_INVALID_ARGUMENT, "null output handle pointer");
  *out = nullptr;
  if (!d) return fail(MMR_ERR_INVALID_ARGUMENT, "null descriptor");
  const int dev = d->device_ordinal;
  Layout l;
  Ref rows, w, res, o;
  MMR_TRY(read_layout(d->layout, dev, &l));
  MMR_TRY(read_tensor(d->rows, "rows", dev, 2, kFloat, &rows));
  if (present(d->weights)) MMR_TRY(read_tensor(d->weights, "weights", dev, 2, kF32, &w));
  if (present(d->residual)) MMR_TRY(read_tensor(d->residual, "residual", dev, 2, kFloat, &res));
  MMR_TRY(read_tensor(d->out, "out", dev, 2, kFloat, &o));
  MMR_TRY(same_dtype(o, rows.dtype));
  if (res.on) MMR_TRY(same_dtype(res, rows.dtype));
  const int64_t width = rows.d[2];
  MMR_TRY(want_dims(rows, {l.rows, width}));
  MMR_TRY(want_dims(o, {l.tokens, width}));
  if (w.on) MMR_TRY(want_dims(w, {l.tokens, l.top_k}));
  if (res.on) MMR_TRY(want_dims(res, {l.tokens, width}));
  MMR_TRY(check_aliasing({&o}, {&rows, &w, &res, &l.slots}, &res));
  int vb = 16;
  MMR_TRY(row_vector({&rows, &res, &o}, width, &vb));
  int sms = 0;
  MMR_TRY(check_device(dev, {&rows, &w, &res, &o, &l.slots, &l.sources, &l.offsets, &l.counts}, &sms));
  DeviceGuard guard(dev);
  if (!guard.ok) return fail(MMR_ERR_CUDA, "cudaSetDevice(%d) failed", dev);
  Owned h;
  MMR_TRY(new_handle(dev, sms, d->stream, &h));
  if (l.tokens > 0 && width > 0) {
    mmr::CombineParams p;
    p.slots = l.p(l.slots);
    p.tokens = int(l.tokens);
    p.top_k = int(l.top_k);
    p.n_rows = int(l.rows);
    p.weights = reinterpret_cast<const float*>(w.on ? w.base : 0);
    p.w_t = w.s[1];
    p.w_j = w.s[2];
    p.rows = row_mat(rows);
    p.residual = row_mat(res);
    p.out = row_mat(o);
    p.row_vecs = int(width * rows.es / vb);
    const int64_t units = l.tokens * ((p.row_vecs + 127) / 128);
    const int grid = int(std::min<int64_t>(units, int64_t(1) << 30));
    auto kernel = MMR_PICK(mmr::mmr_combine_kernel, rows.dtype, vb, 4);
    add_step(h.get(), "mmr_combine_kernel grid %lld, %lld-byte vectors", [=](cudaStream_t s) {
      return mmr::launch_kernel(kernel, dim3(grid), dim3(128), 0, s, dim3(1, 1, 1), p);
    }, grid, vb);
  }
  *out = h.release();
  return MMR_OK;
}

int32_t combine_grad_bind(const mmr_combine_grad_desc* d, Handle** out) {
  if (!out) return fail(MMR_ERR_INVALID_ARGUMENT, "null output handle pointer");
  *out = nullptr;
  if (!d) return fail(MMR_ERR_INVALID_ARGUMENT, "null descriptor");
  const int dev = d->device_ordinal;
  Layout l;
  Ref dy, rows, w, dr, dw;
  MMR_TRY(read_layout(d->layout, dev, &l));
  MMR_TRY(read_tensor(d->d_out, "d_out", dev, 2, kFloat, &dy));
  if (present(d->weights)) MMR_TRY(read_tensor(d->weights, "weights", dev, 2, kF32, &w));
  if (present(d->d_rows)) MMR_TRY(read_tensor(d->d_rows, "d_rows", dev, 2, kFloat, &dr));
  if (present(d->d_weights)) {
    MMR_TRY(read_tensor(d->d_weights, "d_weights", dev, 2, kF32, &dw));
    MMR_TRY(read_tensor(d->rows, "rows", dev, 2, kFloat, &rows));
  }
  if (!dr.on && !dw.on) return fail(MMR_ERR_INVALID_ARGUMENT, "no gradient is asked for");
  const int64_t width = dy.d[2];
  MMR_TRY(want_dims(dy, {l.tokens, width}));
  for (const Ref* r : {&rows, &dr})
    if (r->on) {
      MMR_TRY(same_dtype(*r, dy.dtype));
      MMR_TRY(want_dims(*r, {l.rows, width}));
    }
  for (const Ref* r : {&w, &dw})
    if (r->on) MMR_TRY(want_dims(*r, {l.tokens, l.top_k}));
  MMR_TRY(check_aliasing({&dr, &dw}, {&dy, &rows, &w, &l.slots, &l.sources}));
  int vb = 16;
  MMR_TRY(row_vector({&dy, &rows, &dr}, width, &vb));
  int sms = 0;
  MMR_TRY(check_device(dev, {&dy, &rows, &w, &dr, &dw, &l.slots, &l.sources, &l.offsets, &l.counts}, &sms));
  DeviceGuard guard(dev);
  if (!guard.ok) return fail(MMR_ERR_CUDA, "cudaSetDevice(%d) failed", dev);
  Owned h;
  MMR_TRY(new_handle(dev, sms, d->stream, &h));
  mmr::CombineGradParams p;
  p.slots = l.p(l.slots);
  p.sources = l.p(l.sources);
  p.tokens = int(l.tokens);
  p.top_k = int(l.top_k);
  p.n_rows = l.rows;
  p.weights = reinterpret_cast<const float*>(w.on ? w.base : 0);
  p.w_t = w.s[1];
  p.w_j = w.s[2];
  p.d_out = row_mat(dy);
  p.rows = row_mat(rows);
  p.d_rows = row_mat(dr);
  p.d_weights = reinterpret_cast<float*>(dw.on ? dw.base : 0);
  p.dw_t = dw.s[1];
  p.dw_j = dw.s[2];
  p.row_vecs = int(width * dy.es / vb);
  p.zero_blocks = dr.on && width > 0 ? int(std::min<int64_t>((l.rows + 255) / 256, 4 * sms)) : 0;
  // A warp a token from eight warps an SM on; below that a block a token.
  const bool warps = l.tokens >= 8 * sms;
  const int grid = int(warps ? (l.tokens + 7) / 8 : l.tokens) + p.zero_blocks;
  auto kernel = warps ? MMR_PICK(mmr::mmr_combine_grad_kernel, dy.dtype, vb, 1)
                      : MMR_PICK(mmr::mmr_combine_grad_kernel, dy.dtype, vb, 8);
  if (grid > 0)
    add_step(h.get(), "mmr_combine_grad_kernel grid %lld, %lld-byte vectors", [=](cudaStream_t s) {
      return mmr::launch_kernel(kernel, dim3(grid), dim3(256), 0, s, dim3(1, 1, 1), p);
    }, grid, vb);
  *out = h.release();
  return MMR_OK;
}

// The experts' weights as a product's B: batch e, mn = columns of the product.
Operand weights_operand(const Ref& w, bool axis1_is_mn) {
  Operand o = operand(w, axis1_is_mn);
  o.batch = w.d[0];
  o.s_b = w.s[0];
  return o;
}

int32_t expert_linear_bind(const mmr_expert_linear_desc* d, Handle** out) {
  if (!out) return fail(MMR_ERR_INVALID_ARGUMENT, "null output handle pointer");
  *out = nullptr;
  if (!d) return fail(MMR_ERR_INVALID_ARGUMENT, "null descriptor");
  const int dev = d->device_ordinal;
  Layout l;
  Ref rows, w, bias, o, pre;
  MMR_TRY(check_act(d->activation));
  MMR_TRY(read_layout(d->layout, dev, &l));
  MMR_TRY(read_tensor(d->rows, "rows", dev, 2, kHalf, &rows));
  MMR_TRY(read_tensor(d->weights, "weights", dev, 3, kHalf, &w));
  MMR_TRY(read_tensor(d->out, "out", dev, 2, kHalf, &o));
  if (present(d->bias)) MMR_TRY(read_tensor(d->bias, "bias", dev, 2, kHalf, &bias));
  if (present(d->pre)) MMR_TRY(read_tensor(d->pre, "pre", dev, 2, kHalf, &pre));
  for (const Ref* r : {&w, &o, &bias, &pre})
    if (r->on) MMR_TRY(same_dtype(*r, rows.dtype));
  if (d->transpose_rhs) untranspose(&w);
  const int64_t k = rows.d[2], n = w.d[2];
  MMR_TRY(want_dims(rows, {l.rows, k}));
  MMR_TRY(want_dims(w, {l.experts, k, n}));
  MMR_TRY(want_dims(o, {l.rows, n}));
  if (pre.on) MMR_TRY(want_dims(pre, {l.rows, n}));
  if (bias.on) MMR_TRY(want_dims(bias, {l.experts, n}));
  MMR_TRY(check_aliasing({&o, &pre}, {&rows, &w, &bias, &l.offsets, &l.counts}));
  int sms = 0;
  MMR_TRY(check_device(dev, {&rows, &w, &o, &bias, &pre, &l.slots, &l.sources, &l.offsets, &l.counts}, &sms));
  DeviceGuard guard(dev);
  if (!guard.ok) return fail(MMR_ERR_CUDA, "cudaSetDevice(%d) failed", dev);
  Owned h;
  MMR_TRY(new_handle(dev, sms, d->stream, &h));
  mmr::EpiParams epi;
  epi.out = epi_mat(o);
  epi.pre = epi_mat(pre);
  epi.bias = reinterpret_cast<const void*>(bias.on ? bias.base : 0);
  epi.bias_bs = bias.s[1];
  epi.bias_s = bias.s[2];
  epi.act = d->activation;
  const Groups g = l.groups();
  MMR_TRY(add_product(h.get(), rows.dtype, operand(rows, true), weights_operand(w, false), epi, &g));
  *out = h.release();
  return MMR_OK;
}

int32_t expert_linear_grad_bind(const mmr_expert_linear_grad_desc* d, Handle** out) {
  if (!out) return fail(MMR_ERR_INVALID_ARGUMENT, "null output handle pointer");
  *out = nullptr;
  if (!d) return fail(MMR_ERR_INVALID_ARGUMENT, "null descriptor");
  const int dev = d->device_ordinal;
  Layout l;
  Ref dy, rows, w, pre, dr, dw, db;
  MMR_TRY(check_act(d->activation));
  MMR_TRY(read_layout(d->layout, dev, &l));
  MMR_TRY(read_tensor(d->d_out, "d_out", dev, 2, kHalf, &dy));
  MMR_TRY(read_tensor(d->rows, "rows", dev, 2, kHalf, &rows));
  MMR_TRY(read_tensor(d->weights, "weights", dev, 3, kHalf, &w));
  if (d->activation != MMR_ACT_NONE) MMR_TRY(read_tensor(d->pre, "pre", dev, 2, kHalf, &pre));
  if (present(d->d_rows)) MMR_TRY(read_tensor(d->d_rows, "d_rows", dev, 2, kHalf, &dr));
  if (present(d->d_weights)) MMR_TRY(read_tensor(d->d_weights, "d_weights", dev, 3, kHalf, &dw));
  if (present(d->d_bias)) MMR_TRY(read_tensor(d->d_bias, "d_bias", dev, 2, kHalf, &db));
  if (!dr.on && !dw.on && !db.on) return fail(MMR_ERR_INVALID_ARGUMENT, "no gradient is asked for");
  for (const Ref* r : {&rows, &w, &pre, &dr, &dw, &db})
    if (r->on) MMR_TRY(same_dtype(*r, dy.dtype));
  if (d->transpose_rhs) {
    untranspose(&w);
    untranspose(&dw);
  }
  const int64_t k = rows.d[2], n = dy.d[2];
  MMR_TRY(want_dims(dy, {l.rows, n}));
  MMR_TRY(want_dims(rows, {l.rows, k}));
  MMR_TRY(want_dims(w, {l.experts, k, n}));
  if (pre.on) MMR_TRY(want_dims(pre, {l.rows, n}));
  if (dr.on) MMR_TRY(want_dims(dr, {l.rows, k}));
  if (dw.on) MMR_TRY(want_dims(dw, {l.experts, k, n}));
  if (db.on) MMR_TRY(want_dims(db, {l.experts, n}));
  if ((dw.on || db.on) && l.align % mmr::AG_ROWS)
    return fail(MMR_ERR_UNSUPPORTED_LAYOUT, "d_weights and d_bias need a row_align of 64 or 128, not %lld", (long long)l.align);
  MMR_TRY(check_aliasing({&dr, &dw, &db}, {&dy, &rows, &w, &pre, &l.offsets, &l.counts, &l.sources}));
  int sms = 0;
  MMR_TRY(check_device(dev, {&dy, &rows, &w, &pre, &dr, &dw, &db, &l.slots, &l.sources, &l.offsets, &l.counts}, &sms));
  DeviceGuard guard(dev);
  if (!guard.ok) return fail(MMR_ERR_CUDA, "cudaSetDevice(%d) failed", dev);
  Owned h;
  MMR_TRY(new_handle(dev, sms, d->stream, &h));
  const Groups g = l.groups();
  Ref dp;
  MMR_TRY(add_act_grad(h.get(), d->activation, dy, pre, db, &dp, &g, l.p(l.sources)));
  if (dr.on) {
    mmr::EpiParams epi;
    epi.out = epi_mat(dr);
    MMR_TRY(add_product(h.get(), dy.dtype, operand(dp, true), weights_operand(w, true), epi, &g));
  }
  if (dw.on) {
    // d_weights[e] = rows_e^T d_pre_e, written along its unit stride
    Operand a = operand(rows, false), b = operand(dp, false);
    if (dw.s[2] != 1 && dw.s[1] == 1) {
      std::swap(a, b);
      untranspose(&dw);
    }
    MMR_TRY(add_segment_product(h.get(), dy.dtype, a, b, epi_mat(dw), g));
  }
  *out = h.release();
  return MMR_OK;
}

int32_t poll_event(cudaEvent_t ev, uint64_t timeout_ns) {
  const auto t0 = std::chrono::steady_clock::now();
  for (;;) {
    const cudaError_t e = cudaEventQuery(ev);
    if (e == cudaSuccess) return MMR_OK;
    if (e != cudaErrorNotReady) return fail(MMR_ERR_CUDA, "cudaEventQuery: %s", cudaGetErrorString(e));
    const auto el = std::chrono::duration_cast<std::chrono::nanoseconds>(std::chrono::steady_clock::now() - t0).count();
    if (uint64_t(el) > timeout_ns)
      return fail(MMR_ERR_TIMEOUT, "work did not complete within %llu ns", (unsigned long long)timeout_ns);
    std::this_thread::sleep_for(std::chrono::microseconds(50));
  }
}

int32_t run_on(Handle* h, cudaStream_t s) {
  std::lock_guard<std::mutex> lock(h->run_mu);
  DeviceGuard guard(h->device);
  if (!guard.ok) return fail(MMR_ERR_CUDA, "cudaSetDevice(%d) failed", h->device);
  cudaStreamCaptureStatus cap = cudaStreamCaptureStatusNone;
  MMR_CUDA(cudaStreamIsCapturing(s, &cap));
  const bool capturing = cap != cudaStreamCaptureStatusNone;
  // The workspaces are the handle's own: a run follows the last. Only the legacy
  // default stream is known by its value to be the stream of the last run: any
  // other value may have been destroyed and given out again, and
  // cudaStreamPerThread is another stream in every thread.
  if (!capturing && h->ran && (s != nullptr || h->last_stream != nullptr)) MMR_CUDA(cudaStreamWaitEvent(s, h->done, 0));
  int32_t rc = MMR_OK;
  for (const auto& step : h->steps)
    if ((rc = step.launch(s))) break;
  h->launched = true;
  if (!capturing) {  // also after a failed launch: those before it use the workspaces
    MMR_CUDA(cudaEventRecord(h->done, s));
    h->ran = true;
    h->last_stream = s;
  }
  return rc;
}

int32_t quiesce(Handle* h, uint64_t timeout_ns) {
  std::lock_guard<std::mutex> lock(h->quiesce_mu);
  bool ran = false, launched = false;
  {
    std::lock_guard<std::mutex> run_lock(h->run_mu);
    ran = h->ran;
    launched = h->launched;
  }
  if (!launched) return MMR_OK;
  DeviceGuard guard(h->device);
  if (!guard.ok) return fail(MMR_ERR_CUDA, "cudaSetDevice(%d) failed", h->device);
  if (ran) MMR_TRY(poll_event(h->done, timeout_ns));
  for (mmr_gemm_handle* g : h->products) MMR_TRY(mmr::gemm_read_error(g, timeout_ns));
  MMR_CUDA(cudaMemcpyAsync(h->h_err, h->d_err, sizeof(int), cudaMemcpyDeviceToHost, h->stream));
  MMR_CUDA(cudaEventRecord(h->err_ev, h->stream));
  MMR_TRY(poll_event(h->err_ev, timeout_ns));
  if (const int code = *h->h_err) {
    *h->h_err = 0;
    cudaMemsetAsync(h->d_err, 0, sizeof(int), h->stream);
    return fail(MMR_ERR_TIMEOUT, "kernel reported device error word %d (a bounded wait expired)", code);
  }
  return MMR_OK;
}

}  // namespace

extern "C" {

int32_t mmr_expert_rows(int64_t tokens, int64_t top_k, int64_t experts, int64_t row_align, int64_t* rows) {
  return guarded([&] {
    if (!rows) return fail(MMR_ERR_INVALID_ARGUMENT, "null output pointer");
    return expert_rows(tokens, top_k, experts, row_align, rows);
  });
}

int32_t mmr_linear_bind(const mmr_linear_desc* d, mmr_op_handle** out) {
  return guarded([&] { return linear_bind(d, out); });
}
int32_t mmr_linear_grad_bind(const mmr_linear_grad_desc* d, mmr_op_handle** out) {
  return guarded([&] { return linear_grad_bind(d, out); });
}
int32_t mmr_dispatch_bind(const mmr_dispatch_desc* d, mmr_op_handle** out) {
  return guarded([&] { return dispatch_bind(d, out); });
}
int32_t mmr_combine_bind(const mmr_combine_desc* d, mmr_op_handle** out) {
  return guarded([&] { return combine_bind(d, out); });
}
int32_t mmr_combine_grad_bind(const mmr_combine_grad_desc* d, mmr_op_handle** out) {
  return guarded([&] { return combine_grad_bind(d, out); });
}
int32_t mmr_expert_linear_bind(const mmr_expert_linear_desc* d, mmr_op_handle** out) {
  return guarded([&] { return expert_linear_bind(d, out); });
}
int32_t mmr_expert_linear_grad_bind(const mmr_expert_linear_grad_desc* d, mmr_op_handle** out) {
  return guarded([&] { return expert_linear_grad_bind(d, out); });
}

int32_t mmr_op_run_on(mmr_op_handle* h, void* stream) {
  return guarded([&] {
    if (!h) return fail(MMR_ERR_INVALID_ARGUMENT, "null handle");
    return run_on(h, reinterpret_cast<cudaStream_t>(stream));
  });
}
int32_t mmr_op_run(mmr_op_handle* h) {
  return guarded([&] {
    if (!h) return fail(MMR_ERR_INVALID_ARGUMENT, "null handle");
    return run_on(h, h->stream);
  });
}
int32_t mmr_op_quiesce(mmr_op_handle* h, uint64_t timeout_ns) {
  return guarded([&] {
    if (!h) return fail(MMR_ERR_INVALID_ARGUMENT, "null handle");
    return quiesce(h, timeout_ns);
  });
}
int32_t mmr_op_destroy(mmr_op_handle* h) {
  return guarded([&] {
    if (!h) return int32_t(MMR_OK);
    int32_t rc = MMR_OK;
    {
      DeviceGuard guard(h->device);
      if (h->ran && h->done) rc = poll_event(h->done, 10000000000ull);
      for (mmr_gemm_handle* g : h->products) {
        const int32_t r = mmr_gemm_destroy(g);
        if (rc == MMR_OK) rc = r;
      }
      for (void* p : h->workspaces) cudaFree(p);
      if (h->done) cudaEventDestroy(h->done);
      if (h->err_ev) cudaEventDestroy(h->err_ev);
      if (h->d_err) cudaFree(h->d_err);
      if (h->h_err) cudaFreeHost(h->h_err);
    }
    delete h;
    return rc;
  });
}
const char* mmr_op_plan(const mmr_op_handle* h) { return h ? h->plan.c_str() : ""; }

}  // extern "C"
