// qmm_api.hip — the C ABI of include/qmm.h: argument checks, the choice of
// kernel by activation rows (QCudaStorage::fwd's policy,
// vendor/candle/candle-core/src/quantized/cuda.rs:1653-1680, decided anew
// for MI355X), status codes, launch counters and host-side fault injection.
#include <atomic>
#include <cstdlib>
#include <cstring>
#include <mutex>
#include <set>
#include <utility>
#include <vector>

#include "../../include/qmm.h"
#include "qmm_device.h"
#include "qmm_launch.h"
#include "value_types.h"

namespace {

std::atomic<uint64_t> g_matvec_launches{0};
std::atomic<uint64_t> g_gemm_launches{0};
std::atomic<bool> g_fail_next{false};
std::atomic<uint64_t> g_moe_launches{0};
std::atomic<uint64_t> g_moe_prefill_launches{0};
// set_force_dmmv (quantized/cuda.rs:29-33): products of qmm_forward and its
// shared / GLU forms dequantize the weight against the f32 activation.
std::atomic<bool> g_force_dmmv{false};

int block_size(int type) {
  switch (type) {
    case qmm::T_Q8_0: case qmm::T_IQ4_NL: case qmm::T_MXFP4: return 32;
    case qmm::T_Q4_K: case qmm::T_Q6_K: return 256;
    default: return 0;
  }
}
int type_size(int type) {
  switch (type) {
    case qmm::T_Q8_0: return 34;
    case qmm::T_IQ4_NL: return 18;
    case qmm::T_MXFP4: return 17;
    case qmm::T_Q4_K: return 144;
    case qmm::T_Q6_K: return 210;
    default: return 0;
  }
}

// SWARMLLM_Q8K_SCALE=128: candle's Q8_K scale before SwarmLLM's #404 patch,
// the reference's A/B knob (vendor/candle/candle-core/src/quantized/k_quants.rs:145-152). Read once.
float q8k_scale() {
  static const float s = [] {
    const char* v = std::getenv("SWARMLLM_Q8K_SCALE");
    return (v && std::strcmp(v, "128") == 0) ? 128.0f : 127.0f;
  }();
  return s;
}

int status_of(hipError_t e) { return e == hipSuccess ? QMM_OK : QMM_DEVICE_ERROR; }

// A launch is judged by the runtime's last error afterwards; an error an
// earlier, unrelated call left behind is cleared first (mmq_entry.cu:120-122).
void clear_stale_error() { (void)hipGetLastError(); }

bool shape_ok(int type, int64_t k, int64_t n, int64_t rows) {
  const int qk = block_size(type);
  return qk != 0 && k > 0 && k % qk == 0 && n > 0 && rows > 0 && k <= (int64_t)1 << 30 && n <= ((int64_t)1 << 31) - 1;
}

// As the planes of an activation or a cache, or partial results, have to lie.
bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

// Rows of `width` bytes, `stride` (at least that) apart.
typedef __int128 wide;  // (a stride can be any number)
struct Region {
  const void* at;
  int64_t rows, width;
  wide stride;
};

// Whether two of them have a byte in common (rows between the other's rows have none).
bool overlap(const Region& a, const Region& b) {
  if (!a.at || !b.at || a.rows < 1 || b.rows < 1 || a.width < 1 || b.width < 1) return false;
  const wide pa = (uintptr_t)a.at, pb = (uintptr_t)b.at;
  if (pa + (wide)(a.rows - 1) * a.stride + a.width <= pb || pb + (wide)(b.rows - 1) * b.stride + b.width <= pa) return false;
  if (a.rows > b.rows) return overlap(b, a);
  auto floor_div = [](wide n, wide d) { return n / d - (n % d < 0 ? 1 : 0); };
  if (a.rows == 1 || a.stride == b.stride) {
    // b's row j lies pb - pa + m stride behind a's row i, m = j - i: the least m at which it ends behind its start
    const wide first = floor_div(pa - pb - b.width, b.stride) + 1, least = 1 - (wide)a.rows, m = first > least ? first : least;
    return m < b.rows && pb - pa + m * b.stride < a.width;
  }
  for (wide i = 0; i < a.rows; i++) {
    const wide at = pa + i * a.stride, first = floor_div(at - pb - b.width, b.stride) + 1, j = first > 0 ? first : 0;
    if (j < b.rows && pb + j * b.stride < at + a.width) return true;
  }
  return false;
}

// Whether an output (or the workspace) shares memory with an array that the call reads or writes, but for an
// output in its own y's place.
bool adapters_overlap(const qmm::LoraArgs& a, int x_dtype, int w_dtype, const void* workspace, size_t bytes) {
  const int64_t wb = qmm::value_bytes(w_dtype), slots = a.slots;
  auto whole = [](const void* p, int64_t n) { return Region{p, 1, n, n}; };
  auto rows = [&](const void* p, int64_t n, int64_t stride, int64_t size) { return Region{p, a.rows, n * size, (wide)stride * size}; };
  Region read[2 + 3 * qmm::kMaxTargets], out[qmm::kMaxTargets];
  int n = 0;
  read[n++] = rows(a.x, a.k, a.xs, qmm::value_bytes(x_dtype));
  read[n++] = whole(a.ids, 4 * a.rows);
  for (int i = 0; i < a.count; i++) {
    const qmm::LoraTarget& t = a.t[i];
    out[i] = rows(t.out, t.n, t.ldo, 4);
    read[n++] = whole(t.a, slots * t.rank * a.k * wb);
    read[n++] = whole(t.b, slots * t.n * t.rank * wb);
    read[n++] = whole(t.scales, 4 * slots);
  }
  const Region ws = whole(workspace, (int64_t)bytes);
  for (int i = 0; i < n; i++) {
    if (overlap(ws, read[i])) return true;
    for (int j = 0; j < a.count; j++)
      if (overlap(out[j], read[i])) return true;
  }
  for (int i = 0; i < a.count; i++) {
    const Region y = rows(a.t[i].y, a.t[i].n, a.t[i].ldy, 4);
    if (overlap(ws, out[i]) || overlap(ws, y)) return true;
    for (int j = 0; j < a.count; j++)
      if ((i < j && overlap(out[i], out[j])) || ((i != j || a.t[i].y != a.t[i].out) && overlap(y, out[j]))) return true;
  }
  return false;
}

// A paged cache's sizes: pages of 16 to 256 positions (a power of two), heads
// of a dim the attention kernels are built for, planes inside an int64.
bool cache_shape_ok(int64_t pages, int kv_heads, int head_dim, int page) {
  const bool hd = head_dim == 64 || head_dim == 96 || head_dim == 128 || head_dim == 256;
  return hd && page >= 16 && page <= 256 && (page & (page - 1)) == 0 && kv_heads >= 1 && kv_heads <= 65535 &&
         pages >= 1 && pages <= INT32_MAX;
}
bool cache_ok(const qmm_cache* c) {
  return c && cache_shape_ok(c->pages, c->kv_heads, c->head_dim, c->page) && c->k_codes && c->k_scales && c->v_codes &&
         c->v_scales && aligned16(c->k_codes) && aligned16(c->k_scales) && aligned16(c->v_codes) && aligned16(c->v_scales);
}
// Tokens of a cache write or read: 2^23 workgroups of 64 (a launch's threads stay below 2^32).
constexpr int64_t kMostCacheTokens = (int64_t)1 << 29;
qmm::CachePlanes planes_of(const qmm_cache& c) {
  return qmm::CachePlanes{(int8_t*)c.k_codes, (uint16_t*)c.k_scales, (int8_t*)c.v_codes, (uint16_t*)c.v_scales,
                          c.pages, c.kv_heads, c.head_dim, c.page};
}

// Compute units of the current device (256 on an MI355X), read once per device.
int cu_count() {
  static std::mutex mu;
  static int cached[64];
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) {
    (void)hipGetLastError();
    return 256;
  }
  std::lock_guard<std::mutex> lock(mu);
  if (!cached[dev]) {
    hipDeviceProp_t prop;
    cached[dev] = hipGetDeviceProperties(&prop, dev) == hipSuccess && prop.multiProcessorCount > 0
                      ? prop.multiProcessorCount
                      : 256;
    (void)hipGetLastError();
  }
  return cached[dev];
}

// The reference's few-rows line (mmq_takes_few_rows, mmq_fewest_rows_default,
// quantized/cuda.rs:775-839): K-quant products of 4 to 8 rows against a
// weight of 2 MiB or more go to the matrix cores, as do all of more than 8.
// The 32-value formats keep the decode kernels to 8 rows (their GEMM from 9:
// on MI355X the decode kernels read such a weight faster than a 128-row tile
// of 7-8 useful rows computes it).
constexpr int64_t kFewRowsLeastBytes = (int64_t)2 << 20;
constexpr int kFewRowsKQuant = 4;

// The reference's A/B switches for that line, each read once
// (quantized/cuda.rs:737-872):
//   SWARMLLM_QMATMUL_MMQ=dp4a|0|off|false   no matrix-core kernel (products
//       past the decode rows run on the decode kernels, 8 rows a launch);
//   SWARMLLM_QMATMUL_MMQ_MAX_ROWS=N         the matrix-core kernels take at most N rows;
//   SWARMLLM_QMATMUL_MMQ_MIN_ROWS=N         one few-rows line for every type
//       (N > 8: never below 9 rows);
//   SWARMLLM_QMATMUL_MMQ_FEW_ROWS_BYTES=B   the least weight bytes for a few-rows product (0: any);
//   SWARMLLM_QMATMUL_MMQ_CAPTURED=0|off|false  products of at most 8 rows on a
//       stream being captured stay on the decode kernels.
// A value that does not parse as a count leaves the default, as there.
struct MmqPolicy {
  bool on = true;
  int64_t max_rows = INT64_MAX;
  int64_t min_rows = -1;  // -1: per type
  int64_t few_bytes = kFewRowsLeastBytes;
  bool captured = true;
};

bool env_is_off(const char* v) {
  return v && (std::strcmp(v, "0") == 0 || std::strcmp(v, "off") == 0 || std::strcmp(v, "false") == 0);
}

// A decimal count (usize::parse: digits only, no sign or space), or -1.
int64_t env_count(const char* name) {
  const char* v = std::getenv(name);
  if (!v || !*v) return -1;
  int64_t r = 0;
  for (const char* c = v; *c; c++) {
    if (*c < '0' || *c > '9') return -1;
    if (r > (INT64_MAX - 9) / 10) return INT64_MAX;
    r = r * 10 + (*c - '0');
  }
  return r;
}

const MmqPolicy& mmq_policy() {
  static const MmqPolicy pol = [] {
    MmqPolicy p;
    const char* v = std::getenv("SWARMLLM_QMATMUL_MMQ");
    p.on = !(env_is_off(v) || (v && std::strcmp(v, "dp4a") == 0));
    const int64_t mx = env_count("SWARMLLM_QMATMUL_MMQ_MAX_ROWS");
    if (mx >= 0) p.max_rows = mx;
    p.min_rows = env_count("SWARMLLM_QMATMUL_MMQ_MIN_ROWS");
    const int64_t fb = env_count("SWARMLLM_QMATMUL_MMQ_FEW_ROWS_BYTES");
    if (fb >= 0) p.few_bytes = fb;
    p.captured = !env_is_off(std::getenv("SWARMLLM_QMATMUL_MMQ_CAPTURED"));
    return p;
  }();
  return pol;
}

bool is_kquant(int type) { return type == qmm::T_Q4_K || type == qmm::T_Q6_K; }

// SWARMLLM_QMATMUL_EXACT=1|on|true, read once: the exact Q4_K / Q6_K kernels
// only. Without it, three kernels feed the matrix cores a rounded product of
// a code and its sub-block scale (the single-pass Q4_K and Q6_K GEMMs from
// gemm_q4k_sp_min_rows() rows, the single-product form of the few-row Q6_K
// kernel from k = 2048), so a product's bits can depend on how many rows
// its batch has; with it, every row count sums exact int32 products.
bool env_is_on(const char* v) {
  return v && (std::strcmp(v, "1") == 0 || std::strcmp(v, "on") == 0 || std::strcmp(v, "true") == 0);
}

// The few-rows line of a type: (fewest rows, least weight bytes).
void few_rows_line(int type, int64_t& rows, int64_t& bytes) {
  const MmqPolicy& pol = mmq_policy();
  rows = pol.min_rows >= 0 ? pol.min_rows : (is_kquant(type) ? kFewRowsKQuant : qmm::gemm_b32_min_rows());
  bytes = pol.few_bytes;
}

// Types prepared on a device (qmm_prepare), a bit each: the reference's
// MMQ_FEW_ROWS_READY (quantized/cuda.rs:890-932). A product of at most 8
// rows on a stream being captured takes a matrix-core kernel only once its
// type is prepared on the current device; the first such product outside a
// capture prepares it (mmq_prepare_few_rows_once).
constexpr int kMaxDevices = 64;
std::atomic<uint32_t> g_prepared[kMaxDevices];
std::atomic<uint32_t> g_prepare_tried[kMaxDevices];

int type_bit(int type) {
  switch (type) {
    case qmm::T_Q8_0: return 1;
    case qmm::T_Q4_K: return 2;
    case qmm::T_Q6_K: return 4;
    case qmm::T_IQ4_NL: return 8;
    case qmm::T_MXFP4: return 16;
    default: return 0;
  }
}

int current_device() {
  int dev = -1;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= kMaxDevices) {
    (void)hipGetLastError();
    return -1;
  }
  return dev;
}

bool prepared(int type) {
  const int dev = current_device();
  return dev >= 0 && (g_prepared[dev].load(std::memory_order_acquire) & (uint32_t)type_bit(type)) != 0;
}

bool stream_is_capturing(hipStream_t st) {
  hipStreamCaptureStatus s = hipStreamCaptureStatusNone;
  const hipError_t e = hipStreamIsCapturing(st, &s);
  if (e != hipSuccess) (void)hipGetLastError();
  return e == hipSuccess && s != hipStreamCaptureStatusNone;
}

// Whether a product of rows <= matvec_max_rows() against wbytes of weight
// goes to a matrix-core kernel (mmq_takes_few_rows, cuda.rs:823-839).
bool few_rows_take(int type, int64_t rows, int64_t wbytes, hipStream_t st) {
  int64_t fewest, least;
  few_rows_line(type, fewest, least);
  if (rows < (fewest > 2 ? fewest : 2) || wbytes < least) return false;
  if (!stream_is_capturing(st)) {
    const int dev = current_device();
    const uint32_t bit = (uint32_t)type_bit(type);
    if (dev >= 0 && !(g_prepare_tried[dev].fetch_or(bit, std::memory_order_acq_rel) & bit)) (void)qmm_prepare(type);
    return true;
  }
  return mmq_policy().captured && prepared(type);
}

bool mmq_allows(int64_t rows) {
  const MmqPolicy& pol = mmq_policy();
  return pol.on && rows <= pol.max_rows;
}

// Q4_K and Q6_K at 17-128 rows and Q6_K's up to 256 that the single-pass GEMM
// does not take (gemm_kq_mid.hip): the weight cut along K.
bool mid_takes(int type, const void* w, const void* xq, int64_t n, int64_t k, int64_t rows) {
  return mmq_allows(rows) && aligned16(w) && aligned16(xq) && qmm::gemm_kq_mid_fits(type, n, k, rows);
}

// The few-row matrix-core kernels (Q4_K, Q6_K): up to
// gemm_q4k_skinny_max_rows() rows past the few-rows line that mid_takes leaves.
bool skinny_takes(int type, const void* w, const void* xq, int64_t n, int64_t k, int64_t rows, hipStream_t st) {
  if (!mmq_allows(rows) || rows > qmm::gemm_q4k_skinny_max_rows() || !aligned16(w) || !aligned16(xq)) return false;
  if (mid_takes(type, w, xq, n, k, rows)) return false;
  int64_t wbytes;
  if (type == qmm::T_Q4_K && qmm::gemm_q4k_skinny_fits(k, rows))
    wbytes = n * (k / 256) * 144;
  else if (type == qmm::T_Q6_K && qmm::gemm_q6k_skinny_fits(k, rows))
    wbytes = n * (k / 256) * 210;
  else
    return false;
  if (rows > qmm::matvec_max_rows()) return true;
  return few_rows_take(type, rows, wbytes, st);
}

hipError_t launch_skinny(int type, const qmm::MvTargets& t, int64_t k, const qmm::ActPlanes& p, int64_t rows,
                         hipStream_t st, bool exact = qmm::exact_forms()) {
  if (type == qmm::T_Q6_K) return qmm::launch_gemm_q6k_skinny(t, k, p, rows, exact, st);
  return qmm::launch_gemm_q4k_skinny(t, k, p, rows, (int)cu_count(), st);
}

// The tiled int8 matrix-core GEMMs: Q4_K and Q6_K past the skinny kernels'
// rows, Q8_0 / IQ4_NL / MXFP4 past the decode kernels' rows (or from the
// few-rows line, where SWARMLLM_QMATMUL_MMQ_MIN_ROWS moves it below); weight
// and quantized activation 16-byte aligned (their 16-byte copies), sizes
// inside their 32-bit offsets.
bool gemm_takes(int type, const void* w, const void* xq, int64_t n, int64_t k, int64_t rows, hipStream_t st) {
  if (!mmq_allows(rows) || !aligned16(w) || !aligned16(xq)) return false;
  if (type == qmm::T_Q4_K) return rows >= qmm::gemm_q4k_min_rows() && qmm::gemm_q4k_fits(n, k, rows);
  if (type == qmm::T_Q6_K) return rows >= qmm::gemm_q6k_min_rows() && qmm::gemm_q6k_fits(n, k, rows);
  if (!qmm::gemm_b32_fits(type, n, k, rows)) return false;
  if (rows > qmm::matvec_max_rows()) return true;
  return few_rows_take(type, rows, n * (k / 32) * type_size(type), st);
}

hipError_t launch_mid(int type, const qmm::MvTargets& t, int64_t k, const qmm::ActPlanes& p, int64_t rows, void* slots,
                      size_t slot_bytes, float** parts, hipStream_t st) {
  return type == qmm::T_Q6_K ? qmm::launch_gemm_q6k_mid(t, k, p, rows, slots, slot_bytes, parts, st)
                             : qmm::launch_gemm_q4k_mid(t, k, p, rows, slots, slot_bytes, parts, st);
}

// Whether a product goes to a matrix-core kernel rather than the decode kernels.
bool matrix_takes(int type, const void* w, const void* xq, int64_t n, int64_t k, int64_t rows, hipStream_t st) {
  return mid_takes(type, w, xq, n, k, rows) || gemm_takes(type, w, xq, n, k, rows, st) ||
         skinny_takes(type, w, xq, n, k, rows, st);
}

// One more weight of a launch (at most kMaxTargets).
void add_target(qmm::MvTargets& t, const void* w, int64_t n, float* dst, int64_t ldd) {
  const int i = t.count++;
  t.w[i] = w;
  t.dst[i] = dst;
  t.ldd[i] = ldd;
  t.row_end[i] = n + (i ? t.row_end[i - 1] : 0);
}

qmm::MvTargets one_target(const void* w, int64_t n, float* dst, int64_t ldd) {
  qmm::MvTargets t{};
  add_target(t, w, n, dst, ldd);
  return t;
}

// Past mid_takes' rows. Q4_K: the single-pass GEMM (256-row tiles); rows
// shorter than its k keep the exact two-pass kernel.
hipError_t launch_gemm(int type, const void* w, int64_t n, int64_t k, const qmm::ActPlanes& p, int64_t rows,
                       float* dst, int64_t ldd, hipStream_t st) {
  if (qmm::exact_forms()) {
    if (type == qmm::T_Q6_K) return qmm::launch_gemm_q6k(w, n, k, p, rows, dst, ldd, st);
    if (type == qmm::T_Q4_K) return qmm::launch_gemm_q4k(w, n, k, p, rows, dst, ldd, st);
  }
  if (type == qmm::T_Q6_K) {
    // without a workspace for K splits, the single-pass Q6_K GEMM only where
    // its tiles fill the CUs (uncut, its per-super-block work is ~1.5x the
    // exact kernel's share of a narrow product)
    if (rows >= qmm::gemm_q4k_sp_min_rows() && qmm::gemm_q6k_sp_fits(n, k, rows) &&
        qmm::gemm_q4k_sp_splits(n, k, rows, (int)cu_count()) == 1)
      return qmm::launch_gemm_q6k_sp(w, n, k, p, rows, dst, ldd, st);
    return qmm::launch_gemm_q6k(w, n, k, p, rows, dst, ldd, st);
  }
  if (type != qmm::T_Q4_K) return qmm::launch_gemm_b32(type, one_target(w, n, dst, ldd), k, p, rows, st);
  if (rows >= qmm::gemm_q4k_sp_min_rows() && qmm::gemm_q4k_sp_fits(n, k, rows))
    return qmm::launch_gemm_q4k_sp(w, n, k, p, rows, dst, ldd, st);
  return qmm::launch_gemm_q4k(w, n, k, p, rows, dst, ldd, st);
}

// Products the single-pass Q4_K GEMM takes: those it can cut along K and
// launch several of at once (launch_gemm_q4k_sp_targets).
bool sp_takes(int type, const void* w, const void* xq, int64_t n, int64_t k, int64_t rows, hipStream_t st) {
  if ((type != qmm::T_Q4_K && type != qmm::T_Q6_K) || qmm::exact_forms()) return false;
  if (!gemm_takes(type, w, xq, n, k, rows, st) || rows < qmm::gemm_q4k_sp_min_rows()) return false;
  return type == qmm::T_Q4_K ? qmm::gemm_q4k_sp_fits(n, k, rows) : qmm::gemm_q6k_sp_fits(n, k, rows);
}

hipError_t launch_sp(int type, const qmm::MvTargets& t, int64_t k, const qmm::ActPlanes& p, int64_t rows, void* ws,
                     size_t ws_bytes, hipStream_t st) {
  return type == qmm::T_Q6_K ? qmm::launch_gemm_q6k_sp_targets(t, k, p, rows, ws, ws_bytes, (int)cu_count(), st)
                             : qmm::launch_gemm_q4k_sp_targets(t, k, p, rows, ws, ws_bytes, (int)cu_count(), st);
}

// Weights i0 .. of a shared product, at most kMaxTargets.
qmm::MvTargets targets_of(const void* const* w, const int64_t* n, float* const* dst, const int64_t* ldd, int i0,
                          int count) {
  qmm::MvTargets t{};
  for (int i = i0; i < count && t.count < qmm::kMaxTargets; i++) add_target(t, w[i], n[i], dst[i], ldd[i]);
  return t;
}

// The streaming decode kernels (Q4_K, Q6_K at 1-2 activation rows).
bool stream_supported(int type, int64_t k, int64_t rows) {
  if (qmm::mv_b32_rows_supported(type, k, rows)) return true;
  if (type == qmm::T_Q4_K) return qmm::mv_q4k_rows_supported(k, rows);
  if (type == qmm::T_Q6_K) return qmm::mv_q6k_rows_supported(k, rows);
  return false;
}

// Whether the streaming kernel is the one for an activation whose planes are
// made. A lane of it holds its part of a weight row and of the activation in
// registers, which for Q4_K at 2 rows of more than 4096 values and 1 of more
// than 8192 do not fit (up to 187 are spilled); the multi-row kernel reads the
// planes from the caches (with their own launch: 1 row, 8192 x 11008 53 -> 15
// us, 8192 x 16384 57 -> 20; 2 rows, 28672 x 8192 78 -> 36, 14336 x 5120 43
// -> 19, 128 x 8192 12 -> 8).
bool stream_from_planes(int type, int64_t k, int64_t rows) {
  return stream_supported(type, k, rows) && (type != qmm::T_Q4_K || k <= (rows == 1 ? 8192 : 4096));
}

// Whether it also takes, quantizing the activation itself, these `count`
// weights of n_total rows together. Where the multi-row kernel is faster, the
// quantizer's launch and one a weight still cost the host 3.5 us each past
// the first (a forward of one launch 14 us), so the streaming kernel keeps what it
// does in under about 17 us: 1 row while a wave has one weight row (4096 x
// 14336 17 us), 2 rows up to 3072 weight rows, and 2560 more for each further
// weight. Without room for the planes it takes all that it supports.
bool stream_takes(int type, int64_t k, int64_t n_total, int count, int64_t rows) {
  return stream_from_planes(type, k, rows) ||
         (stream_supported(type, k, rows) &&
          n_total <= (int64_t)cu_count() * ((rows == 1 ? 16 : 12) + 10 * (count - 1)));
}

// The same of the launch that also applies the GLU, at 2 rows of more than
// 4096 values, against the two products and the GLU in launches of their own
// (4352 x 4352 78 -> 23 us, 13824 x 5120 157 -> 37, 28672 x 8192 287 -> 69;
// four launches cost the host about 24 us).
bool stream_glu_takes(int64_t k, int64_t n, int64_t rows) {
  return rows == 1 || k <= 4096 || n <= (int64_t)cu_count() * 6;
}

// Launch shape of the Q4_K decode kernel for n_total weight rows, in 16-wave
// workgroups (one activation fill per 16 waves): a row per wave up to 16
// waves a CU; beyond that, about 1.5 rows per wave up to 32 waves a CU, the
// next row's loads in flight whenever a wave has more than one row.
qmm::MvShape stream_shape(int64_t n_total, int64_t k) {
  const int64_t cus = cu_count();
  // a row per wave while the rows fit one 16-wave workgroup a CU (o, 4096
  // rows: 5.5 us against 6.2 us for 2736 waves with the next row in flight)
  if (n_total <= cus * 16) return qmm::MvShape{(n_total + 15) / 16 * 16, 16, false};
  // Rows of more than 4096 values hold twice the registers: one 16-wave
  // workgroup a CU is resident, so the grid is one round of cus * 16 waves
  // with the rows spread over it (8192 rows of 8192: two a wave; 5472 waves
  // ran as 256 workgroups and then 86 on a third of the GPU).
  if (k > 4096) return qmm::MvShape{cus * 16, 16, true};
  int64_t waves = n_total * 2 / 3;
  if (waves < 1024) waves = 1024;
  if (waves > cus * 32) waves = cus * 32;
  waves = (waves + 15) / 16 * 16;
  return qmm::MvShape{waves, 16, n_total > waves};
}

// One streaming launch over up to kMaxTargets weights.
hipError_t launch_stream_targets(int type, int count, const void* const* w, const int64_t* n, float* const* dst,
                                 const int64_t* ldd, int64_t k, int64_t rows, const float* x, int64_t x_stride,
                                 const qmm::ActPlanes* pre, hipStream_t st) {
  qmm::MvTargets t{};
  int64_t end = 0;
  for (int i = 0; i < count; i++) {
    t.w[i] = w[i];
    t.dst[i] = dst[i];
    t.ldd[i] = ldd[i];
    end += n[i];
    t.row_end[i] = end;
  }
  t.count = count;
  if (type == qmm::T_Q6_K) return qmm::launch_mv_q6k_rows(t, k, rows, x, x_stride, pre, q8k_scale(), (int)cu_count(), st);
  if (type != qmm::T_Q4_K) return qmm::launch_mv_b32_rows(type, t, k, rows, x, x_stride, pre, (int)cu_count(), st);
  return qmm::launch_mv_q4k_rows(t, k, rows, x, x_stride, pre, q8k_scale(), stream_shape(end, k), st);
}

}  // namespace

namespace qmm {
bool exact_forms() {
  static const bool on = env_is_on(std::getenv("SWARMLLM_QMATMUL_EXACT"));
  return on;
}

namespace {
std::atomic<const char*> g_last_kernel{""};

// The kernels that may ask for more than 64 KiB of LDS (registered as the
// library loads) and the (device, kernel) pairs whose limit is raised.
std::mutex& lds_mu() {
  static std::mutex m;
  return m;
}
std::vector<const void*>& lds_kernels() {
  static std::vector<const void*> v;
  return v;
}
std::set<std::pair<int, const void*>>& lds_raised() {
  static std::set<std::pair<int, const void*>> s;
  return s;
}
}  // namespace
void note_launch(const char* what) { g_last_kernel.store(what, std::memory_order_relaxed); }

bool big_lds_register(const void* fn) {
  std::lock_guard<std::mutex> lock(lds_mu());
  lds_kernels().push_back(fn);
  return true;
}

hipError_t raise_lds_limit(const void* fn) {
  int dev = -1;
  const hipError_t g = hipGetDevice(&dev);
  if (g != hipSuccess) return g;
  std::lock_guard<std::mutex> lock(lds_mu());
  if (lds_raised().count({dev, fn})) return hipSuccess;
  const hipError_t e = hipFuncSetAttribute(fn, hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024);
  if (e == hipSuccess) lds_raised().insert({dev, fn});
  return e;
}

hipError_t raise_all_lds_limits() {
  std::vector<const void*> all;
  {
    std::lock_guard<std::mutex> lock(lds_mu());
    all = lds_kernels();
  }
  for (const void* fn : all) {
    const hipError_t e = raise_lds_limit(fn);
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}
}  // namespace qmm

extern "C" {

const char* qmm_last_kernel(void) { return qmm::g_last_kernel.load(std::memory_order_relaxed); }

int qmm_available(void) {
  static std::mutex mu;
  static int cached[64];
  static bool known[64];
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) {
    (void)hipGetLastError();
    return 0;
  }
  std::lock_guard<std::mutex> lock(mu);
  if (!known[dev]) {
    hipDeviceProp_t prop;
    int ok = 0;
    if (hipGetDeviceProperties(&prop, dev) == hipSuccess) ok = std::strncmp(prop.gcnArchName, "gfx950", 6) == 0;
    (void)hipGetLastError();
    cached[dev] = ok;
    known[dev] = true;
  }
  return cached[dev];
}

int qmm_prepare(int type) {
  const uint32_t bit = (uint32_t)type_bit(type);
  if (!bit) return QMM_UNSUPPORTED;
  const int dev = current_device();
  if (dev < 0) return QMM_DEVICE_ERROR;
  if (!qmm_available()) return QMM_NO_TILE;
  (void)cu_count();
  (void)mmq_policy();
  const bool scratch = qmm::noalloc_prepare();
  const hipError_t e = qmm::raise_all_lds_limits();
  (void)hipGetLastError();  // not sticky: leave nothing for a later check to read
  if (!scratch || e != hipSuccess) return QMM_DEVICE_ERROR;
  g_prepared[dev].fetch_or(bit, std::memory_order_acq_rel);
  return QMM_OK;
}

int qmm_prepared(int type) { return prepared(type) ? 1 : 0; }

// Every product here sums in int32 / f32 (no f16 accumulator to widen).
int qmm_accumulate_in_f32(int type) { return type_bit(type) ? QMM_OK : QMM_UNSUPPORTED; }

int qmm_block_size(int type) { return block_size(type); }

size_t qmm_type_bytes(int type, int64_t nelem) {
  const int qk = block_size(type);
  if (qk == 0 || nelem < 0 || nelem % qk) return 0;
  return (size_t)(nelem / qk) * (size_t)type_size(type);
}

int qmm_act_layout(int type, int64_t rows) {
  (void)rows;
  switch (type) {
    case qmm::T_Q4_K: case qmm::T_Q6_K: return QMM_ACT_Q8K;
    case qmm::T_Q8_0: case qmm::T_IQ4_NL: case qmm::T_MXFP4: return QMM_ACT_Q8_0;
    default: return -1;
  }
}

size_t qmm_act_bytes(int layout, int64_t k, int64_t rows) {
  if ((layout != QMM_ACT_Q8K && layout != QMM_ACT_Q8_0) || k <= 0 || rows <= 0) return 0;
  if (k % (layout == QMM_ACT_Q8K ? 256 : 32)) return 0;
  return qmm::act_bytes(layout, k, rows);
}

int qmm_act_planes(int layout, int64_t k, int64_t rows, size_t* codes_off, size_t* scales_off, size_t* sums_off) {
  if (qmm_act_bytes(layout, k, rows) == 0) return QMM_UNSUPPORTED;
  size_t so = 0, uo = 0;
  qmm::act_plane_offsets(layout, k, rows, &so, &uo);
  if (codes_off) *codes_off = 0;
  if (scales_off) *scales_off = so;
  if (sums_off) *sums_off = uo;
  return QMM_OK;
}

int qmm_quantize_act(const float* x, void* xq, int layout, int64_t k, int64_t rows, int64_t stride, int64_t stream) {
  if (qmm_act_bytes(layout, k, rows) == 0 || stride < k || x == nullptr || xq == nullptr) return QMM_UNSUPPORTED;
  clear_stale_error();
  return status_of(qmm::launch_act_quantize(layout, x, stride, k, rows, xq, q8k_scale(), (hipStream_t)stream));
}

int qmm_dequantize_act(const void* xq, int layout, void* out, int out_dtype, int64_t k, int64_t rows, int64_t stream) {
  if (qmm_act_bytes(layout, k, rows) == 0 || !qmm::value_type_ok(out_dtype) || xq == nullptr || !aligned16(xq) ||
      out == nullptr)
    return QMM_UNSUPPORTED;
  clear_stale_error();
  return status_of(qmm::launch_dequantize_act(xq, layout, out, out_dtype, k, rows, (hipStream_t)stream));
}

int qmm_rms_norm_act(const void* x, int dtype, int64_t x_stride, const void* residual, int64_t r_stride, const float* w,
                     float eps, void* h, int64_t h_stride, void* xq, int layout, void* y, int y_dtype,
                     int64_t y_stride, int64_t k, int64_t rows, int64_t stream) {
  if (!x || !w || !(xq || y) || !qmm::value_type_ok(dtype) || k < 1 || k > (int64_t)1 << 30 || rows < 1 ||
      x_stride < k || (residual && r_stride < k) || (h && h_stride < k) || !(eps >= 0.0f))
    return QMM_UNSUPPORTED;
  if (xq && (qmm_act_bytes(layout, k, rows) == 0 || !aligned16(xq))) return QMM_UNSUPPORTED;
  if (k % 4 != 0 || (y && (!qmm::value_type_ok(y_dtype) || y_stride < k))) return QMM_UNSUPPORTED;
  clear_stale_error();
  return status_of(qmm::launch_rms_norm_act(x, dtype, x_stride, residual, r_stride, w, eps, h, h_stride, xq, layout, y,
                                            y_dtype, y_stride, k, rows, q8k_scale(), (hipStream_t)stream));
}

int qmm_matvec_max_rows(void) { return qmm::matvec_max_rows(); }

void qmm_set_force_dmmv(int on) { g_force_dmmv.store(on != 0, std::memory_order_relaxed); }
int qmm_force_dmmv(void) { return g_force_dmmv.load(std::memory_order_relaxed) ? 1 : 0; }

int qmm_mmq_few_rows_line(int type, int64_t* rows, int64_t* bytes) {
  if (block_size(type) == 0 || !rows || !bytes) return QMM_UNSUPPORTED;
  few_rows_line(type, *rows, *bytes);
  return QMM_OK;
}

int64_t qmm_mmq_max_rows(void) {
  const MmqPolicy& pol = mmq_policy();
  return pol.on ? pol.max_rows : 0;
}

int qmm_mmq_captured(void) { return mmq_policy().captured ? 1 : 0; }

int qmm_exact_forms(void) { return qmm::exact_forms() ? 1 : 0; }

int qmm_matvec(int type, const void* w, const void* xq, float* dst, int64_t ldd, int64_t k, int64_t n, int64_t rows,
               int64_t stream) {
  if (!shape_ok(type, k, n, rows) || rows > qmm::matvec_max_rows() || ldd < n || !w || !xq || !dst)
    return QMM_UNSUPPORTED;
  const int layout = qmm_act_layout(type, rows);
  const qmm::ActPlanes p = qmm::act_planes(layout, (void*)xq, k, rows);
  clear_stale_error();
  hipError_t e;
  if (stream_from_planes(type, k, rows))
    e = launch_stream_targets(type, 1, &w, &n, &dst, &ldd, k, rows, nullptr, 0, &p, (hipStream_t)stream);
  else
    e = qmm::launch_matvec(type, w, n, k, p, rows, dst, ldd, (hipStream_t)stream);
  if (e == hipSuccess) g_matvec_launches.fetch_add(1, std::memory_order_relaxed);
  return status_of(e);
}

// A product of the short-batch kernel with no room for its split slots
// (qmm_matmul has none). A workgroup of it then walks a tile's whole K, which
// takes 1.2 to 1.7 us a super-block, so where that leaves CUs idle the kernels
// without slots take the product, as exactly: Q6_K past 32 rows the tiled GEMM,
// otherwise the few-row kernel, 32 rows a launch, while the launches times their
// rounds of the CUs (one per 4096 weight rows) are few. Uncut / here, us: Q4_K
// 4096 x 14336 at 24 rows 99 / 20, 4096 x 4096 at 64 71 / 19, 8192 x 8192 at 96
// 98 / 70; Q6_K 4096 x 14336 at 24 rows 135 / 34, 4096 x 4096 at 64 82 / 35;
// but Q4_K 14336 x 4096 at 64 39 / 50, Q6_K at 24 40 / 49.
int launch_mid_without_slots(int type, const void* w, int64_t n, int64_t k, const qmm::ActPlanes& p, int layout,
                             int64_t rows, float* dst, int64_t ldd, hipStream_t st) {
  if (qmm::gemm_kq_mid_splits(n, k, rows) > 1) {
    if (type == qmm::T_Q6_K && rows >= qmm::gemm_q6k_min_rows() && qmm::gemm_q6k_fits(n, k, rows)) {
      if (qmm::launch_gemm_q6k(w, n, k, p, rows, dst, ldd, st) != hipSuccess) return QMM_DEVICE_ERROR;
      g_gemm_launches.fetch_add(1, std::memory_order_relaxed);
      return QMM_OK;
    }
    const int64_t step = qmm::gemm_q4k_skinny_max_rows();
    if ((rows + step - 1) / step * ((n + 4095) / 4096) <= (type == qmm::T_Q6_K ? 3 : 6)) {
      for (int64_t r0 = 0; r0 < rows; r0 += step) {
        const int64_t nr = rows - r0 < step ? rows - r0 : step;
        if (launch_skinny(type, one_target(w, n, dst + r0 * ldd, ldd), k, qmm::act_rows(layout, p, k, r0), nr, st,
                          true) != hipSuccess)
          return QMM_DEVICE_ERROR;
        g_gemm_launches.fetch_add(1, std::memory_order_relaxed);
      }
      return QMM_OK;
    }
  }
  if (launch_mid(type, one_target(w, n, dst, ldd), k, p, rows, nullptr, 0, nullptr, st) != hipSuccess)
    return QMM_DEVICE_ERROR;
  g_gemm_launches.fetch_add(1, std::memory_order_relaxed);
  return QMM_OK;
}

// One product from an activation already quantized into planes p (buffer
// xq): the matrix-core kernels past the few-rows line, else the decode
// kernels a chunk of at most matvec_max_rows() rows at a time.
int launch_product(int type, const void* w, int64_t n, int64_t k, const void* xq, const qmm::ActPlanes& p,
                   int layout, int64_t rows, float* dst, int64_t ldd, hipStream_t st) {
  if (mid_takes(type, w, xq, n, k, rows))
    return launch_mid_without_slots(type, w, n, k, p, layout, rows, dst, ldd, st);
  if (gemm_takes(type, w, xq, n, k, rows, st)) {
    if (launch_gemm(type, w, n, k, p, rows, dst, ldd, st) != hipSuccess) return QMM_DEVICE_ERROR;
    g_gemm_launches.fetch_add(1, std::memory_order_relaxed);
    return QMM_OK;
  }
  if (skinny_takes(type, w, xq, n, k, rows, st)) {
    if (launch_skinny(type, one_target(w, n, dst, ldd), k, p, rows, st) != hipSuccess) return QMM_DEVICE_ERROR;
    g_gemm_launches.fetch_add(1, std::memory_order_relaxed);
    return QMM_OK;
  }
  const int64_t step = qmm::matvec_max_rows();
  for (int64_t r0 = 0; r0 < rows; r0 += step) {
    const int64_t nr = rows - r0 < step ? rows - r0 : step;
    const qmm::ActPlanes pr = qmm::act_rows(layout, p, k, r0);
    float* d = dst + r0 * ldd;
    const hipError_t e = stream_from_planes(type, k, nr)
                             ? launch_stream_targets(type, 1, &w, &n, &d, &ldd, k, nr, nullptr, 0, &pr, st)
                             : qmm::launch_matvec(type, w, n, k, pr, nr, d, ldd, st);
    if (e != hipSuccess) return QMM_DEVICE_ERROR;
    g_matvec_launches.fetch_add(1, std::memory_order_relaxed);
  }
  return QMM_OK;
}

int qmm_matmul(int type, const void* w, const void* xq, float* dst, int64_t ldd, int64_t k, int64_t n, int64_t rows,
               int64_t stream) {
  if (!shape_ok(type, k, n, rows) || ldd < n || !w || !xq || !dst) return QMM_UNSUPPORTED;
  const int layout = qmm_act_layout(type, rows);
  const qmm::ActPlanes p = qmm::act_planes(layout, (void*)xq, k, rows);
  clear_stale_error();
  return launch_product(type, w, n, k, xq, p, layout, rows, dst, ldd, (hipStream_t)stream);
}

// qmm_forward (pre false: from the f32 activation x, quantized into the
// workspace) and qmm_forward_act (pre: from the planes at xq, the workspace
// holding a K split's slots only).
static int forward_impl(int type, const void* w, bool pre, const void* xq, const float* x, int64_t x_stride, float* dst,
                        int64_t ldd, void* workspace, size_t workspace_bytes, size_t* need, int64_t k, int64_t n,
                        int64_t rows, int launch, int64_t stream) {
  if (!shape_ok(type, k, n, rows) || need == nullptr || ldd < n || (pre ? !aligned16(xq) || !aligned16(workspace) : x_stride < k))
    return QMM_UNSUPPORTED;
  const int layout = qmm_act_layout(type, rows);
  const size_t bytes = pre ? 0 : qmm::act_bytes(layout, k, rows);
  const void* acts = pre ? xq : workspace;
  const hipStream_t st = (hipStream_t)stream;
  // a single-pass GEMM that leaves CUs idle is cut along K when the
  // workspace also holds its split slots (need reports them; with only the
  // activation's bytes it runs uncut)
  const bool mid = mid_takes(type, w, acts, n, k, rows);
  const size_t split = mid ? qmm::gemm_kq_mid_slot_bytes(one_target(w, n, dst, ldd), k, rows, false)
                       : sp_takes(type, w, acts, n, k, rows, st)
                           ? qmm::gemm_q4k_sp_split_bytes(one_target(w, n, dst, ldd), k, rows, (int)cu_count())
                           : 0;
  *need = split ? qmm::align_up(bytes, 256) + split : bytes;
  if (!launch) return QMM_OK;
  if (g_fail_next.exchange(false)) return QMM_NO_ROOM;
  if (!pre && (workspace_bytes < bytes || workspace == nullptr)) return QMM_WORKSPACE_TOO_SMALL;
  if (!w || !(pre ? xq : x) || !dst) return QMM_UNSUPPORTED;
  if (workspace == nullptr) workspace_bytes = 0;
  clear_stale_error();
  if (!pre && g_force_dmmv.load(std::memory_order_relaxed))
    return status_of(qmm::launch_dmmv(type, w, n, k, x, x_stride, rows, dst, ldd, st));
  if (!pre && stream_takes(type, k, n, 1, rows) && qmm::mv_q4k_rows_fusable(x, x_stride) &&
      !matrix_takes(type, w, acts, n, k, rows, st)) {
    // the activation is quantized inside the product's own launch
    const hipError_t e = launch_stream_targets(type, 1, &w, &n, &dst, &ldd, k, rows, x, x_stride, nullptr, st);
    if (e != hipSuccess) return QMM_DEVICE_ERROR;
    g_matvec_launches.fetch_add(1, std::memory_order_relaxed);
    return QMM_OK;
  }
  if (!pre && qmm::launch_act_quantize(layout, x, x_stride, k, rows, workspace, q8k_scale(), st) != hipSuccess)
    return QMM_DEVICE_ERROR;
  const qmm::ActPlanes p = qmm::act_planes(layout, (void*)acts, k, rows);
  if (mid && split && workspace_bytes >= *need) {
    if (launch_mid(type, one_target(w, n, dst, ldd), k, p, rows, (char*)workspace + qmm::align_up(bytes, 256), split,
                   nullptr, st) != hipSuccess)
      return QMM_DEVICE_ERROR;
    g_gemm_launches.fetch_add(1, std::memory_order_relaxed);
    return QMM_OK;
  }
  // Q6_K takes the single-pass GEMM only cut as planned (uncut, a narrow
  // product runs faster on the exact kernel)
  if (!mid && sp_takes(type, w, acts, n, k, rows, st) &&
      (type == qmm::T_Q4_K || split == 0 || workspace_bytes >= *need)) {
    const size_t off = qmm::align_up(bytes, 256);
    void* sws = workspace_bytes > off ? (char*)workspace + off : nullptr;
    if (launch_sp(type, one_target(w, n, dst, ldd), k, p, rows, sws, workspace_bytes > off ? workspace_bytes - off : 0,
                  st) != hipSuccess)
      return QMM_DEVICE_ERROR;
    g_gemm_launches.fetch_add(1, std::memory_order_relaxed);
    return QMM_OK;
  }
  return launch_product(type, w, n, k, acts, p, layout, rows, dst, ldd, st);
}

int qmm_forward(int type, const void* w, const float* x, int64_t x_stride, float* dst, int64_t ldd, void* workspace,
                size_t workspace_bytes, size_t* need, int64_t k, int64_t n, int64_t rows, int launch, int64_t stream) {
  return forward_impl(type, w, false, nullptr, x, x_stride, dst, ldd, workspace, workspace_bytes, need, k, n, rows,
                      launch, stream);
}

int qmm_forward_act(int type, const void* w, const void* xq, float* dst, int64_t ldd, void* workspace,
                    size_t workspace_bytes, size_t* need, int64_t k, int64_t n, int64_t rows, int launch,
                    int64_t stream) {
  return forward_impl(type, w, true, xq, nullptr, 0, dst, ldd, workspace, workspace_bytes, need, k, n, rows, launch,
                      stream);
}

// qmm_forward_shared and qmm_forward_shared_act, as forward_impl.
static int shared_impl(int type, int count, const void* const* w, const int64_t* n, float* const* dst,
                       const int64_t* ldd, bool pre, const void* xq, const float* x, int64_t x_stride, void* workspace,
                       size_t workspace_bytes, size_t* need, int64_t k, int64_t rows, int launch, int64_t stream) {
  if (count < 1 || !w || !n || !dst || !ldd || need == nullptr || (pre ? !aligned16(xq) || !aligned16(workspace) : x_stride < k))
    return QMM_UNSUPPORTED;
  for (int i = 0; i < count; i++)
    if (!shape_ok(type, k, n[i], rows) || ldd[i] < n[i]) return QMM_UNSUPPORTED;
  const int layout = qmm_act_layout(type, rows);
  const size_t bytes = pre ? 0 : qmm::act_bytes(layout, k, rows);
  const void* acts = pre ? xq : workspace;
  const hipStream_t st = (hipStream_t)stream;
  // the short-batch kernel's weights share its launches, kMaxTargets each, and
  // so do those of the single-pass GEMM; their split slots follow the
  // activation (one launch's worth, reused launch after launch)
  auto mid_i = [&](int i) { return mid_takes(type, w[i], acts, n[i], k, rows); };
  auto sp_i = [&](int i) { return !mid_i(i) && sp_takes(type, w[i], acts, n[i], k, rows, st); };
  size_t split = 0;
  qmm::MvTargets midg{}, spg{};
  for (int i = 0; i <= count; i++) {
    if (i < count && mid_i(i))
      add_target(midg, w[i], n[i], dst[i], ldd[i]);
    else if (i < count && sp_i(i))
      add_target(spg, w[i], n[i], dst[i], ldd[i]);
    if (midg.count == qmm::kMaxTargets || (i == count && midg.count > 0)) {
      const size_t b = qmm::gemm_kq_mid_slot_bytes(midg, k, rows, false);
      split = b > split ? b : split;
      midg = qmm::MvTargets{};
    }
    if (spg.count == qmm::kMaxTargets || (i == count && spg.count > 0)) {
      const size_t b = qmm::gemm_q4k_sp_split_bytes(spg, k, rows, (int)cu_count());
      split = b > split ? b : split;
      spg = qmm::MvTargets{};
    }
  }
  *need = split ? qmm::align_up(bytes, 256) + split : bytes;
  if (!launch) return QMM_OK;
  if (g_fail_next.exchange(false)) return QMM_NO_ROOM;
  if (!(pre ? xq : x)) return QMM_UNSUPPORTED;
  for (int i = 0; i < count; i++)
    if (!w[i] || !dst[i]) return QMM_UNSUPPORTED;
  clear_stale_error();
  if (workspace == nullptr) workspace_bytes = 0;
  if (!pre && g_force_dmmv.load(std::memory_order_relaxed)) {
    for (int i = 0; i < count; i++)
      if (qmm::launch_dmmv(type, w[i], n[i], k, x, x_stride, rows, dst[i], ldd[i], st) != hipSuccess)
        return QMM_DEVICE_ERROR;
    return QMM_OK;
  }
  int64_t n_total = 0;
  for (int i = 0; i < count; i++) n_total += n[i];
  const bool room = workspace != nullptr && workspace_bytes >= bytes;
  bool fused = pre ? stream_from_planes(type, k, rows)
                   : (room ? stream_takes(type, k, n_total, count, rows) : stream_supported(type, k, rows)) &&
                         qmm::mv_q4k_rows_fusable(x, x_stride);
  for (int i = 0; fused && i < count; i++) fused = !matrix_takes(type, w[i], acts, n[i], k, rows, st);
  const qmm::ActPlanes p = acts ? qmm::act_planes(layout, (void*)acts, k, rows) : qmm::ActPlanes{};
  if (fused) {
    // one launch per kMaxTargets weights, each quantizing the activation in LDS (or reading its planes)
    for (int i0 = 0; i0 < count; i0 += qmm::kMaxTargets) {
      const int c = count - i0 < qmm::kMaxTargets ? count - i0 : qmm::kMaxTargets;
      if (launch_stream_targets(type, c, w + i0, n + i0, dst + i0, ldd + i0, k, rows, x, x_stride,
                                pre ? &p : nullptr, st) != hipSuccess)
        return QMM_DEVICE_ERROR;
      g_matvec_launches.fetch_add(1, std::memory_order_relaxed);
    }
    return QMM_OK;
  }
  // otherwise: the activation quantized once into the workspace, then each product
  if (!pre && (workspace_bytes < bytes || workspace == nullptr)) return QMM_WORKSPACE_TOO_SMALL;
  if (!pre && qmm::launch_act_quantize(layout, x, x_stride, k, rows, workspace, q8k_scale(), st) != hipSuccess)
    return QMM_DEVICE_ERROR;
  if (!is_kquant(type)) {
    bool gemm = true;
    for (int i = 0; i < count; i++) gemm = gemm && gemm_takes(type, w[i], acts, n[i], k, rows, st);
    if (gemm) {
      for (int i0 = 0; i0 < count; i0 += qmm::kMaxTargets) {
        if (qmm::launch_gemm_b32(type, targets_of(w, n, dst, ldd, i0, count), k, p, rows, st) != hipSuccess)
          return QMM_DEVICE_ERROR;
        g_gemm_launches.fetch_add(1, std::memory_order_relaxed);
      }
      return QMM_OK;
    }
  }
  // the weights each of the short-batch, single-pass and few-row kernels takes
  // share its launches
  qmm::MvTargets grp{};
  const size_t off = qmm::align_up(bytes, 256);
  void* sws = workspace_bytes > off ? (char*)workspace + off : nullptr;
  const size_t sbytes = workspace_bytes > off ? workspace_bytes - off : 0;
  auto flush = [&](qmm::MvTargets& t, auto&& launch_group) -> bool {
    if (t.count == 0) return true;
    if (launch_group(t) != hipSuccess) return false;
    g_gemm_launches.fetch_add(1, std::memory_order_relaxed);
    t = qmm::MvTargets{};
    return true;
  };
  auto mid_group = [&](const qmm::MvTargets& t) {
    return launch_mid(type, t, k, p, rows, split ? sws : nullptr, split ? sbytes : 0, nullptr, st);
  };
  auto sp_group = [&](const qmm::MvTargets& t) { return launch_sp(type, t, k, p, rows, sws, sbytes, st); };
  auto few_group = [&](const qmm::MvTargets& t) { return launch_skinny(type, t, k, p, rows, st); };
  const bool room_split = split == 0 || workspace_bytes >= *need;
  for (int i = 0; i < count; i++) {
    const bool mid = mid_i(i);
    if (mid && room_split) {
      add_target(midg, w[i], n[i], dst[i], ldd[i]);
      if (midg.count == qmm::kMaxTargets && !flush(midg, mid_group)) return QMM_DEVICE_ERROR;
    } else if (!mid && (type == qmm::T_Q4_K || room_split) && sp_i(i)) {
      add_target(spg, w[i], n[i], dst[i], ldd[i]);
      if (spg.count == qmm::kMaxTargets && !flush(spg, sp_group)) return QMM_DEVICE_ERROR;
    } else if (!mid && !gemm_takes(type, w[i], acts, n[i], k, rows, st) &&
               skinny_takes(type, w[i], acts, n[i], k, rows, st)) {
      add_target(grp, w[i], n[i], dst[i], ldd[i]);
      if (grp.count == qmm::kMaxTargets && !flush(grp, few_group)) return QMM_DEVICE_ERROR;
    } else {
      const int r = launch_product(type, w[i], n[i], k, acts, p, layout, rows, dst[i], ldd[i], st);
      if (r != QMM_OK) return r;
    }
  }
  return flush(midg, mid_group) && flush(spg, sp_group) && flush(grp, few_group) ? QMM_OK : QMM_DEVICE_ERROR;
}

int qmm_forward_shared(int type, int count, const void* const* w, const int64_t* n, float* const* dst,
                       const int64_t* ldd, const float* x, int64_t x_stride, void* workspace, size_t workspace_bytes,
                       size_t* need, int64_t k, int64_t rows, int launch, int64_t stream) {
  return shared_impl(type, count, w, n, dst, ldd, false, nullptr, x, x_stride, workspace, workspace_bytes, need, k,
                     rows, launch, stream);
}

int qmm_forward_shared_act(int type, int count, const void* const* w, const int64_t* n, float* const* dst,
                           const int64_t* ldd, const void* xq, void* workspace, size_t workspace_bytes, size_t* need,
                           int64_t k, int64_t rows, int launch, int64_t stream) {
  return shared_impl(type, count, w, n, dst, ldd, true, xq, nullptr, 0, workspace, workspace_bytes, need, k, rows,
                     launch, stream);
}

// qmm_forward_glu and qmm_forward_glu_act, as forward_impl.
static int glu_impl(int type, int act, const void* w_gate, const void* w_up, bool pre, const void* xq, const float* x,
                    int64_t x_stride, float* dst, int64_t ldd, void* workspace, size_t workspace_bytes, size_t* need,
                    int64_t k, int64_t n, int64_t rows, int launch, int64_t stream) {
  if (!shape_ok(type, k, n, rows) || act < QMM_GLU_SILU || act > QMM_GLU_GELU || need == nullptr || ldd < n ||
      (pre ? !aligned16(xq) || !aligned16(workspace) : x_stride < k))
    return QMM_UNSUPPORTED;
  // workspace: the quantized activation, then the gate and up products of
  // the two-launch form
  const int layout = qmm_act_layout(type, rows);
  const size_t abytes = pre ? 0 : qmm::act_bytes(layout, k, rows);
  const void* acts = pre ? xq : workspace;
  const bool dmmv = !pre && g_force_dmmv.load(std::memory_order_relaxed);
  const size_t obytes = qmm::align_up((size_t)(rows * n) * 4, 256);
  const size_t bytes = abytes + 2 * obytes;
  // in the short-batch kernel's range the GLU adds the products' K-split slots itself, when the
  // workspace holds them
  const bool mid = mid_takes(type, w_gate, acts, n, k, rows) && mid_takes(type, w_up, acts, n, k, rows);
  const void* w[2] = {w_gate, w_up};
  const int64_t ns[2] = {n, n};
  float* none[2] = {nullptr, nullptr};
  const size_t aoff = qmm::align_up(abytes, 256);
  const size_t slots = mid ? qmm::gemm_kq_mid_slot_bytes(targets_of(w, ns, none, ns, 0, 2), k, rows, true) : 0;
  *need = aoff + slots > bytes ? aoff + slots : bytes;
  if (!launch) return QMM_OK;
  if (g_fail_next.exchange(false)) return QMM_NO_ROOM;
  if (!w_gate || !w_up || !(pre ? xq : x) || !dst) return QMM_UNSUPPORTED;
  const hipStream_t st = (hipStream_t)stream;
  clear_stale_error();
  const qmm::ActPlanes p = acts ? qmm::act_planes(layout, (void*)acts, k, rows) : qmm::ActPlanes{};
  if (type == qmm::T_Q4_K && !dmmv && qmm::mv_q4k_glu_supported(k, rows) &&
      (pre ? stream_from_planes(type, k, rows)
           : (stream_glu_takes(k, n, rows) || workspace == nullptr || workspace_bytes < bytes) &&
                 qmm::mv_q4k_rows_fusable(x, x_stride)) &&
      !matrix_takes(type, w_gate, acts, n, k, rows, st) && !matrix_takes(type, w_up, acts, n, k, rows, st)) {
    if (qmm::launch_mv_q4k_glu(act, w_gate, w_up, n, k, rows, x, x_stride, pre ? &p : nullptr,
                               q8k_scale(), dst, ldd, cu_count(), st) != hipSuccess)
      return QMM_DEVICE_ERROR;
    g_matvec_launches.fetch_add(1, std::memory_order_relaxed);
    return QMM_OK;
  }
  if (workspace_bytes < bytes || workspace == nullptr) return QMM_WORKSPACE_TOO_SMALL;
  if (mid && workspace_bytes >= aoff + slots && !dmmv) {
    if (!pre && qmm::launch_act_quantize(layout, x, x_stride, k, rows, workspace, q8k_scale(), st) != hipSuccess)
      return QMM_DEVICE_ERROR;
    float* parts[2];
    if (launch_mid(type, targets_of(w, ns, none, ns, 0, 2), k, p, rows, (char*)workspace + aoff, slots, parts, st) !=
        hipSuccess)
      return QMM_DEVICE_ERROR;
    g_gemm_launches.fetch_add(1, std::memory_order_relaxed);
    return status_of(qmm::launch_glu(act, parts[0], parts[1], qmm::gemm_kq_mid_splits(n, k, rows), dst, ldd, n, rows,
                                     st));
  }
  // the single-pass GEMM, neither weight cut (together they have twice a
  // weight's tiles): gate, up and the GLU in one launch
  if (type == qmm::T_Q4_K && !dmmv &&
      sp_takes(type, w_gate, acts, n, k, rows, st) && sp_takes(type, w_up, acts, n, k, rows, st)) {
    if (!pre && qmm::launch_act_quantize(layout, x, x_stride, k, rows, workspace, q8k_scale(), st) != hipSuccess)
      return QMM_DEVICE_ERROR;
    if (qmm::launch_gemm_q4k_sp_glu(act, w_gate, w_up, n, k, p, rows, dst, ldd, st) != hipSuccess)
      return QMM_DEVICE_ERROR;
    g_gemm_launches.fetch_add(1, std::memory_order_relaxed);
    return QMM_OK;
  }
  float* gbuf = (float*)((char*)workspace + abytes);
  float* ubuf = (float*)((char*)gbuf + obytes);
  float* outs[2] = {gbuf, ubuf};
  size_t need2 = 0;
  const int r = shared_impl(type, 2, w, ns, outs, ns, pre, xq, x, x_stride, workspace, abytes, &need2, k, rows, 1,
                            stream);
  if (r != QMM_OK) return r;
  return status_of(qmm::launch_glu(act, gbuf, n, ubuf, n, dst, ldd, n, rows, st));
}

int qmm_forward_glu(int type, int act, const void* w_gate, const void* w_up, const float* x, int64_t x_stride,
                    float* dst, int64_t ldd, void* workspace, size_t workspace_bytes, size_t* need, int64_t k,
                    int64_t n, int64_t rows, int launch, int64_t stream) {
  return glu_impl(type, act, w_gate, w_up, false, nullptr, x, x_stride, dst, ldd, workspace, workspace_bytes, need, k,
                  n, rows, launch, stream);
}

int qmm_forward_glu_act(int type, int act, const void* w_gate, const void* w_up, const void* xq, float* dst,
                        int64_t ldd, void* workspace, size_t workspace_bytes, size_t* need, int64_t k, int64_t n,
                        int64_t rows, int launch, int64_t stream) {
  return glu_impl(type, act, w_gate, w_up, true, xq, nullptr, 0, dst, ldd, workspace, workspace_bytes, need, k, n,
                  rows, launch, stream);
}

int qmm_glu(int act, const float* gate, const float* up, float* out, int64_t n, int64_t stream) {
  if (act < QMM_GLU_SILU || act > QMM_GLU_GELU || n < 0 || (n > 0 && (!gate || !up || !out))) return QMM_UNSUPPORTED;
  clear_stale_error();
  return status_of(qmm::launch_glu(act, gate, n, up, n, out, n, n, 1, (hipStream_t)stream));
}

int qmm_dequantize(int type, const void* w, void* out, int out_f16, int64_t nelem, int64_t stream) {
  if (qmm_type_bytes(type, nelem) == 0 || !w || !out) return QMM_UNSUPPORTED;
  clear_stale_error();
  return status_of(qmm::launch_dequantize(type, w, out, out_f16, nelem, (hipStream_t)stream));
}

size_t qmm_quantize_scratch_bytes(int type, int64_t nelem) {
  if (qmm_type_bytes(type, nelem) == 0) return 0;
  return qmm::weight_quantize_scratch_bytes(type, nelem);
}

int qmm_quantize_weights(int type, const float* x, void* w, int64_t nelem, void* scratch, size_t scratch_bytes,
                         int64_t stream) {
  if (qmm_type_bytes(type, nelem) == 0 || !x || !w) return QMM_UNSUPPORTED;
  if (scratch_bytes < qmm::weight_quantize_scratch_bytes(type, nelem)) return QMM_WORKSPACE_TOO_SMALL;
  clear_stale_error();
  return status_of(qmm::launch_weight_quantize(type, x, w, nelem, scratch, (hipStream_t)stream));
}

int qmm_cache_plane_bytes(int64_t pages, int kv_heads, int head_dim, int page, size_t* codes, size_t* scales) {
  if (!cache_shape_ok(pages, kv_heads, head_dim, page) || !codes || !scales) return QMM_UNSUPPORTED;
  *codes = (size_t)pages * (size_t)page * (size_t)kv_heads * (size_t)head_dim;
  *scales = *codes / 32 * 2;
  return QMM_OK;
}

int qmm_cache_write(const qmm_cache* cache, const void* k, int64_t k_stride, int64_t k_head_stride, const void* v,
                    int64_t v_stride, int64_t v_head_stride, int dtype, const int64_t* slots, int64_t tokens,
                    int64_t stream) {
  if (!cache_ok(cache) || !qmm::value_type_ok(dtype) || tokens < 0 || tokens > kMostCacheTokens ||
      k_head_stride < cache->head_dim ||
      v_head_stride < cache->head_dim || k_stride < 0 || v_stride < 0)
    return QMM_UNSUPPORTED;
  if (tokens == 0) return QMM_OK;
  if (!k || !v || !slots) return QMM_UNSUPPORTED;
  clear_stale_error();
  return status_of(qmm::launch_cache_write(planes_of(*cache), k, v, dtype, k_stride, k_head_stride, v_stride,
                                           v_head_stride, slots, tokens, (hipStream_t)stream));
}

int qmm_cache_read(const qmm_cache* cache, const int64_t* slots, int64_t tokens, void* k, void* v, int out_dtype,
                   int64_t stream) {
  if (!cache_ok(cache) || !qmm::value_type_ok(out_dtype) || tokens < 0 || tokens > kMostCacheTokens) return QMM_UNSUPPORTED;
  if (tokens == 0) return QMM_OK;
  if (!k || !v || !slots) return QMM_UNSUPPORTED;
  clear_stale_error();
  return status_of(
      qmm::launch_cache_read(planes_of(*cache), slots, tokens, k, v, out_dtype, (hipStream_t)stream));
}

int qmm_attend(const qmm_cache* cache, const void* q, int q_dtype, int64_t q_stride, int64_t q_head_stride,
               int64_t tokens, int heads, const int32_t* q_starts, const int32_t* kv_lens, const int32_t* tables,
               int64_t table_stride, int64_t seqs, int64_t max_q, int64_t max_kv, float scale, int64_t window,
               const float* sinks, void* out, int out_dtype, int64_t out_stride, void* workspace,
               size_t workspace_bytes, size_t* need, int launch, int64_t stream) {
  if (!cache_ok(cache) || need == nullptr || !qmm::value_type_ok(q_dtype) || !qmm::value_type_ok(out_dtype) ||
      heads < 1 || heads > 65535 || heads % cache->kv_heads != 0 || tokens < 0 || seqs < 0 || seqs > 65535 ||
      max_q < 0 || max_kv < 0 || table_stride < 0 || window < 0 || q_head_stride < cache->head_dim || q_stride < 0 ||
      out_stride < (int64_t)heads * cache->head_dim || max_q > INT32_MAX || !(scale >= -1e30f && scale <= 1e30f))
    return QMM_UNSUPPORTED;
  *need = 0;
  if (tokens == 0 || seqs == 0 || max_q == 0) return QMM_OK;
  qmm::AttendArgs a{};
  a.c = planes_of(*cache);
  a.q = q; a.out = out; a.q_starts = q_starts; a.kv_lens = kv_lens; a.tables = tables; a.sinks = sinks;
  a.qs = q_stride; a.qhs = q_head_stride; a.os = out_stride; a.table_stride = table_stride; a.tokens = tokens;
  a.seqs = (int)seqs; a.heads = heads; a.group = heads / cache->kv_heads;
  a.max_q = (int)(max_q < tokens ? max_q : tokens);
  // a sequence's positions lie inside its row of the table
  constexpr int64_t kMostPositions = (int64_t)1 << 30;
  if (table_stride > kMostPositions / cache->page) return QMM_UNSUPPORTED;
  const int64_t cap = table_stride * cache->page;
  a.max_kv = (int)(max_kv < cap ? max_kv : cap);
  a.window = window < a.max_kv ? window : 0;  // a longer one hides nothing (and must not pass 64 bits in the plan)
  a.qdt = q_dtype; a.odt = out_dtype;
  a.sc = scale == 0.0f ? 1.0f : (scale < 0.0f ? -scale : scale) * 1.4426950408889634f;
  a.q_sign = scale == 0.0f ? 0.0f : scale < 0.0f ? -1.0f : 1.0f;
  const int64_t q16 = 16 / qmm::value_bytes(q_dtype);
  a.q_vec = (uintptr_t)q % 16 == 0 && q_stride % q16 == 0 && q_head_stride % q16 == 0;
  a.out_vec = (uintptr_t)out % (4 * qmm::value_bytes(out_dtype)) == 0 && out_stride % 4 == 0;
  a.group_inv = a.group > 1 ? (uint32_t)((((uint64_t)1 << 32) + a.group - 1) / a.group) : 0;
  a.page_bits = __builtin_ctz((unsigned)cache->page);
  if (!qmm::attend_fits(a)) return QMM_UNSUPPORTED;
  *need = qmm::attend_workspace_bytes(a, cu_count());
  if (!launch) return QMM_OK;
  if (g_fail_next.exchange(false)) return QMM_NO_ROOM;
  if (!q || !out || !q_starts || !kv_lens || (!tables && a.max_kv > 0) || !aligned16(workspace)) return QMM_UNSUPPORTED;
  if (*need > 0 && (workspace == nullptr || workspace_bytes < *need)) return QMM_WORKSPACE_TOO_SMALL;
  clear_stale_error();
  return status_of(qmm::launch_attend(a, cu_count(), workspace, (hipStream_t)stream));
}

int qmm_pages_step(const qmm_pages* pages, const int32_t* keep, const int32_t* fresh, int64_t tokens, int32_t* q_starts,
                   int32_t* taken, int64_t* slots, int32_t* positions, int32_t* seq, int64_t stream) {
  if (!pages || pages->seqs < 0 || pages->seqs > qmm::pages_most_seqs() || tokens < 0 || tokens > kMostCacheTokens ||
      pages->page < 16 || pages->page > 256 || (pages->page & (pages->page - 1)) != 0 || pages->row_pages < 0 ||
      pages->table_stride < pages->row_pages || pages->pool < 0 || pages->pool > INT32_MAX ||
      pages->row_pages > ((int64_t)1 << 30) / pages->page ||
      pages->table_stride > INT32_MAX || (int64_t)pages->seqs * pages->table_stride > (int64_t)1 << 30 || !pages->free_count || !q_starts ||
      (pages->row_pages > 0 && pages->seqs > 0 && !pages->tables) || (pages->pool > 0 && !pages->free_pages) ||
      (pages->seqs > 0 && (!pages->lens || !taken)) || (tokens > 0 && !slots))
    return QMM_UNSUPPORTED;
  qmm::PagesArgs a{};
  a.tables = pages->tables; a.lens = pages->lens; a.free_pages = pages->free_pages; a.free_count = pages->free_count;
  a.keep = keep; a.fresh = fresh; a.q_starts = q_starts; a.taken = taken; a.slots = slots; a.positions = positions;
  a.seq = seq; a.table_stride = pages->table_stride; a.row_pages = pages->row_pages; a.pool = pages->pool;
  a.tokens = tokens; a.seqs = pages->seqs; a.page_bits = __builtin_ctz((unsigned)pages->page);
  clear_stale_error();
  return status_of(qmm::launch_pages_step(a, (hipStream_t)stream));
}

int qmm_adapters_add(int count, const qmm_adapter* adapters, int slots, int w_dtype, const void* x, int x_dtype,
                     int64_t x_stride, const int32_t* ids, int64_t k, int64_t rows, void* workspace,
                     size_t workspace_bytes, size_t* need, int launch, int64_t stream) {
  if (count < 1 || count > qmm::kMaxTargets || !adapters || slots < 0 || slots > qmm::lora_most_slots() || !qmm::value_type_ok(w_dtype) ||
      !qmm::value_type_ok(x_dtype) || need == nullptr || k < 32 || k % 32 != 0 || k > (int64_t)1 << 30 ||
      x_stride < k || rows < 0 || rows > (int64_t)1 << 20)
    return QMM_UNSUPPORTED;
  qmm::LoraArgs a{};
  a.x = x; a.ids = ids; a.xs = x_stride; a.k = k; a.rows = rows; a.count = count; a.slots = slots;
  a.x_vec = aligned16(x) && x_stride * qmm::value_bytes(x_dtype) % 16 == 0;
  for (int i = 0; i < count; i++) {
    const qmm_adapter& d = adapters[i];
    if (d.n < 1 || d.n > INT32_MAX || d.rank < 8 || d.rank > qmm::lora_most_rank() || d.rank % 8 != 0 ||
        d.y_stride < d.n || d.out_stride < d.n || (d.y == d.out && d.y && d.y_stride != d.out_stride) ||
        !aligned16(d.a) || !aligned16(d.b))
      return QMM_UNSUPPORTED;
    if (d.out && d.out == x) return QMM_UNSUPPORTED;  // one in the place that all read
    // two projections in one place, or one in the place that another reads
    for (int j = 0; j < i; j++)
      if (d.out && (d.out == adapters[j].out || d.out == adapters[j].y || d.y == adapters[j].out)) return QMM_UNSUPPORTED;
    qmm::LoraTarget& t = a.t[i];
    t.a = d.a; t.b = d.b; t.scales = d.scales; t.y = d.y; t.out = d.out;
    t.n = d.n; t.ldy = d.y_stride; t.ldo = d.out_stride; t.rank = d.rank;
    t.vec = aligned16(d.y) && aligned16(d.out) && d.y_stride % 4 == 0 && d.out_stride % 4 == 0;
  }
  *need = 0;
  if (rows == 0) return QMM_OK;
  if (!qmm::lora_fits(a)) return QMM_UNSUPPORTED;
  *need = qmm::lora_plan(a, workspace, cu_count());
  if (!launch) return QMM_OK;
  if (g_fail_next.exchange(false)) return QMM_NO_ROOM;
  if (!x || !ids || !aligned16(workspace)) return QMM_UNSUPPORTED;
  for (int i = 0; i < count; i++)
    if (!a.t[i].y || !a.t[i].out || (slots > 0 && (!a.t[i].a || !a.t[i].b))) return QMM_UNSUPPORTED;
  if (*need > 0 && (workspace == nullptr || workspace_bytes < *need)) return QMM_WORKSPACE_TOO_SMALL;
  if (adapters_overlap(a, x_dtype, w_dtype, workspace, *need)) return QMM_UNSUPPORTED;
  clear_stale_error();
  return status_of(qmm::launch_lora(a, x_dtype, w_dtype, (hipStream_t)stream));
}

int qmm_sample(const void* logits, int dtype, int64_t stride, const float* u, const float* temperature,
               const int32_t* top_k, const float* top_p, const float* min_p, int32_t* ids, float* probs, int64_t vocab,
               int64_t rows, void* workspace, size_t workspace_bytes, size_t* need, int launch, int64_t stream) {
  if (!qmm::value_type_ok(dtype) || need == nullptr || vocab < 1 || vocab > qmm::sample_most_vocab() || stride < vocab ||
      rows < 0 || rows > 65535)
    return QMM_UNSUPPORTED;
  *need = 0;
  if (rows == 0) return QMM_OK;
  qmm::SampleArgs a{};
  a.logits = logits; a.u = u; a.temperature = temperature; a.top_k = top_k; a.top_p = top_p; a.min_p = min_p;
  a.ids = ids; a.probs = probs; a.stride = stride; a.rows = (int)rows; a.vocab = (int)vocab;
  a.vec = (uintptr_t)logits % (4 * qmm::value_bytes(dtype)) == 0 && stride % 4 == 0;
  *need = qmm::sample_plan(a, workspace, cu_count());
  if (!launch) return QMM_OK;
  if (g_fail_next.exchange(false)) return QMM_NO_ROOM;
  if (!logits || !u || !ids || !aligned16(workspace)) return QMM_UNSUPPORTED;
  if (workspace == nullptr || workspace_bytes < *need) return QMM_WORKSPACE_TOO_SMALL;
  clear_stale_error();
  return status_of(qmm::launch_sample(a, dtype, (hipStream_t)stream));
}

int qmm_moe_forward(int type, const void* w, int num_experts, const float* x, int64_t x_stride,
                    const int32_t* sorted_ids, const int32_t* expert_ids, const float* topk_w, int topk, float* dst,
                    int64_t ldd, void* workspace, size_t workspace_bytes, size_t* need, int64_t k, int64_t n,
                    int64_t size_m, int launch, int64_t stream) {
  if (!qmm::moe_supported(type, k) || !shape_ok(type, k, n, size_m) || need == nullptr || ldd < n || x_stride < k ||
      num_experts < 1 || topk < 1 || (topk_w == nullptr && size_m % topk != 0) || size_m > ((int64_t)1 << 30))
    return QMM_UNSUPPORTED;
  const int64_t in_rows = topk_w ? size_m : size_m / topk;
  const int layout = qmm::moe_act_layout(type);
  const size_t act = (qmm::act_bytes(layout, k, in_rows) + 255) / 256 * 256;
  const size_t bytes = act + qmm::moe_runs_bytes(size_m);
  *need = bytes;
  if (!launch) return QMM_OK;
  if (g_fail_next.exchange(false)) return QMM_NO_ROOM;
  if (workspace_bytes < bytes || workspace == nullptr) return QMM_WORKSPACE_TOO_SMALL;
  if (!w || !x || !dst || !sorted_ids || !expert_ids) return QMM_UNSUPPORTED;
  const hipStream_t st = (hipStream_t)stream;
  clear_stale_error();
  if (qmm::moe_fp4_fused_takes(type, k, size_m)) {
    if (qmm::launch_moe_fp4_fused(w, num_experts, n, k, x, x_stride, expert_ids, sorted_ids, topk_w, topk, size_m, dst,
                                  ldd, st) != hipSuccess)
      return QMM_DEVICE_ERROR;
    g_moe_launches.fetch_add(1, std::memory_order_relaxed);
    return QMM_OK;
  }
  if (layout == qmm::ACT_Q8K && qmm::moe_kq_fused_takes(type, k, size_m)) {
    if (qmm::launch_moe_kq_fused(type, w, num_experts, n, k, x, x_stride, expert_ids, sorted_ids, topk_w, topk, size_m,
                                 dst, ldd, q8k_scale(), (int)cu_count(), st) != hipSuccess)
      return QMM_DEVICE_ERROR;
    g_moe_launches.fetch_add(1, std::memory_order_relaxed);
    return QMM_OK;
  }
  // the activation's planes (Q8_K for Q4_K / Q6_K, else Q8_0) and the run
  // table, one launch; then the grouped kernel
  int32_t* runs = (int32_t*)((char*)workspace + act);
  if (qmm::launch_act_quantize_moe(layout, x, x_stride, k, in_rows, workspace, expert_ids, size_m, runs, q8k_scale(),
                                   st) != hipSuccess)
    return QMM_DEVICE_ERROR;
  const qmm::ActPlanes p = qmm::act_planes(layout, workspace, k, in_rows);
  const hipError_t e =
      layout == qmm::ACT_Q8K
          ? qmm::launch_moe_kq(type, w, num_experts, n, k, p, runs, sorted_ids, topk_w, topk, size_m, dst, ldd,
                               (int)cu_count(), st)
          : qmm::launch_moe(type, w, num_experts, n, k, p, runs, sorted_ids, topk_w, topk, size_m, dst, ldd,
                            (int)cu_count(), st);
  if (e != hipSuccess) return QMM_DEVICE_ERROR;
  g_moe_launches.fetch_add(1, std::memory_order_relaxed);
  return QMM_OK;
}

uint64_t qmm_moe_launches(void) { return g_moe_launches.load(std::memory_order_relaxed); }

int qmm_moe_forward_prefill(int type, const void* w, int num_experts, const void* x, int x_dtype, int64_t x_stride,
                            const int32_t* sorted_ids, const int32_t* expert_ids, const float* topk_w, int topk,
                            float* dst, int64_t ldd, void* workspace, size_t workspace_bytes, size_t* need, int64_t k,
                            int64_t n, int64_t size_m, int launch, int64_t stream) {
  if (!qmm::moe_pf_supported(type, k) || !shape_ok(type, k, n, size_m) || need == nullptr || ldd < n ||
      x_stride < k || num_experts < 1 || topk < 1 || (topk_w == nullptr && size_m % topk != 0) ||
      size_m > ((int64_t)1 << 30) || x_dtype < QMM_X_F16 || x_dtype > QMM_X_F32)
    return QMM_UNSUPPORTED;
  const int64_t in_rows = topk_w ? size_m : size_m / topk;
  // 32-bit byte offsets inside the kernel: an expert's weights, the 16-bit rows
  if (n * qmm::moe_pf_row_bytes(type, k) >= ((int64_t)1 << 31) || in_rows * k * 2 >= ((int64_t)1 << 31))
    return QMM_UNSUPPORTED;
  const size_t runs_b = qmm::align_up(qmm::moe_runs_bytes(size_m), 256);
  const size_t chunks_b = qmm::align_up(qmm::moe_pf_chunks_bytes(size_m), 256);
  const size_t xo_b = qmm::align_up((size_t)(in_rows * k * 2), 256);
  *need = runs_b + chunks_b + xo_b;
  if (!launch) return QMM_OK;
  if (g_fail_next.exchange(false)) return QMM_NO_ROOM;
  if (workspace_bytes < *need || workspace == nullptr) return QMM_WORKSPACE_TOO_SMALL;
  if (!w || !x || !dst || !sorted_ids || !expert_ids || !qmm::moe_pf_weights_ok(type, w)) return QMM_UNSUPPORTED;
  const hipStream_t st = (hipStream_t)stream;
  clear_stale_error();
  int32_t* runs = (int32_t*)workspace;
  int32_t* chunks = (int32_t*)((char*)workspace + runs_b);
  uint16_t* xo = (uint16_t*)((char*)workspace + runs_b + chunks_b);
  // A 16-bit input with 16-byte aligned rows is read in place; an f32 input
  // is rounded to f16 (the reference's caller converts a prompt's input to
  // f16, moe_card.rs:113-121) and any other is copied aligned, in the
  // prologue that writes the routing tables.
  const bool direct = x_dtype != QMM_X_F32 && ((uintptr_t)x & 15) == 0 && x_stride % 8 == 0 &&
                      in_rows * x_stride * 2 < ((int64_t)1 << 31);
  const int kind = direct ? -1 : x_dtype == QMM_X_F32 ? 2 : x_dtype;
  if (qmm::launch_moe_pf_prep(expert_ids, size_m, runs, chunks, x, kind, x_stride, k, in_rows, xo, (int)cu_count(),
                              st) != hipSuccess)
    return QMM_DEVICE_ERROR;
  const hipError_t e = qmm::launch_moe_pf(type, x_dtype == QMM_X_BF16, w, num_experts, n, k,
                                          direct ? (const uint16_t*)x : xo, direct ? x_stride : k, chunks, sorted_ids,
                                          topk_w, topk, size_m, dst, ldd, st);
  if (e != hipSuccess) return QMM_DEVICE_ERROR;
  g_moe_prefill_launches.fetch_add(1, std::memory_order_relaxed);
  return QMM_OK;
}

uint64_t qmm_moe_prefill_launches(void) { return g_moe_prefill_launches.load(std::memory_order_relaxed); }

size_t qmm_wire_bytes(int64_t n) {
  const int64_t b = qmm::wire_bytes(n);
  return b < 0 ? 0 : (size_t)b;
}

int qmm_wire_encode(const float* x, int64_t n, void* out, int64_t stream) {
  if (n < 0 || qmm::wire_bytes(n) < 0 || (n > 0 && (!x || !out))) return QMM_UNSUPPORTED;
  if (n == 0) return QMM_OK;
  clear_stale_error();
  return status_of(qmm::launch_wire_encode(x, n, out, (hipStream_t)stream));
}

int qmm_wire_decode(const void* in, size_t in_bytes, int64_t n, float* out, int64_t stream) {
  // the reference rejects a payload whose length is not the one n values take
  // (dequantize_q8_0, src/inference/quant.rs:65-77)
  const int64_t want = qmm::wire_bytes(n);
  if (want < 0 || (int64_t)in_bytes != want || (n > 0 && (!in || !out))) return QMM_UNSUPPORTED;
  if (n == 0) return QMM_OK;
  clear_stale_error();
  return status_of(qmm::launch_wire_decode(in, n, out, (hipStream_t)stream));
}

void qmm_fail_next_launch(void) { g_fail_next.store(true); }

int qmm_fill_normal(float* out, int64_t n, uint64_t seed, float mean, float std, int64_t stream) {
  if (!out || n < 0) return QMM_UNSUPPORTED;
  if (n == 0) return QMM_OK;
  clear_stale_error();
  return status_of(qmm::launch_fill_normal(out, n, seed, mean, std, (hipStream_t)stream));
}

uint64_t qmm_matvec_launches(void) { return g_matvec_launches.load(); }
uint64_t qmm_gemm_launches(void) { return g_gemm_launches.load(); }

}  // extern "C"
