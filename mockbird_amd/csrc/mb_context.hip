// Context lifetime, errors, weights, ring bookkeeping and the host-pointer
// entry points of the C ABI (include/mockbird_hip.h).  Kernels live in
// ring.hip; this file only allocates, validates, stages and launches.
#include <algorithm>
#include <cmath>
#include <cstring>

#include "kv_types.h"
#include "mb_internal.h"

namespace mb {

const DeviceTensor* find(mb_ctx* ctx, const std::string& name, std::initializer_list<int64_t> dims,
                         std::string& missing) {
  auto it = ctx->weights.find(name);
  if (it == ctx->weights.end()) {
    if (missing.empty()) missing = "weight not uploaded: " + name;
    return nullptr;
  }
  const DeviceTensor& t = it->second;
  if (t.dims.size() != dims.size() || !std::equal(dims.begin(), dims.end(), t.dims.begin())) {
    if (missing.empty()) missing = "weight has the wrong shape: " + name;
    return nullptr;
  }
  return &t;
}

// A device tensor owned by the context under an internal name (freed with
// the uploaded weights); reallocated only when its size changes.
float* internal_tensor(mb_ctx* ctx, const std::string& name, int64_t numel) {
  DeviceTensor& t = ctx->weights[name];
  if (t.ptr && t.numel != numel) {
    (void)hipStreamSynchronize(ctx->stream);
    (void)hipFree(t.ptr);
    ctx->device_bytes -= t.numel * 4;
    t.ptr = nullptr;
  }
  if (!t.ptr) {
    if (hipMalloc(&t.ptr, (size_t)numel * 4) != hipSuccess) {
      ctx->weights.erase(name);
      return nullptr;
    }
    ctx->device_bytes += numel * 4;
    ctx->graph_gen++;
  }
  t.numel = numel;
  t.dims = {numel};
  return t.ptr;
}

void drop_internal(mb_ctx* ctx, const std::string& name) {
  auto it = ctx->weights.find(name);
  if (it == ctx->weights.end()) return;
  if (it->second.ptr) {
    (void)hipStreamSynchronize(ctx->stream);  // no launch in flight still reads it
    (void)hipFree(it->second.ptr);
    ctx->device_bytes -= it->second.numel * 4;
    ctx->graph_gen++;
  }
  ctx->weights.erase(it);
}


int fail(mb_ctx* ctx, int code, const char* fmt, ...) {
  if (ctx) {
    char buf[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof buf, fmt, ap);
    va_end(ap);
    ctx->err = buf;
  }
  return code;
}

int hip_fail(mb_ctx* ctx, hipError_t e, const char* what) {
  if (e == hipErrorOutOfMemory)
    return fail(ctx, MB_ERR_NOMEM, "%s: %s", what, hipGetErrorString(e));
  return fail(ctx, MB_ERR_HIP, "%s: %s", what, hipGetErrorString(e));
}

// The AttnSplit of a kernel-level attention call: its stream's set, a free one
// if it has none, else none, and none while the stream is captured (a replay
// would share it with later calls).  A set goes by the stream's handle: the
// runtime's hipStreamDestroy waits for the stream's work (43 ms of it, queued
// before), so a handle that another stream gets later brings none along.
static AttnSplit claim_split(mb_ctx* ctx) {
  hipStreamCaptureStatus st = hipStreamCaptureStatusNone;
  if (hipStreamIsCapturing(ctx->stream, &st) != hipSuccess || st != hipStreamCaptureStatusNone) {
    (void)hipGetLastError();
    return {};
  }
  int set = 0;
  for (int i = 1; i < kSplitSets; i++) {
    if (ctx->split_taken[i] && ctx->split_stream[i] == ctx->stream) return split_set(ctx, i);
    if (!ctx->split_taken[i] && !set) set = i;
  }
  if (!set) return {};
  ctx->split_taken[set] = true;
  ctx->split_stream[set] = ctx->stream;
  return split_set(ctx, set);
}

hipError_t sync_stream(mb_ctx* ctx) {
  const hipError_t e = hipStreamSynchronize(ctx->stream);
  if (e == hipSuccess)
    for (int i = 1; i < kSplitSets; i++)
      if (ctx->split_stream[i] == ctx->stream) ctx->split_taken[i] = false;
  return e;
}

void drop_scratch(mb_ctx* ctx, const char* name) {
  Scratch& s = ctx->scratch[name];
  if (!s.ptr) return;
  (void)hipStreamSynchronize(ctx->stream);
  (void)hipFree(s.ptr);
  ctx->device_bytes -= (int64_t)s.bytes;
  ctx->graph_gen++;
  s.ptr = nullptr;
  s.bytes = 0;
}

void* scratch(mb_ctx* ctx, const char* name, size_t bytes) {
  Scratch& s = ctx->scratch[name];
  if (s.bytes >= bytes && s.ptr) return s.ptr;
  drop_scratch(ctx, name);
  size_t want = bytes < 4096 ? 4096 : bytes;
  ctx->graph_gen++;
  if (hipMalloc(&s.ptr, want) != hipSuccess) {
    s.ptr = nullptr;
    return nullptr;
  }
  s.bytes = want;
  ctx->device_bytes += (int64_t)want;
  return s.ptr;
}

}  // namespace mb

using namespace mb;

namespace {

int check_cfg(const mb_config& c, std::string& why) {
  char buf[256];
  if (c.n_layers < 1 || c.n_layers > 64) {
    snprintf(buf, sizeof buf, "n_layers %d out of [1, 64]", c.n_layers);
  } else if (c.capacity < 1 || c.capacity > (1 << 20)) {
    snprintf(buf, sizeof buf, "capacity %d out of [1, 2^20]", c.capacity);
  } else if (c.max_seqs < 1 || c.max_seqs > 65535) {
    snprintf(buf, sizeof buf, "max_seqs %d out of [1, 65535]", c.max_seqs);
  } else if (c.max_rows < 1 || c.max_rows > (1 << 20)) {
    snprintf(buf, sizeof buf, "max_rows %d out of [1, 2^20]", c.max_rows);
  } else if (c.kv_dtype != MB_KV_F32 && c.kv_dtype != MB_KV_BF16) {
    snprintf(buf, sizeof buf, "kv_dtype %d is neither MB_KV_F32 nor MB_KV_BF16", c.kv_dtype);
  } else if (c.wrap != 0 && c.wrap != 1) {
    snprintf(buf, sizeof buf, "wrap must be 0 or 1, got %d", c.wrap);
  } else if (c.vocab < 0) {
    snprintf(buf, sizeof buf, "vocab %d is negative", c.vocab);
  } else if (c.device < 0) {
    snprintf(buf, sizeof buf, "device %d is negative", c.device);
  } else {
    return 0;
  }
  why = buf;
  return 1;
}

// Validate positions of a host-pointer call against the ring's rule.
int check_positions(mb_ctx* ctx, int B, const int32_t* pos0, const int32_t* n_rows, int rows_max) {
  for (int b = 0; b < B; b++) {
    const int64_t n = n_rows ? n_rows[b] : 1;
    if (pos0[b] < 0) return fail(ctx, MB_ERR_ARG, "sequence %d: negative position %d", b, pos0[b]);
    if (n < 0 || n > rows_max || n > ctx->cfg.capacity)
      return fail(ctx, MB_ERR_ARG, "sequence %d: n_rows %lld out of [0, min(%d, capacity %d)]", b,
                  (long long)n, rows_max, ctx->cfg.capacity);
    const int64_t last = (int64_t)pos0[b] + n - 1;
    if (last > INT32_MAX - 1) return fail(ctx, MB_ERR_ARG, "sequence %d: position overflow", b);
    if (!ctx->cfg.wrap && n > 0 && last >= ctx->cfg.capacity)
      return fail(ctx, MB_ERR_RANGE,
                  "decode position %lld exceeds the KV ring (%d slots); it must be sized "
                  "prefill_rows + max_new_frames",
                  (long long)last, ctx->cfg.capacity);
  }
  return MB_OK;
}

int check_common(mb_ctx* ctx, int layer, int B) {
  if (!ctx) return MB_ERR_ARG;
  if (layer < 0 || layer >= ctx->cfg.n_layers)
    return fail(ctx, MB_ERR_ARG, "layer %d out of [0, %d)", layer, ctx->cfg.n_layers);
  if (B < 0 || B > ctx->cfg.max_seqs)
    return fail(ctx, MB_ERR_ARG, "B %d out of [0, %d]", B, ctx->cfg.max_seqs);
  return MB_OK;
}

// (cos, sin) of float(pos) * inv_freq[i], in double, rounded to fp32; made once
// per process (some 25 ms), for every context.
const std::vector<float2>& rope_table() {
  static const std::vector<float2> table = [] {
    std::vector<float2> tab((size_t)kRopeTab * 32);
    for (int i = 0; i < 32; i++) {
      float inv;
      memcpy(&inv, &kInvFreqBits[i], 4);
      for (int p = 0; p < kRopeTab; p++) {
        const float a = (float)p * inv;
        tab[(size_t)p * 32 + i] = make_float2((float)cos((double)a), (float)sin((double)a));
      }
    }
    return tab;
  }();
  return table;
}

int check_layers(mb_ctx* ctx, int layer0, int n_layers, int B) {
  const int rc = check_common(ctx, layer0, B);
  if (rc) return rc;
  if (n_layers < 0 || n_layers > ctx->cfg.n_layers - layer0)
    return fail(ctx, MB_ERR_ARG, "%d layers from %d on, of %d", n_layers, layer0, ctx->cfg.n_layers);
  return MB_OK;
}

int check_tree(mb_ctx* ctx, int layer0, int n_layers, int B, int rows_max) {
  const int rc = check_layers(ctx, layer0, n_layers, B);
  if (rc) return rc;
  if (rows_max < 1 || rows_max > kTreeMaxNodes)
    return fail(ctx, MB_ERR_ARG, "rows_max %d out of [1, %d]", rows_max, kTreeMaxNodes);
  return MB_OK;
}

int check_groups(mb_ctx* ctx, int layer0, int n_layers, int B, int width, const void* pos_from,
                 const void* pos_to) {
  const int rc = check_layers(ctx, layer0, n_layers, B);
  if (rc) return rc;
  if (width < 1 || width > kBeamMax || B % width)
    return fail(ctx, MB_ERR_ARG, "width %d out of [1, %d], or not a divisor of B %d", width, kBeamMax, B);
  if (!pos_from != !pos_to) return fail(ctx, MB_ERR_ARG, "pos_from and pos_to come together");
  return MB_OK;
}

int check_beam(mb_ctx* ctx, int B, int width, int vocab, int n_out) {
  if (!ctx) return MB_ERR_ARG;
  if (B < 0 || width < 1 || width > kBeamMax || n_out < 1 || n_out > kBeamMax)
    return fail(ctx, MB_ERR_ARG, "B %d voices of %d beams, %d chosen: beams and choices are 1 .. %d", B,
                width, n_out, kBeamMax);
  // (ids are int32, with room for one scan past the last)
  if (vocab < 1 || vocab > (1 << 30)) return fail(ctx, MB_ERR_ARG, "vocab %d out of [1, 2^30]", vocab);
  return MB_OK;
}

bool overlap(const void* a, int64_t an, const void* b, int64_t bn) {
  return a && b && (uintptr_t)a < (uintptr_t)b + bn && (uintptr_t)b < (uintptr_t)a + an;
}

int check_beam_options(mb_ctx* ctx, int B, int width, int vocab, int n_out, const void* scores,
                       const void* done, int32_t end_id, const void* seen, double penalty,
                       const void* scores_out, const void* done_out, const void* seen_out) {
  if (end_id < -1 || end_id >= vocab || (done && end_id < 0))
    return fail(ctx, MB_ERR_ARG, "end_id %d is no id of %d (-1 where no beam is done)", end_id, vocab);
  if (seen_out && !seen) return fail(ctx, MB_ERR_ARG, "seen_out needs seen");
  if (seen && (!((float)penalty > 0.f) || !((float)penalty < INFINITY)))
    return fail(ctx, MB_ERR_ARG, "penalty %g is not a positive fp32 number", penalty);
  const int64_t rows = (int64_t)B * width * 4, outs = (int64_t)B * n_out * 4, words = ((int64_t)vocab + 31) / 32;
  if (overlap(scores, rows, scores_out, outs) || overlap(done, rows, done_out, outs) ||
      overlap(seen, rows * words, seen_out, outs * words))
    return fail(ctx, MB_ERR_ARG, "an output overlaps its input");
  return MB_OK;
}

// Rows `stride` elements of e bytes apart start at multiples of 16 bytes.
bool aligned_rows(const void* p, int64_t stride, int e) {
  return ((uintptr_t)p & 15) == 0 && (stride * e & 15) == 0;
}

int check_work(mb_ctx* ctx, const void* work, int64_t bytes, int64_t need) {
  if (need == 0) return MB_OK;
  if (!work || bytes < need)
    return fail(ctx, MB_ERR_ARG, "the workspace holds %lld bytes of %lld", (long long)(work ? bytes : 0),
                (long long)need);
  if ((uintptr_t)work & 15) return fail(ctx, MB_ERR_ARG, "the workspace must be 16-byte aligned");
  return MB_OK;
}

}  // namespace

extern "C" {

int mb_abi_version(void) { return MB_ABI_VERSION; }

int mb_create(const mb_config* cfg, mb_ctx** out) {
  if (!cfg || !out) return MB_ERR_ARG;
  *out = nullptr;
  std::string why;
  if (check_cfg(*cfg, why)) {
    fprintf(stderr, "mb_create: %s\n", why.c_str());
    return MB_ERR_ARG;
  }
  // the caller's current device is given back on return
  mb::DeviceGuard guard(cfg->device);
  mb_ctx* ctx = new mb_ctx();
  ctx->cfg = *cfg;
  ctx->device = cfg->device;
  int rc = MB_OK;
  do {
    hipError_t e = hipSetDevice(cfg->device);
    if (e != hipSuccess) { rc = hip_fail(ctx, e, "hipSetDevice"); break; }
    {
      int cus = 0, xccs = 0;
      if (hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, cfg->device) ==
              hipSuccess &&
          hipDeviceGetAttribute(&xccs, hipDeviceAttributeNumberOfXccs, cfg->device) == hipSuccess &&
          xccs > 0 && cus >= xccs) {
        ctx->xcds = xccs;
        ctx->cus_per_xcd = cus / xccs;
      }
    }
    if ((rc = noalloc_init(ctx))) break;
    e = hipStreamCreateWithFlags(&ctx->own_stream, hipStreamNonBlocking);
    if (e != hipSuccess) { rc = hip_fail(ctx, e, "hipStreamCreate"); break; }
    ctx->stream = ctx->own_stream;
    const int64_t slots = (int64_t)cfg->n_layers * cfg->max_seqs * cfg->capacity;
    ctx->ring_bytes = (size_t)slots * H * HD * kv_elem_bytes(ctx);
    e = hipMalloc(&ctx->ring_k, ctx->ring_bytes);
    if (e != hipSuccess) { rc = hip_fail(ctx, e, "hipMalloc(ring K)"); break; }
    e = hipMalloc(&ctx->ring_v, ctx->ring_bytes);
    if (e != hipSuccess) { rc = hip_fail(ctx, e, "hipMalloc(ring V)"); break; }
    e = hipMalloc(&ctx->slot_pos, (size_t)slots * sizeof(int32_t));
    if (e != hipSuccess) { rc = hip_fail(ctx, e, "hipMalloc(slot_pos)"); break; }
    {
      const std::vector<float2>& tab = rope_table();
      e = hipMalloc(&ctx->rope_tab, tab.size() * sizeof(float2));
      if (e != hipSuccess) { rc = hip_fail(ctx, e, "hipMalloc(rope table)"); break; }
      e = hipMemcpy(ctx->rope_tab, tab.data(), tab.size() * sizeof(float2), hipMemcpyHostToDevice);
      if (e != hipSuccess) { rc = hip_fail(ctx, e, "hipMemcpy(rope table)"); break; }
    }
    e = hipMalloc(&ctx->split_part, kSplitSets * (kSplitFloats + kSplitMaxUnits) * 4);
    if (e != hipSuccess) { rc = hip_fail(ctx, e, "hipMalloc(attention split)"); break; }
    ctx->split_count = (int32_t*)(ctx->split_part + kSplitSets * kSplitFloats);
    rc = launch_fill_i32(ctx, ctx->split_count, kSplitSets * kSplitMaxUnits, 0);
    if (rc) break;
    ctx->device_bytes = 2 * (int64_t)ctx->ring_bytes + slots * 4 + (int64_t)kRopeTab * 32 * 8 +
                        (int64_t)kSplitSets * (kSplitFloats + kSplitMaxUnits) * 4;
    // every slot empty; K/V zero so a read of an unwritten slot is well defined
    rc = launch_fill_kv(ctx, ctx->ring_k, (int64_t)(ctx->ring_bytes / kv_elem_bytes(ctx)), 0.f);
    if (rc) break;
    rc = launch_fill_kv(ctx, ctx->ring_v, (int64_t)(ctx->ring_bytes / kv_elem_bytes(ctx)), 0.f);
    if (rc) break;
    rc = launch_fill_i32(ctx, ctx->slot_pos, slots, -1);
    if (rc) break;
    e = hipStreamSynchronize(ctx->stream);
    if (e != hipSuccess) { rc = hip_fail(ctx, e, "hipStreamSynchronize"); break; }
  } while (0);
  if (rc != MB_OK) {
    fprintf(stderr, "mb_create: %s\n", ctx->err.c_str());
    mb_destroy(ctx);
    return rc;
  }
  *out = ctx;
  return MB_OK;
}

void mb_destroy(mb_ctx* ctx) {
  MB_DEVICE_GUARD(ctx);
  if (!ctx) return;
  if (ctx->stream) (void)hipStreamSynchronize(ctx->stream);
  mb::codec_free(ctx);
  for (auto& kv : ctx->weights) (void)hipFree(kv.second.ptr);
  for (auto& kv : ctx->scratch) (void)hipFree(kv.second.ptr);
  (void)hipFree(ctx->ring_k);
  (void)hipFree(ctx->ring_v);
  (void)hipFree(ctx->slot_pos);
  (void)hipFree(ctx->rope_tab);
  (void)hipFree(ctx->split_part);
  for (void* p : {(void*)ctx->local_k, (void*)ctx->local_v, (void*)ctx->local_sp,
                  (void*)ctx->local_pos, (void*)ctx->seen, (void*)ctx->tokens, (void*)ctx->cont})
    (void)hipFree(p);
  if (ctx->frame_exec) (void)hipGraphExecDestroy(ctx->frame_exec);
  if (ctx->capture_stream) (void)hipStreamDestroy(ctx->capture_stream);
  if (ctx->own_stream) (void)hipStreamDestroy(ctx->own_stream);
  delete ctx;
}

const char* mb_last_error(const mb_ctx* ctx) { return ctx ? ctx->err.c_str() : "null context"; }

int mb_set_stream(mb_ctx* ctx, void* hip_stream) {
  if (!ctx) return MB_ERR_ARG;
  ctx->stream = (hipStream_t)hip_stream;
  return MB_OK;
}

void* mb_get_stream(mb_ctx* ctx) { return ctx ? (void*)ctx->stream : nullptr; }

int mb_synchronize(mb_ctx* ctx) {
  MB_DEVICE_GUARD(ctx);
  if (!ctx) return MB_ERR_ARG;
  MB_HIP(ctx, sync_stream(ctx));
  return MB_OK;
}

int64_t mb_device_bytes(const mb_ctx* ctx) { return ctx ? ctx->device_bytes : 0; }

int mb_cancel(mb_ctx* ctx, int on) {
  if (!ctx) return MB_ERR_ARG;
  ctx->cancel.store(on ? 1 : 0);
  return MB_OK;
}

int mb_upload_tensor(mb_ctx* ctx, const char* name, const float* data, const int64_t* dims,
                     int ndims) {
  MB_DEVICE_GUARD(ctx);
  if (!ctx) return MB_ERR_ARG;
  if (!name || !data || !dims || ndims < 1 || ndims > 4)
    return fail(ctx, MB_ERR_ARG, "mb_upload_tensor: bad arguments");
  if (name[0] == '#')  // the context's own derived tensors live under '#' names
    return fail(ctx, MB_ERR_ARG, "mb_upload_tensor: names starting with '#' are reserved");
  int64_t numel = 1;
  for (int i = 0; i < ndims; i++) {
    if (dims[i] < 1) return fail(ctx, MB_ERR_ARG, "mb_upload_tensor(%s): dim %d is %lld", name, i,
                                 (long long)dims[i]);
    if (dims[i] > ((int64_t)1 << 40) / numel)
      return fail(ctx, MB_ERR_ARG, "mb_upload_tensor(%s): more than 2^40 elements", name);
    numel *= dims[i];
  }
  DeviceTensor& t = ctx->weights[name];
  if (t.ptr && t.numel != numel) {
    MB_HIP(ctx, sync_stream(ctx));
    (void)hipFree(t.ptr);
    ctx->device_bytes -= t.numel * 4;
    t.ptr = nullptr;
  }
  if (!t.ptr) {
    hipError_t e = hipMalloc(&t.ptr, (size_t)numel * 4);
    if (e != hipSuccess) {
      ctx->weights.erase(name);
      return hip_fail(ctx, e, "hipMalloc(weight)");
    }
    ctx->device_bytes += numel * 4;
  }
  t.numel = numel;
  t.dims.assign(dims, dims + ndims);
  ctx->model_ok = false;
  ctx->codec_ok = false;
  ctx->graph_gen++;
  MB_HIP(ctx, hipMemcpyAsync(t.ptr, data, (size_t)numel * 4, hipMemcpyHostToDevice, ctx->stream));
  MB_HIP(ctx, sync_stream(ctx));
  return MB_OK;
}

int mb_ring_reset(mb_ctx* ctx, int n, const int32_t* seq_ids) {
  MB_DEVICE_GUARD(ctx);
  if (!ctx) return MB_ERR_ARG;
  const int64_t C = ctx->cfg.capacity;
  if (n < 0) {
    const int64_t slots = (int64_t)ctx->cfg.n_layers * ctx->cfg.max_seqs * C;
    int rc = launch_fill_i32(ctx, ctx->slot_pos, slots, -1);
    if (rc) return rc;
  } else {
    if (n > 0 && !seq_ids) return fail(ctx, MB_ERR_ARG, "mb_ring_reset: seq_ids is null");
    for (int i = 0; i < n; i++)
      if (seq_ids[i] < 0 || seq_ids[i] >= ctx->cfg.max_seqs)
        return fail(ctx, MB_ERR_ARG, "mb_ring_reset: sequence %d out of range", seq_ids[i]);
    for (int l = 0; l < ctx->cfg.n_layers; l++)
      for (int i = 0; i < n; i++) {
        int rc = launch_fill_i32(ctx, ctx->slot_pos + slot_base(ctx, l, seq_ids[i]), C, -1);
        if (rc) return rc;
      }
  }
  MB_HIP(ctx, sync_stream(ctx));
  return MB_OK;
}

int mb_ring_poison(mb_ctx* ctx, int layer, int seq, int n_slots, float sentinel) {
  MB_DEVICE_GUARD(ctx);
  int rc = check_common(ctx, layer, 0);
  if (rc) return rc;
  if (seq < 0 || seq >= ctx->cfg.max_seqs || n_slots < 0 || n_slots > ctx->cfg.capacity)
    return fail(ctx, MB_ERR_ARG, "mb_ring_poison: seq %d / n_slots %d out of range", seq, n_slots);
  const int64_t C = ctx->cfg.capacity;
  const size_t e = kv_elem_bytes(ctx);
  for (int h = 0; h < H; h++) {
    const int64_t off = ring_base(ctx, layer, seq) + (int64_t)h * C * HD;
    rc = launch_fill_kv(ctx, (char*)ctx->ring_k + off * e, (int64_t)n_slots * HD, sentinel);
    if (rc) return rc;
    rc = launch_fill_kv(ctx, (char*)ctx->ring_v + off * e, (int64_t)n_slots * HD, sentinel);
    if (rc) return rc;
  }
  MB_HIP(ctx, sync_stream(ctx));
  return MB_OK;
}

int mb_read_ring(mb_ctx* ctx, int layer, int seq, int slot0, int n, float* k, float* v,
                 int32_t* slot_pos) {
  MB_DEVICE_GUARD(ctx);
  int rc = check_common(ctx, layer, 0);
  if (rc) return rc;
  const int C = ctx->cfg.capacity;
  if (seq < 0 || seq >= ctx->cfg.max_seqs || slot0 < 0 || n < 0 || slot0 + n > C)
    return fail(ctx, MB_ERR_ARG, "mb_read_ring: seq %d slots [%d, %d) out of range", seq, slot0,
                slot0 + n);
  if (n == 0) return MB_OK;
  const size_t e = kv_elem_bytes(ctx);
  std::vector<uint8_t> host((size_t)H * n * HD * e);
  for (int which = 0; which < 2; which++) {
    float* dst = which == 0 ? k : v;
    if (!dst) continue;
    const char* src = (const char*)(which == 0 ? ctx->ring_k : ctx->ring_v);
    for (int h = 0; h < H; h++) {
      const int64_t off = ring_base(ctx, layer, seq) + ((int64_t)h * C + slot0) * HD;
      MB_HIP(ctx, hipMemcpyAsync(host.data() + (size_t)h * n * HD * e, src + off * e,
                                 (size_t)n * HD * e, hipMemcpyDeviceToHost, ctx->stream));
    }
    MB_HIP(ctx, sync_stream(ctx));
    // device [head][slot][dim] -> reference [slot][head*64 + dim]
    for (int h = 0; h < H; h++)
      for (int s = 0; s < n; s++)
        for (int d = 0; d < HD; d++) {
          const size_t i = ((size_t)h * n + s) * HD + d;
          float f;
          if (e == 2) {
            uint32_t u = (uint32_t)((const uint16_t*)host.data())[i] << 16;
            memcpy(&f, &u, 4);
          } else {
            f = ((const float*)host.data())[i];
          }
          dst[(size_t)s * D + h * HD + d] = f;
        }
  }
  if (slot_pos) {
    MB_HIP(ctx, hipMemcpyAsync(slot_pos, ctx->slot_pos + slot_base(ctx, layer, seq) + slot0,
                               (size_t)n * 4, hipMemcpyDeviceToHost, ctx->stream));
    MB_HIP(ctx, sync_stream(ctx));
  }
  return MB_OK;
}

int mb_write_ring(mb_ctx* ctx, int layer, int seq, int slot0, int n, const float* k,
                  const float* v, const int32_t* slot_pos) {
  MB_DEVICE_GUARD(ctx);
  int rc = check_common(ctx, layer, 0);
  if (rc) return rc;
  const int C = ctx->cfg.capacity;
  if (seq < 0 || seq >= ctx->cfg.max_seqs || slot0 < 0 || n < 0 || slot0 + n > C)
    return fail(ctx, MB_ERR_ARG, "mb_write_ring: seq %d slots [%d, %d) out of range", seq, slot0,
                slot0 + n);
  if (n == 0) return MB_OK;
  // Every stored position must be one the ring's own writes could have left
  // in that slot: empty (-1), or pos mod C (pos itself on a non-wrapping ring).
  if (slot_pos)
    for (int i = 0; i < n; i++) {
      const int32_t p = slot_pos[i], s = slot0 + i;
      const bool ok = p == -1 || (p >= 0 && (ctx->cfg.wrap ? p % C == s : p == s));
      if (!ok)
        return fail(ctx, MB_ERR_ARG, "mb_write_ring: position %d cannot sit in slot %d of a "
                    "%s ring of %d slots", p, s, ctx->cfg.wrap ? "wrapping" : "non-wrapping", C);
    }
  const size_t e = kv_elem_bytes(ctx);
  std::vector<uint8_t> host((size_t)H * n * HD * e);
  for (int which = 0; which < 2; which++) {
    const float* src = which == 0 ? k : v;
    if (!src) continue;
    // reference [slot][head*64 + dim] -> device [head][slot][dim]
    for (int h = 0; h < H; h++)
      for (int s = 0; s < n; s++)
        for (int d = 0; d < HD; d++) {
          const size_t i = ((size_t)h * n + s) * HD + d;
          const float f = src[(size_t)s * D + h * HD + d];
          if (e == 2) ((uint16_t*)host.data())[i] = f32_to_bf16(f);  // the kernels' rounding
          else ((float*)host.data())[i] = f;
        }
    char* dst = (char*)(which == 0 ? ctx->ring_k : ctx->ring_v);
    for (int h = 0; h < H; h++) {
      const int64_t off = ring_base(ctx, layer, seq) + ((int64_t)h * C + slot0) * HD;
      MB_HIP(ctx, hipMemcpyAsync(dst + off * e, host.data() + (size_t)h * n * HD * e,
                                 (size_t)n * HD * e, hipMemcpyHostToDevice, ctx->stream));
    }
    MB_HIP(ctx, sync_stream(ctx));
  }
  if (slot_pos) {
    MB_HIP(ctx, hipMemcpyAsync(ctx->slot_pos + slot_base(ctx, layer, seq) + slot0, slot_pos,
                               (size_t)n * 4, hipMemcpyHostToDevice, ctx->stream));
    MB_HIP(ctx, sync_stream(ctx));
  }
  return MB_OK;
}

int mb_ring_write_rows_dev(mb_ctx* ctx, int layer, int B, int rows_max, const void* qkv,
                           int qkv_dtype, const int32_t* pos0, const int32_t* n_rows, void* q_out,
                           int q_dtype) {
  MB_DEVICE_GUARD(ctx);
  int rc = check_common(ctx, layer, B);
  if (rc) return rc;
  if (rows_max < 1 || rows_max > ctx->cfg.max_rows)
    return fail(ctx, MB_ERR_ARG, "rows_max %d out of [1, %d]", rows_max, ctx->cfg.max_rows);
  if ((qkv_dtype != MB_DT_F32 && qkv_dtype != MB_DT_BF16) ||
      (q_dtype != MB_DT_F32 && q_dtype != MB_DT_BF16))
    return fail(ctx, MB_ERR_ARG, "unknown dtype");
  if (B == 0) return MB_OK;
  if (!qkv || !pos0 || !n_rows) return fail(ctx, MB_ERR_ARG, "null pointer");
  return launch_ring_write(ctx, global_ring(ctx, layer), B, rows_max, qkv, qkv_dtype,
                           dense_rows(QKV, rows_max), pos0, n_rows, q_out, q_dtype,
                           dense_rows(D, rows_max));
}

int mb_ring_append_dev(mb_ctx* ctx, int layer, int B, const void* qkv, int qkv_dtype,
                       int64_t qkv_stride, const int32_t* pos, float* q_out, int64_t q_stride) {
  MB_DEVICE_GUARD(ctx);
  int rc = check_common(ctx, layer, B);
  if (rc) return rc;
  if (qkv_dtype != MB_DT_F32 && qkv_dtype != MB_DT_BF16)
    return fail(ctx, MB_ERR_ARG, "unknown dtype");
  if (qkv_stride < QKV || (q_out && q_stride < D))
    return fail(ctx, MB_ERR_ARG, "row stride too small");
  if (B == 0) return MB_OK;
  if (!qkv || !pos) return fail(ctx, MB_ERR_ARG, "null pointer");
  return launch_ring_write(ctx, global_ring(ctx, layer), B, 1, qkv, qkv_dtype,
                           dense_rows(qkv_stride, 1), pos, nullptr, q_out, MB_DT_F32,
                           dense_rows(q_stride, 1));
}

int mb_decode_attention_dev(mb_ctx* ctx, int layer, int B, const float* q, int64_t q_stride,
                            const int32_t* pos, int32_t max_pos, float* out, int64_t out_stride) {
  MB_DEVICE_GUARD(ctx);
  int rc = check_common(ctx, layer, B);
  if (rc) return rc;
  if (q_stride < D || out_stride < D) return fail(ctx, MB_ERR_ARG, "row stride too small");
  if (max_pos < 0) return fail(ctx, MB_ERR_ARG, "max_pos %d is negative", max_pos);
  if (B == 0) return MB_OK;
  if (!q || !pos || !out) return fail(ctx, MB_ERR_ARG, "null pointer");
  return launch_attn(ctx, global_ring(ctx, layer), B, 1, q, dense_rows(q_stride, 1), pos, nullptr,
                     (int64_t)max_pos + 1, out, dense_rows(out_stride, 1), claim_split(ctx));
}

int mb_append_attend_dev(mb_ctx* ctx, int layer, int B, const void* qkv, int qkv_dtype,
                         int64_t qkv_stride, const int32_t* pos, int32_t max_pos, float* q_out,
                         int64_t q_stride, float* out, int64_t out_stride) {
  MB_DEVICE_GUARD(ctx);
  int rc = check_common(ctx, layer, B);
  if (rc) return rc;
  if (qkv_dtype != MB_DT_F32 && qkv_dtype != MB_DT_BF16)
    return fail(ctx, MB_ERR_ARG, "unknown dtype");
  if (qkv_stride < QKV || out_stride < D || (q_out && q_stride < D))
    return fail(ctx, MB_ERR_ARG, "row stride too small");
  if (max_pos < 0) return fail(ctx, MB_ERR_ARG, "max_pos %d is negative", max_pos);
  if (!ctx->cfg.wrap && max_pos >= ctx->cfg.capacity)
    return fail(ctx, MB_ERR_RANGE,
                "decode position %d exceeds the KV ring (%d slots); it must be sized "
                "prefill_rows + max_new_frames",
                max_pos, ctx->cfg.capacity);
  if (B == 0) return MB_OK;
  if (!qkv || !pos || !out) return fail(ctx, MB_ERR_ARG, "null pointer");
  return launch_append_attn(ctx, global_ring(ctx, layer), B, qkv, qkv_dtype,
                            dense_rows(qkv_stride, 1), pos, (int64_t)max_pos + 1, q_out,
                            dense_rows(q_stride, 1), out, dense_rows(out_stride, 1), -1,
                            claim_split(ctx));
}

int mb_prefill_attention_dev(mb_ctx* ctx, int layer, int B, int rows_max, const void* q,
                             int q_dtype, const int32_t* pos0, const int32_t* n_rows, float* out) {
  MB_DEVICE_GUARD(ctx);
  int rc = check_common(ctx, layer, B);
  if (rc) return rc;
  if (rows_max < 1 || rows_max > ctx->cfg.max_rows)
    return fail(ctx, MB_ERR_ARG, "rows_max %d out of [1, %d]", rows_max, ctx->cfg.max_rows);
  if (q_dtype != MB_DT_F32 && q_dtype != MB_DT_BF16) return fail(ctx, MB_ERR_ARG, "unknown dtype");
  if (B == 0) return MB_OK;
  if (!q || !pos0 || !n_rows || !out) return fail(ctx, MB_ERR_ARG, "null pointer");
  return launch_prefill_attention(ctx, global_ring(ctx, layer), B, rows_max, q, q_dtype,
                                  dense_rows(D, rows_max), pos0, n_rows, out,
                                  dense_rows(D, rows_max));
}

// ------------------------------------------- several hypotheses per voice

int mb_ring_view(mb_ctx* ctx, void** k, void** v, int32_t** slot_pos) {
  if (!ctx) return MB_ERR_ARG;
  if (k) *k = ctx->ring_k;
  if (v) *v = ctx->ring_v;
  if (slot_pos) *slot_pos = ctx->slot_pos;
  return MB_OK;
}

int mb_tree_attention_work(mb_ctx* ctx, int B, int rows_max, int32_t max_pos, int64_t* bytes) {
  int rc = check_tree(ctx, 0, 1, B, rows_max);
  if (rc) return rc;
  if (max_pos < 0) return fail(ctx, MB_ERR_ARG, "max_pos %d is negative", max_pos);
  if (!bytes) return fail(ctx, MB_ERR_ARG, "null pointer");
  *bytes = tree_work_bytes(ctx, B, rows_max, max_pos);
  return MB_OK;
}

int mb_tree_attention_dev(mb_ctx* ctx, int layer, int B, int rows_max, const void* qkv,
                          int qkv_dtype, int64_t qkv_stride, const int32_t* parent,
                          const int32_t* pos0, const int32_t* n_nodes, int32_t max_pos, float* out,
                          int64_t out_stride, void* work, int64_t work_bytes) {
  MB_DEVICE_GUARD(ctx);
  int rc = check_tree(ctx, layer, 1, B, rows_max);
  if (rc) return rc;
  if (qkv_dtype != MB_DT_F32 && qkv_dtype != MB_DT_BF16)
    return fail(ctx, MB_ERR_ARG, "unknown dtype");
  if (qkv_stride < QKV || out_stride < D) return fail(ctx, MB_ERR_ARG, "row stride too small");
  if (max_pos < 0) return fail(ctx, MB_ERR_ARG, "max_pos %d is negative", max_pos);
  if (!ctx->cfg.wrap && max_pos >= ctx->cfg.capacity)
    return fail(ctx, MB_ERR_RANGE,
                "decode position %d exceeds the KV ring (%d slots); it must be sized "
                "prefill_rows + max_new_frames",
                max_pos, ctx->cfg.capacity);
  if (B == 0) return MB_OK;
  if (!qkv || !parent || !pos0 || !out) return fail(ctx, MB_ERR_ARG, "null pointer");
  if (!aligned_rows(qkv, qkv_stride, qkv_dtype == MB_DT_BF16 ? 2 : 4) || !aligned_rows(out, out_stride, 4))
    return fail(ctx, MB_ERR_ARG, "rows must start at multiples of 16 bytes");
  rc = check_work(ctx, work, work_bytes, tree_work_bytes(ctx, B, rows_max, max_pos));
  if (rc) return rc;
  const int64_t n = (int64_t)B * rows_max - 1, in = qkv_stride * (qkv_dtype == MB_DT_BF16 ? 2 : 4),
                row = QKV * (qkv_dtype == MB_DT_BF16 ? 2 : 4);
  if (overlap(qkv, n * in + row, out, (n * out_stride + D) * 4)) {
    // rows that lie between one another are right
    const int64_t at = (((intptr_t)out - (intptr_t)qkv) % in + in) % in;
    if (in != out_stride * 4 || at < row || at + D * 4 > in)
      return fail(ctx, MB_ERR_ARG, "out overlaps qkv");
  }
  return launch_tree_attention(ctx, global_ring(ctx, layer), B, rows_max, qkv, qkv_dtype, qkv_stride,
                               parent, pos0, n_nodes, max_pos, out, out_stride, work);
}

int mb_tree_commit_dev(mb_ctx* ctx, int layer0, int n_layers, int B, int rows_max, const void* qkv,
                       int qkv_dtype, int64_t qkv_stride, int64_t layer_stride,
                       const int32_t* pos0, int path_max, const int32_t* path,
                       const int32_t* n_path) {
  MB_DEVICE_GUARD(ctx);
  int rc = check_tree(ctx, layer0, n_layers, B, rows_max);
  if (rc) return rc;
  if (qkv_dtype != MB_DT_F32 && qkv_dtype != MB_DT_BF16)
    return fail(ctx, MB_ERR_ARG, "unknown dtype");
  if (qkv_stride < QKV) return fail(ctx, MB_ERR_ARG, "row stride too small");
  if (path_max < 0) return fail(ctx, MB_ERR_ARG, "path_max %d is negative", path_max);
  if (B == 0 || n_layers == 0 || path_max == 0) return MB_OK;
  if (!qkv || !pos0 || !path) return fail(ctx, MB_ERR_ARG, "null pointer");
  const int e = qkv_dtype == MB_DT_BF16 ? 2 : 4;
  if (!aligned_rows(qkv, qkv_stride, e) || (n_layers > 1 && !aligned_rows(qkv, layer_stride, e)))
    return fail(ctx, MB_ERR_ARG, "rows must start at multiples of 16 bytes");
  if (n_layers > 1 && layer_stride < (int64_t)B * rows_max * qkv_stride)
    return fail(ctx, MB_ERR_ARG, "layer stride too small");
  return launch_tree_commit(ctx, layer0, n_layers, B, rows_max, qkv, qkv_dtype, qkv_stride,
                            layer_stride, pos0, path_max, path, n_path);
}

int mb_beam_select_work(mb_ctx* ctx, int B, int width, int vocab, int n_out, int64_t* bytes) {
  int rc = check_beam(ctx, B, width, vocab, n_out);
  if (rc) return rc;
  if (!bytes) return fail(ctx, MB_ERR_ARG, "null pointer");
  *bytes = beam_work_bytes(B, width, vocab, n_out);
  return MB_OK;
}

int mb_beam_select_dev(mb_ctx* ctx, int B, int width, int vocab, int n_out, const void* logits,
                       int logits_dtype, int64_t logits_stride, const float* scores,
                       const int32_t* done, int32_t end_id, const uint32_t* seen, double penalty,
                       float* scores_out, int32_t* parent, int32_t* token, int32_t* done_out,
                       uint32_t* seen_out, void* work, int64_t work_bytes) {
  MB_DEVICE_GUARD(ctx);
  int rc = check_beam(ctx, B, width, vocab, n_out);
  if (rc) return rc;
  if (logits_dtype != MB_DT_F32 && logits_dtype != MB_DT_BF16)
    return fail(ctx, MB_ERR_ARG, "unknown dtype");
  if (logits_stride < vocab) return fail(ctx, MB_ERR_ARG, "row stride too small");
  rc = check_beam_options(ctx, B, width, vocab, n_out, scores, done, end_id, seen, penalty, scores_out,
                          done_out, seen_out);
  if (rc) return rc;
  if (B == 0) return MB_OK;
  if (!logits || !scores || !scores_out || !parent || !token)
    return fail(ctx, MB_ERR_ARG, "null pointer");
  rc = check_work(ctx, work, work_bytes, beam_work_bytes(B, width, vocab, n_out));
  if (rc) return rc;
  return launch_beam_select(ctx, B, width, vocab, n_out, logits, logits_dtype, logits_stride, scores,
                            done, end_id, seen, penalty, scores_out, parent, token, done_out,
                            seen_out, work);
}

int mb_ring_reorder_dev(mb_ctx* ctx, int layer0, int n_layers, int B, int width,
                        const int32_t* parent, const int32_t* pos_from, const int32_t* pos_to,
                        int32_t max_rows) {
  MB_DEVICE_GUARD(ctx);
  int rc = check_groups(ctx, layer0, n_layers, B, width, pos_from, pos_to);
  if (rc) return rc;
  if (max_rows < 0) return fail(ctx, MB_ERR_ARG, "max_rows %d is negative", max_rows);
  if (B == 0 || n_layers == 0 || (max_rows == 0 && pos_from)) return MB_OK;
  if (!parent) return fail(ctx, MB_ERR_ARG, "null pointer");
  return launch_ring_reorder(ctx, layer0, n_layers, B, width, parent, pos_from, pos_to,
                             pos_from ? max_rows : ctx->cfg.capacity);
}

int mb_linear_dev(mb_ctx* ctx, int M, int N, int K, const float* A, int64_t lda, const float* W,
                  const float* bias, float* C, int64_t ldc, int epi) {
  MB_DEVICE_GUARD(ctx);
  if (!ctx) return MB_ERR_ARG;
  if (M < 0 || N < 1 || K < 1) return fail(ctx, MB_ERR_ARG, "linear shape M %d N %d K %d", M, N, K);
  if (epi < EPI_STORE || epi > EPI_GELU_ERF) return fail(ctx, MB_ERR_ARG, "unknown epilogue %d", epi);
  if (epi == EPI_SCALE_ADD && !bias)
    return fail(ctx, MB_ERR_ARG, "MB_EPI_SCALE_ADD needs the scale vector in `bias`");
  if (M == 0) return MB_OK;
  if (!A || !W || !C) return fail(ctx, MB_ERR_ARG, "null pointer");
  if (lda < K || ldc < N) return fail(ctx, MB_ERR_ARG, "leading dimension below the row width");
  return launch_gemm(ctx, epi, A, lda, W, N, K, bias, C, ldc, M);
}

int mb_split_weights_dev(mb_ctx* ctx, const float* W, int K, int N, void* Wx) {
  MB_DEVICE_GUARD(ctx);
  if (!ctx) return MB_ERR_ARG;
  if (K < 1 || N < 1) return fail(ctx, MB_ERR_ARG, "split weights shape K %d N %d", K, N);
  if (!W || !Wx) return fail(ctx, MB_ERR_ARG, "null pointer");
  if (((uintptr_t)Wx & 15)) return fail(ctx, MB_ERR_ARG, "Wx must be 16-byte aligned");
  return launch_split_w(ctx, W, K, N, Wx, false);
}

int mb_linear_split_dev(mb_ctx* ctx, int M, int N, int K, const float* A, int64_t lda,
                        const void* Wx, const float* bias, float* C, int64_t ldc, int epi) {
  MB_DEVICE_GUARD(ctx);
  if (!ctx) return MB_ERR_ARG;
  if (M < 0 || N < 1 || K < 1) return fail(ctx, MB_ERR_ARG, "linear shape M %d N %d K %d", M, N, K);
  if (epi < EPI_STORE || epi > EPI_GELU_ERF) return fail(ctx, MB_ERR_ARG, "unknown epilogue %d", epi);
  if (epi == EPI_SCALE_ADD && !bias)
    return fail(ctx, MB_ERR_ARG, "MB_EPI_SCALE_ADD needs the scale vector in `bias`");
  if (M == 0) return MB_OK;
  if (!A || !Wx || !C) return fail(ctx, MB_ERR_ARG, "null pointer");
  if (lda < K || ldc < N) return fail(ctx, MB_ERR_ARG, "leading dimension below the row width");
  return launch_gemm_x3(ctx, epi, A, lda, Wx, N, K, bias, C, ldc, M, nullptr, nullptr);
}

// ---------------------------------------------------------- host pointers

int mb_ring_write_rows(mb_ctx* ctx, int layer, int B, int rows_max, const float* qkv,
                       const int32_t* pos0, const int32_t* n_rows, float* q_out) {
  MB_DEVICE_GUARD(ctx);
  int rc = check_common(ctx, layer, B);
  if (rc) return rc;
  if (rows_max < 1 || rows_max > ctx->cfg.max_rows)
    return fail(ctx, MB_ERR_ARG, "rows_max %d out of [1, %d]", rows_max, ctx->cfg.max_rows);
  if (B == 0) return MB_OK;
  if (!qkv || !pos0 || !n_rows) return fail(ctx, MB_ERR_ARG, "null pointer");
  rc = check_positions(ctx, B, pos0, n_rows, rows_max);
  if (rc) return rc;
  const size_t rows = (size_t)B * rows_max;
  float* d_qkv = (float*)scratch(ctx, "qkv", rows * QKV * 4);
  float* d_q = (float*)scratch(ctx, "q", rows * D * 4);
  int32_t* d_pos = (int32_t*)scratch(ctx, "pos", (size_t)B * 8);
  if (!d_qkv || !d_q || !d_pos) return fail(ctx, MB_ERR_NOMEM, "staging allocation failed");
  MB_HIP(ctx, hipMemcpyAsync(d_qkv, qkv, rows * QKV * 4, hipMemcpyHostToDevice, ctx->stream));
  MB_HIP(ctx, hipMemcpyAsync(d_pos, pos0, (size_t)B * 4, hipMemcpyHostToDevice, ctx->stream));
  MB_HIP(ctx, hipMemcpyAsync(d_pos + B, n_rows, (size_t)B * 4, hipMemcpyHostToDevice, ctx->stream));
  rc = launch_ring_write(ctx, global_ring(ctx, layer), B, rows_max, d_qkv, MB_DT_F32,
                         dense_rows(QKV, rows_max), d_pos, d_pos + B, q_out ? d_q : nullptr,
                         MB_DT_F32, dense_rows(D, rows_max));
  if (rc) return rc;
  if (q_out) MB_HIP(ctx, hipMemcpyAsync(q_out, d_q, rows * D * 4, hipMemcpyDeviceToHost, ctx->stream));
  MB_HIP(ctx, sync_stream(ctx));
  return MB_OK;
}

int mb_ring_append(mb_ctx* ctx, int layer, int B, const float* qkv, const int32_t* pos,
                   float* q_out) {
  MB_DEVICE_GUARD(ctx);
  int rc = check_common(ctx, layer, B);
  if (rc) return rc;
  if (B == 0) return MB_OK;
  if (!qkv || !pos) return fail(ctx, MB_ERR_ARG, "null pointer");
  rc = check_positions(ctx, B, pos, nullptr, 1);
  if (rc) return rc;
  float* d_qkv = (float*)scratch(ctx, "qkv", (size_t)B * QKV * 4);
  float* d_q = (float*)scratch(ctx, "q", (size_t)B * D * 4);
  int32_t* d_pos = (int32_t*)scratch(ctx, "pos", (size_t)B * 8);
  if (!d_qkv || !d_q || !d_pos) return fail(ctx, MB_ERR_NOMEM, "staging allocation failed");
  MB_HIP(ctx, hipMemcpyAsync(d_qkv, qkv, (size_t)B * QKV * 4, hipMemcpyHostToDevice, ctx->stream));
  MB_HIP(ctx, hipMemcpyAsync(d_pos, pos, (size_t)B * 4, hipMemcpyHostToDevice, ctx->stream));
  rc = launch_ring_write(ctx, global_ring(ctx, layer), B, 1, d_qkv, MB_DT_F32, dense_rows(QKV, 1),
                         d_pos, nullptr, q_out ? d_q : nullptr, MB_DT_F32, dense_rows(D, 1));
  if (rc) return rc;
  if (q_out) MB_HIP(ctx, hipMemcpyAsync(q_out, d_q, (size_t)B * D * 4, hipMemcpyDeviceToHost, ctx->stream));
  MB_HIP(ctx, sync_stream(ctx));
  return MB_OK;
}

int mb_decode_attention(mb_ctx* ctx, int layer, int B, const float* q, const int32_t* pos,
                        float* out) {
  MB_DEVICE_GUARD(ctx);
  int rc = check_common(ctx, layer, B);
  if (rc) return rc;
  if (B == 0) return MB_OK;
  if (!q || !pos || !out) return fail(ctx, MB_ERR_ARG, "null pointer");
  int32_t max_pos = 0;
  for (int b = 0; b < B; b++) {
    if (pos[b] < 0) return fail(ctx, MB_ERR_ARG, "sequence %d: negative position %d", b, pos[b]);
    if (pos[b] > max_pos) max_pos = pos[b];
  }
  float* d_q = (float*)scratch(ctx, "q", (size_t)B * D * 4);
  float* d_out = (float*)scratch(ctx, "out", (size_t)B * D * 4);
  int32_t* d_pos = (int32_t*)scratch(ctx, "pos", (size_t)B * 8);
  if (!d_q || !d_out || !d_pos) return fail(ctx, MB_ERR_NOMEM, "staging allocation failed");
  MB_HIP(ctx, hipMemcpyAsync(d_q, q, (size_t)B * D * 4, hipMemcpyHostToDevice, ctx->stream));
  MB_HIP(ctx, hipMemcpyAsync(d_pos, pos, (size_t)B * 4, hipMemcpyHostToDevice, ctx->stream));
  rc = launch_attn(ctx, global_ring(ctx, layer), B, 1, d_q, dense_rows(D, 1), d_pos, nullptr,
                   (int64_t)max_pos + 1, d_out, dense_rows(D, 1), claim_split(ctx));
  if (rc) return rc;
  MB_HIP(ctx, hipMemcpyAsync(out, d_out, (size_t)B * D * 4, hipMemcpyDeviceToHost, ctx->stream));
  MB_HIP(ctx, sync_stream(ctx));
  return MB_OK;
}

int mb_append_attend(mb_ctx* ctx, int layer, int B, const float* qkv, const int32_t* pos,
                     float* q_out, float* out) {
  MB_DEVICE_GUARD(ctx);
  int rc = check_common(ctx, layer, B);
  if (rc) return rc;
  if (B == 0) return MB_OK;
  if (!qkv || !pos || !out) return fail(ctx, MB_ERR_ARG, "null pointer");
  rc = check_positions(ctx, B, pos, nullptr, 1);
  if (rc) return rc;
  int32_t max_pos = 0;
  for (int b = 0; b < B; b++) max_pos = pos[b] > max_pos ? pos[b] : max_pos;
  float* d_qkv = (float*)scratch(ctx, "qkv", (size_t)B * QKV * 4);
  float* d_q = (float*)scratch(ctx, "q", (size_t)B * D * 4);
  float* d_out = (float*)scratch(ctx, "out", (size_t)B * D * 4);
  int32_t* d_pos = (int32_t*)scratch(ctx, "pos", (size_t)B * 8);
  if (!d_qkv || !d_q || !d_out || !d_pos) return fail(ctx, MB_ERR_NOMEM, "staging allocation failed");
  MB_HIP(ctx, hipMemcpyAsync(d_qkv, qkv, (size_t)B * QKV * 4, hipMemcpyHostToDevice, ctx->stream));
  MB_HIP(ctx, hipMemcpyAsync(d_pos, pos, (size_t)B * 4, hipMemcpyHostToDevice, ctx->stream));
  rc = launch_append_attn(ctx, global_ring(ctx, layer), B, d_qkv, MB_DT_F32, dense_rows(QKV, 1),
                          d_pos, (int64_t)max_pos + 1, q_out ? d_q : nullptr, dense_rows(D, 1),
                          d_out, dense_rows(D, 1), -1, claim_split(ctx));
  if (rc) return rc;
  if (q_out) MB_HIP(ctx, hipMemcpyAsync(q_out, d_q, (size_t)B * D * 4, hipMemcpyDeviceToHost, ctx->stream));
  MB_HIP(ctx, hipMemcpyAsync(out, d_out, (size_t)B * D * 4, hipMemcpyDeviceToHost, ctx->stream));
  MB_HIP(ctx, sync_stream(ctx));
  return MB_OK;
}

int mb_prefill_attention(mb_ctx* ctx, int layer, int B, int rows_max, const float* q,
                         const int32_t* pos0, const int32_t* n_rows, float* out) {
  MB_DEVICE_GUARD(ctx);
  int rc = check_common(ctx, layer, B);
  if (rc) return rc;
  if (rows_max < 1 || rows_max > ctx->cfg.max_rows)
    return fail(ctx, MB_ERR_ARG, "rows_max %d out of [1, %d]", rows_max, ctx->cfg.max_rows);
  if (B == 0) return MB_OK;
  if (!q || !pos0 || !n_rows || !out) return fail(ctx, MB_ERR_ARG, "null pointer");
  rc = check_positions(ctx, B, pos0, n_rows, rows_max);
  if (rc) return rc;
  const size_t rows = (size_t)B * rows_max;
  float* d_q = (float*)scratch(ctx, "q", rows * D * 4);
  float* d_out = (float*)scratch(ctx, "out", rows * D * 4);
  int32_t* d_pos = (int32_t*)scratch(ctx, "pos", (size_t)B * 8);
  if (!d_q || !d_out || !d_pos) return fail(ctx, MB_ERR_NOMEM, "staging allocation failed");
  MB_HIP(ctx, hipMemcpyAsync(d_q, q, rows * D * 4, hipMemcpyHostToDevice, ctx->stream));
  MB_HIP(ctx, hipMemcpyAsync(d_pos, pos0, (size_t)B * 4, hipMemcpyHostToDevice, ctx->stream));
  MB_HIP(ctx, hipMemcpyAsync(d_pos + B, n_rows, (size_t)B * 4, hipMemcpyHostToDevice, ctx->stream));
  rc = launch_prefill_attention(ctx, global_ring(ctx, layer), B, rows_max, d_q, MB_DT_F32,
                                dense_rows(D, rows_max), d_pos, d_pos + B, d_out,
                                dense_rows(D, rows_max));
  if (rc) return rc;
  MB_HIP(ctx, hipMemcpyAsync(out, d_out, rows * D * 4, hipMemcpyDeviceToHost, ctx->stream));
  MB_HIP(ctx, sync_stream(ctx));
  return MB_OK;
}

int mb_tree_attention(mb_ctx* ctx, int layer, int B, int rows_max, const float* qkv,
                      const int32_t* parent, const int32_t* pos0, const int32_t* n_nodes, float* out) {
  MB_DEVICE_GUARD(ctx);
  int rc = check_tree(ctx, layer, 1, B, rows_max);
  if (rc) return rc;
  if (B == 0) return MB_OK;
  if (!qkv || !parent || !pos0 || !n_nodes || !out) return fail(ctx, MB_ERR_ARG, "null pointer");
  int32_t max_pos = 0;
  for (int b = 0; b < B; b++) {
    if (n_nodes[b] < 0 || n_nodes[b] > rows_max)
      return fail(ctx, MB_ERR_ARG, "sequence %d: %d nodes out of [0, %d]", b, n_nodes[b], rows_max);
    if (pos0[b] < 0 || pos0[b] > INT32_MAX - kTreeMaxNodes)
      return fail(ctx, MB_ERR_ARG, "sequence %d: position %d out of range", b, pos0[b]);
    int depth[kTreeMaxNodes];
    for (int i = 0; i < n_nodes[b]; i++) {
      const int32_t p = parent[(size_t)b * rows_max + i];
      if (p < -1 || p >= i)
        return fail(ctx, MB_ERR_ARG, "sequence %d: parent %d of node %d is no earlier node", b, p, i);
      depth[i] = p < 0 ? 0 : depth[p] + 1;
      const int32_t pos = pos0[b] + depth[i];
      if (!ctx->cfg.wrap && pos >= ctx->cfg.capacity)
        return fail(ctx, MB_ERR_RANGE,
                    "decode position %d exceeds the KV ring (%d slots); it must be sized "
                    "prefill_rows + max_new_frames",
                    pos, ctx->cfg.capacity);
      max_pos = std::max(max_pos, pos);
    }
  }
  const size_t rows = (size_t)B * rows_max;
  const int64_t need = tree_work_bytes(ctx, B, rows_max, max_pos);
  float* d_qkv = (float*)scratch(ctx, "qkv", rows * QKV * 4);
  float* d_out = (float*)scratch(ctx, "out", rows * D * 4);
  int32_t* d_pos = (int32_t*)scratch(ctx, "pos", ((size_t)B * 2 + rows) * 4);
  void* d_work = need ? scratch(ctx, "tree_work", (size_t)need) : nullptr;
  if (!d_qkv || !d_out || !d_pos || (need && !d_work))
    return fail(ctx, MB_ERR_NOMEM, "staging allocation failed");
  MB_HIP(ctx, hipMemcpyAsync(d_qkv, qkv, rows * QKV * 4, hipMemcpyHostToDevice, ctx->stream));
  MB_HIP(ctx, hipMemcpyAsync(d_pos, pos0, (size_t)B * 4, hipMemcpyHostToDevice, ctx->stream));
  MB_HIP(ctx, hipMemcpyAsync(d_pos + B, n_nodes, (size_t)B * 4, hipMemcpyHostToDevice, ctx->stream));
  MB_HIP(ctx, hipMemcpyAsync(d_pos + 2 * B, parent, rows * 4, hipMemcpyHostToDevice, ctx->stream));
  rc = launch_tree_attention(ctx, global_ring(ctx, layer), B, rows_max, d_qkv, MB_DT_F32, QKV,
                             d_pos + 2 * B, d_pos, d_pos + B, max_pos, d_out, D, d_work);
  if (rc) return rc;
  // only the rows that were attended: the others stay as the caller has them
  for (int b = 0; b < B; b++)
    if (n_nodes[b])
      MB_HIP(ctx, hipMemcpyAsync(out + (size_t)b * rows_max * D, d_out + (size_t)b * rows_max * D,
                                 (size_t)n_nodes[b] * D * 4, hipMemcpyDeviceToHost, ctx->stream));
  MB_HIP(ctx, sync_stream(ctx));
  return MB_OK;
}

int mb_tree_commit(mb_ctx* ctx, int layer0, int n_layers, int B, int rows_max, const float* qkv,
                   const int32_t* pos0, int path_max, const int32_t* path, const int32_t* n_path) {
  MB_DEVICE_GUARD(ctx);
  int rc = check_tree(ctx, layer0, n_layers, B, rows_max);
  if (rc) return rc;
  if (path_max < 0) return fail(ctx, MB_ERR_ARG, "path_max %d is negative", path_max);
  if (B == 0 || n_layers == 0 || path_max == 0) return MB_OK;
  if (!qkv || !pos0 || !path || !n_path) return fail(ctx, MB_ERR_ARG, "null pointer");
  for (int b = 0; b < B; b++) {
    if (pos0[b] < 0) return fail(ctx, MB_ERR_ARG, "sequence %d: negative position %d", b, pos0[b]);
    if (n_path[b] < 0 || n_path[b] > path_max)
      return fail(ctx, MB_ERR_ARG, "sequence %d: a path of %d rows out of [0, %d]", b, n_path[b], path_max);
    const int64_t last = (int64_t)pos0[b] + n_path[b] - 1;
    if (last > INT32_MAX - 1) return fail(ctx, MB_ERR_ARG, "sequence %d: position overflow", b);
    if (!ctx->cfg.wrap && n_path[b] > 0 && last >= ctx->cfg.capacity)
      return fail(ctx, MB_ERR_RANGE,
                  "decode position %lld exceeds the KV ring (%d slots); it must be sized "
                  "prefill_rows + max_new_frames",
                  (long long)last, ctx->cfg.capacity);
    for (int i = 0; i < n_path[b]; i++) {
      const int32_t node = path[(size_t)b * path_max + i];
      if (node < 0 || node >= rows_max)
        return fail(ctx, MB_ERR_ARG, "sequence %d: path node %d out of [0, %d)", b, node, rows_max);
    }
  }
  const size_t rows = (size_t)n_layers * B * rows_max;
  float* d_qkv = (float*)scratch(ctx, "qkv", rows * QKV * 4);
  int32_t* d_pos = (int32_t*)scratch(ctx, "pos", ((size_t)B * (2 + (size_t)path_max)) * 4);
  if (!d_qkv || !d_pos) return fail(ctx, MB_ERR_NOMEM, "staging allocation failed");
  MB_HIP(ctx, hipMemcpyAsync(d_qkv, qkv, rows * QKV * 4, hipMemcpyHostToDevice, ctx->stream));
  MB_HIP(ctx, hipMemcpyAsync(d_pos, pos0, (size_t)B * 4, hipMemcpyHostToDevice, ctx->stream));
  MB_HIP(ctx, hipMemcpyAsync(d_pos + B, n_path, (size_t)B * 4, hipMemcpyHostToDevice, ctx->stream));
  MB_HIP(ctx, hipMemcpyAsync(d_pos + 2 * B, path, (size_t)B * path_max * 4, hipMemcpyHostToDevice, ctx->stream));
  rc = launch_tree_commit(ctx, layer0, n_layers, B, rows_max, d_qkv, MB_DT_F32, QKV,
                          (int64_t)B * rows_max * QKV, d_pos, path_max, d_pos + 2 * B, d_pos + B);
  if (rc) return rc;
  MB_HIP(ctx, sync_stream(ctx));
  return MB_OK;
}

int mb_beam_select(mb_ctx* ctx, int B, int width, int vocab, int n_out, const float* logits,
                   const float* scores, const int32_t* done, int32_t end_id, const uint32_t* seen,
                   double penalty, float* scores_out, int32_t* parent, int32_t* token,
                   int32_t* done_out, uint32_t* seen_out) {
  MB_DEVICE_GUARD(ctx);
  int rc = check_beam(ctx, B, width, vocab, n_out);
  if (rc) return rc;
  rc = check_beam_options(ctx, B, width, vocab, n_out, scores, done, end_id, seen, penalty, scores_out,
                          done_out, seen_out);
  if (rc) return rc;
  if (B == 0) return MB_OK;
  if (!logits || !scores || !scores_out || !parent || !token)
    return fail(ctx, MB_ERR_ARG, "null pointer");
  const size_t rows = (size_t)B * width, outs = (size_t)B * n_out, words = ((size_t)vocab + 31) / 32;
  const int64_t need = beam_work_bytes(B, width, vocab, n_out);
  float* d_logits = (float*)scratch(ctx, "beam_logits", rows * vocab * 4);
  // scores and done, then the outputs
  int32_t* d_in = (int32_t*)scratch(ctx, "beam_in", rows * 8);
  int32_t* d_out = (int32_t*)scratch(ctx, "beam_out", outs * 16);
  uint32_t* d_seen = seen ? (uint32_t*)scratch(ctx, "beam_seen", (rows + outs) * words * 4) : nullptr;
  void* d_work = need ? scratch(ctx, "beam_work", (size_t)need) : nullptr;
  if (!d_logits || !d_in || !d_out || (seen && !d_seen) || (need && !d_work))
    return fail(ctx, MB_ERR_NOMEM, "staging allocation failed");
  MB_HIP(ctx, hipMemcpyAsync(d_logits, logits, rows * vocab * 4, hipMemcpyHostToDevice, ctx->stream));
  MB_HIP(ctx, hipMemcpyAsync(d_in, scores, rows * 4, hipMemcpyHostToDevice, ctx->stream));
  if (done) MB_HIP(ctx, hipMemcpyAsync(d_in + rows, done, rows * 4, hipMemcpyHostToDevice, ctx->stream));
  if (seen) MB_HIP(ctx, hipMemcpyAsync(d_seen, seen, rows * words * 4, hipMemcpyHostToDevice, ctx->stream));
  uint32_t* d_seen_out = seen_out ? d_seen + rows * words : nullptr;
  rc = launch_beam_select(ctx, B, width, vocab, n_out, d_logits, MB_DT_F32, vocab, (float*)d_in,
                          done ? d_in + rows : nullptr, end_id, d_seen, penalty, (float*)d_out,
                          d_out + outs, d_out + 2 * outs, d_out + 3 * outs, d_seen_out, d_work);
  if (rc) return rc;
  MB_HIP(ctx, hipMemcpyAsync(scores_out, d_out, outs * 4, hipMemcpyDeviceToHost, ctx->stream));
  MB_HIP(ctx, hipMemcpyAsync(parent, d_out + outs, outs * 4, hipMemcpyDeviceToHost, ctx->stream));
  MB_HIP(ctx, hipMemcpyAsync(token, d_out + 2 * outs, outs * 4, hipMemcpyDeviceToHost, ctx->stream));
  if (done_out)
    MB_HIP(ctx, hipMemcpyAsync(done_out, d_out + 3 * outs, outs * 4, hipMemcpyDeviceToHost, ctx->stream));
  if (seen_out)
    MB_HIP(ctx, hipMemcpyAsync(seen_out, d_seen_out, outs * words * 4, hipMemcpyDeviceToHost, ctx->stream));
  MB_HIP(ctx, sync_stream(ctx));
  return MB_OK;
}

int mb_ring_reorder(mb_ctx* ctx, int layer0, int n_layers, int B, int width, const int32_t* parent,
                    const int32_t* pos_from, const int32_t* pos_to) {
  MB_DEVICE_GUARD(ctx);
  int rc = check_groups(ctx, layer0, n_layers, B, width, pos_from, pos_to);
  if (rc) return rc;
  if (B == 0 || n_layers == 0) return MB_OK;
  if (!parent) return fail(ctx, MB_ERR_ARG, "null pointer");
  const int G = B / width;
  int64_t most = pos_from ? 0 : ctx->cfg.capacity;
  for (int g = 0; pos_from && g < G; g++) {
    if (pos_from[g] < 0 || pos_to[g] < pos_from[g])
      return fail(ctx, MB_ERR_ARG, "group %d: positions %d .. %d", g, pos_from[g], pos_to[g]);
    if (!ctx->cfg.wrap && pos_to[g] > ctx->cfg.capacity)
      return fail(ctx, MB_ERR_RANGE, "group %d: positions up to %d in a ring of %d slots", g, pos_to[g],
                  ctx->cfg.capacity);
    most = std::max<int64_t>(most, pos_to[g] - pos_from[g]);
  }
  if (most == 0) return MB_OK;
  int32_t* d = (int32_t*)scratch(ctx, "pos", ((size_t)B + 2 * G) * 4);
  if (!d) return fail(ctx, MB_ERR_NOMEM, "staging allocation failed");
  MB_HIP(ctx, hipMemcpyAsync(d, parent, (size_t)B * 4, hipMemcpyHostToDevice, ctx->stream));
  if (pos_from) {
    MB_HIP(ctx, hipMemcpyAsync(d + B, pos_from, (size_t)G * 4, hipMemcpyHostToDevice, ctx->stream));
    MB_HIP(ctx, hipMemcpyAsync(d + B + G, pos_to, (size_t)G * 4, hipMemcpyHostToDevice, ctx->stream));
  }
  rc = launch_ring_reorder(ctx, layer0, n_layers, B, width, d, pos_from ? d + B : nullptr,
                           pos_from ? d + B + G : nullptr, most);
  if (rc) return rc;
  MB_HIP(ctx, sync_stream(ctx));
  return MB_OK;
}

}  // extern "C"
