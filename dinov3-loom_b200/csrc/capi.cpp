// capi.cpp - the exported C ABI (include/dinov3.h, include/dinov3_kernels.h). Every entry point
// converts C++ exceptions into a status code and a thread-local message.
#include <algorithm>
#include <cstring>
#include <new>
#include <string>

#include "dinov3.h"
#include "dinov3_kernels.h"
#include "kernels.h"
#include "model.h"
#include "regions.h"
#include "weights.h"

struct dv3_model {
  dv3::Model impl;
  dv3_model(const std::string &path, dv3_options o) : impl(path, o) {}
};

namespace {

thread_local std::string g_last_error;

int fail(int code, const std::string &message) {
  g_last_error = message;
  return code;
}

template <class F>
int guarded(F &&f) {
  try {
    f();
    return DV3_OK;
  } catch (const dv3::Error &e) {
    return fail(e.code, e.what());
  } catch (const std::bad_alloc &) {
    return fail(DV3_DEVICE, "out of host memory");
  } catch (const std::exception &e) {
    return fail(DV3_DEVICE, e.what());
  }
}

int check_model(dv3_model *m) {
  if (!m) return fail(DV3_INVALID_ARGUMENT, "null model");
  return DV3_OK;
}

}  // namespace

namespace dv3 {
bool hub_weights(bool offline, std::string *path, std::string *err);
}

extern "C" {

dv3_options dv3_default_options(void) {
  dv3_options o;
  o.device = 0;
  o.max_batch = 32;
  return o;
}

int dv3_load(const char *path, dv3_options options, dv3_model **out) {
  if (!out) return fail(DV3_INVALID_ARGUMENT, "null output handle");
  *out = nullptr;
  return guarded([&] {
    if (options.max_batch < 1 || options.max_batch > DV3_MAX_BATCH_LIMIT)
      throw dv3::Error(DV3_INVALID_ARGUMENT, "max_batch must be 1..=64");
    if (!path) throw dv3::Error(DV3_INVALID_ARGUMENT, "null path");
    *out = new dv3_model(path, options);
  });
}

int dv3_from_pretrained(dv3_options options, dv3_model **out) {
  if (!out) return fail(DV3_INVALID_ARGUMENT, "null output handle");
  *out = nullptr;
  if (options.max_batch < 1 || options.max_batch > DV3_MAX_BATCH_LIMIT)
    return fail(DV3_INVALID_ARGUMENT, "max_batch must be 1..=64");
  std::string path, err;
  if (!dv3::hub_weights(false, &path, &err)) return fail(DV3_WEIGHTS, err);
  return dv3_load(path.c_str(), options, out);
}

int dv3_forward(dv3_model *m, const float *pixels, size_t n, float *out, size_t out_n) {
  if (int rc = check_model(m)) return rc;
  return guarded([&] { m->impl.forward(pixels, n, out, out_n); });
}

int dv3_cls(dv3_model *m, const float *pixels, size_t n, float *out, size_t out_n) {
  if (int rc = check_model(m)) return rc;
  return guarded([&] { m->impl.forward(pixels, n, out, out_n, dv3::Model::Readout::Cls); });
}

int dv3_patch_mean(dv3_model *m, const float *pixels, size_t n, float *out, size_t out_n) {
  if (int rc = check_model(m)) return rc;
  return guarded([&] { m->impl.forward(pixels, n, out, out_n, dv3::Model::Readout::PatchMean); });
}

int dv3_benchmark(dv3_model *m, const float *pixels, size_t n, size_t samples, dv3_timings *out) {
  if (int rc = check_model(m)) return rc;
  if (!out) return fail(DV3_INVALID_ARGUMENT, "null timings");
  return guarded([&] { *out = m->impl.benchmark(pixels, n, samples); });
}

void dv3_free(dv3_model *m) { delete m; }

const char *dv3_last_error(void) { return g_last_error.c_str(); }

float *dv3_input_buffer(dv3_model *m) { return m ? m->impl.input_buffer() : nullptr; }
float *dv3_output_buffer(dv3_model *m) { return m ? m->impl.output_buffer() : nullptr; }
void *dv3_stream(dv3_model *m) { return m ? static_cast<void *>(m->impl.stream()) : nullptr; }

int dv3_run(dv3_model *m, size_t batch) {
  if (int rc = check_model(m)) return rc;
  return guarded([&] { m->impl.run(batch); });
}

int dv3_synchronize(dv3_model *m) {
  if (int rc = check_model(m)) return rc;
  return guarded([&] { m->impl.synchronize(); });
}

int dv3_submit(dv3_model *m, const float *pixels, size_t n, float *out, size_t out_n,
               uint64_t *ticket) {
  if (int rc = check_model(m)) return rc;
  if (!ticket) return fail(DV3_INVALID_ARGUMENT, "null ticket");
  return guarded([&] { *ticket = m->impl.submit(pixels, n, out, out_n); });
}

int dv3_wait(dv3_model *m, uint64_t ticket) {
  if (!m) return fail(DV3_INVALID_ARGUMENT, "null model");
  // a poisoned model still reports each ticket's own status, then DV3_POISONED afterwards
  return guarded([&] { m->impl.wait(ticket); });
}

int dv3_forward_device(dv3_model *m, const float *pixels, size_t n, float *out, size_t out_n) {
  if (int rc = check_model(m)) return rc;
  return guarded([&] { m->impl.forward_device(pixels, n, out, out_n); });
}

int dv3_launches_per_forward(dv3_model *m, size_t batch, size_t *out) {
  if (int rc = check_model(m)) return rc;
  if (!out) return fail(DV3_INVALID_ARGUMENT, "null output");
  return guarded([&] { *out = m->impl.launches_per_forward(batch); });
}

int dv3_profile_launches(dv3_model *m, size_t batch, size_t iterations, double *ms,
                         const char **names, size_t capacity, size_t *count) {
  if (int rc = check_model(m)) return rc;
  return guarded([&] {
    auto r = m->impl.profile_launches(batch, iterations);
    for (size_t i = 0; i < r.size() && i < capacity; ++i) {
      if (ms) ms[i] = r[i].second;
      if (names) names[i] = r[i].first;
    }
    if (count) *count = r.size();
  });
}

int dv3_profile_forward(dv3_model *m, size_t batch, size_t replays, size_t flush_bytes,
                        double *ms, const char **names, size_t capacity, size_t *count) {
  if (int rc = check_model(m)) return rc;
  return guarded([&] {
    auto r = m->impl.profile_forward(batch, replays, flush_bytes);
    for (size_t i = 0; i < r.size() && i < capacity; ++i) {
      if (ms) ms[i] = r[i].second;
      if (names) names[i] = r[i].first;
    }
    if (count) *count = r.size();
  });
}

int dv3_debug_inject_fault(dv3_model *m, uint32_t bits) {
  if (int rc = check_model(m)) return rc;
  return guarded([&] { m->impl.inject_fault(bits); });
}

int dv3_hub_weights(int offline, char *path, size_t capacity) {
  if (!path || capacity == 0) return fail(DV3_INVALID_ARGUMENT, "null path buffer");
  std::string p, err;
  if (!dv3::hub_weights(offline != 0, &p, &err)) return fail(DV3_WEIGHTS, err);
  if (p.size() + 1 > capacity)
    return fail(DV3_INVALID_ARGUMENT, "path buffer too small: " + std::to_string(p.size() + 1) +
                                          " bytes needed");
  std::memcpy(path, p.c_str(), p.size() + 1);
  return DV3_OK;
}

int dv3_pack_f16(const char *name, const float *values, size_t n, uint16_t *out, size_t *bad) {
  if ((n && (!values || !out)) || !name) return fail(DV3_INVALID_ARGUMENT, "null argument");
  std::string msg;
  const size_t at = dv3::pack_f16(name, values, n, out, &msg);
  if (bad) *bad = at;
  if (at != SIZE_MAX) return fail(DV3_WEIGHTS, msg);
  return DV3_OK;
}

// ------------------------------------------------------------------------------------------
// Per-kernel entry points
// ------------------------------------------------------------------------------------------

}  // extern "C"

namespace {

bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

int launch_status(cudaError_t e, const char *what) {
  if (e == cudaSuccess) return DV3_OK;
  cudaGetLastError();
  return fail(DV3_DEVICE, std::string(what) + ": " + cudaGetErrorString(e));
}

template <class... P>
bool all_aligned(P... p) {
  return (aligned16(p) && ...);
}

int bad_args(const char *what) { return fail(DV3_INVALID_ARGUMENT, what); }

int current_device() {
  int dev = 0;
  cudaGetDevice(&dev);
  return dev;
}

int gemm_entry(dv3::GemmOp op, const void *a, uint32_t rows, const void *w,
               const dv3::GemmArgs &args, uint32_t *status, void *stream,
               const void *w_aux = nullptr) {
  if (rows == 0) return DV3_OK;
  dv3::GemmMaps maps;
  std::string err;
  const bool ln = op == dv3::GemmOp::ResidLN384 || op == dv3::GemmOp::ResidLN1536;
  const void *ln_out = args.ln_out_f32 ? static_cast<const void *>(args.ln_out_f32)
                                       : static_cast<const void *>(args.ln_out);
  if (!dv3::make_gemm_maps(op, a, rows, w, args.out, &maps, &err, ln ? ln_out : nullptr,
                           args.ln_out_f32 != nullptr))
    return bad_args(err.c_str());
  if (w_aux && !dv3::make_fold_maps(op, args.row_aux, rows, w_aux, &maps, &err))
    return bad_args(err.c_str());
  return launch_status(dv3::launch_gemm(op, maps, rows, args, status, static_cast<cudaStream_t>(stream)),
                       dv3::gemm_name(op));
}

}  // namespace

extern "C" {

int dv3k_bounded_wait_selftest(uint64_t wait_ns, uint32_t *status, void *stream) {
  if (!status) return bad_args("null status");
  if (wait_ns == 0 || wait_ns > 1000000000ull) return bad_args("wait_ns must be 1..1e9");
  return launch_status(dv3::launch_bounded_wait_selftest(wait_ns, status,
                                                         static_cast<cudaStream_t>(stream)),
                       "bounded wait self-test");
}

int dv3k_patchify(const float *images, uint32_t n_images, const float *prefix, uint16_t *patches,
                  uint16_t *x, uint32_t *status, void *stream) {
  if (n_images == 0) return DV3_OK;
  if (!all_aligned(images, prefix, patches, x)) return bad_args("pointers must be 16-byte aligned");
  return launch_status(dv3::launch_patchify(images, n_images, prefix, reinterpret_cast<__half *>(patches),
                                            reinterpret_cast<__half *>(x), status,
                                            static_cast<cudaStream_t>(stream)),
                       "patchify");
}

int dv3k_patch_embed(const uint16_t *patches, uint32_t n_patches, const uint16_t *w,
                     const float *bias, uint16_t *x, uint32_t *status, void *stream) {
  if (!all_aligned(patches, w, bias, x)) return bad_args("pointers must be 16-byte aligned");
  if (n_patches % dv3::kPatches != 0) return bad_args("n_patches must be a multiple of 196");
  dv3::GemmArgs g;
  g.bias = bias;
  g.out = reinterpret_cast<__half *>(x);
  return gemm_entry(dv3::GemmOp::Patch, patches, n_patches, w, g, status, stream);
}

int dv3k_layernorm_f16(const uint16_t *x, uint32_t rows, const float *gamma, const float *beta,
                       uint16_t *out, void *stream) {
  if (!all_aligned(x, gamma, beta, out)) return bad_args("pointers must be 16-byte aligned");
  return launch_status(dv3::launch_layernorm_f16(reinterpret_cast<const __half *>(x), rows, gamma, beta,
                                                 reinterpret_cast<__half *>(out),
                                                 static_cast<cudaStream_t>(stream)),
                       "layernorm_f16");
}

int dv3k_layernorm_f32out(const uint16_t *x, uint32_t rows, const float *gamma, const float *beta,
                          float *out, void *stream) {
  if (!all_aligned(x, gamma, beta, out)) return bad_args("pointers must be 16-byte aligned");
  return launch_status(dv3::launch_layernorm_f32(reinterpret_cast<const __half *>(x), rows, gamma, beta,
                                                 out, static_cast<cudaStream_t>(stream)),
                       "layernorm_f32out");
}

int dv3k_qkv_rope(const uint16_t *h, uint32_t rows, const uint16_t *w, const float *bias,
                  const float *rope_cos, const float *rope_sin, uint16_t *qkv, uint32_t *status,
                  void *stream) {
  if (!all_aligned(h, w, bias, rope_cos, rope_sin, qkv)) return bad_args("pointers must be 16-byte aligned");
  dv3::GemmArgs g;
  g.bias = bias;
  g.rope_cos = rope_cos;
  g.rope_sin = rope_sin;
  g.out = reinterpret_cast<__half *>(qkv);
  return gemm_entry(dv3::GemmOp::QkvRope, h, rows, w, g, status, stream);
}

int dv3k_attention(const uint16_t *qkv, uint32_t rows, uint16_t *out, uint32_t *status, void *stream) {
  if (rows == 0) return DV3_OK;
  if (!all_aligned(qkv, out)) return bad_args("pointers must be 16-byte aligned");
  if (rows % dv3::kTokens != 0) return bad_args("rows must be a multiple of 201");
  dv3::AttentionMaps map;
  std::string err;
  if (!dv3::make_attention_map(qkv, out, rows, &map, &err)) return bad_args(err.c_str());
  return launch_status(dv3::launch_attention(map, rows, status, static_cast<cudaStream_t>(stream)),
                       "attention");
}

int dv3k_matmul_splitk(const uint16_t *a, uint32_t rows, const uint16_t *w, uint32_t splits,
                       float *partials, uint32_t *status, void *stream) {
  if (!all_aligned(a, w, partials)) return bad_args("pointers must be 16-byte aligned");
  if (splits == 0 || (dv3::kMlp / 64) % splits != 0)
    return bad_args("splits must divide 24 (the 64-wide k-blocks of 1536)");
  if (rows == 0) return DV3_OK;
  dv3::GemmMaps maps;
  std::string err;
  if (!dv3::make_gemm_maps(dv3::GemmOp::SplitK1536, a, rows, w, partials, &maps, &err, nullptr,
                           false, splits))
    return bad_args(err.c_str());
  dv3::GemmArgs g;
  g.partials = partials;
  g.splits = splits;
  return launch_status(dv3::launch_gemm(dv3::GemmOp::SplitK1536, maps, rows, g, status,
                                        static_cast<cudaStream_t>(stream)),
                       dv3::gemm_name(dv3::GemmOp::SplitK1536));
}

int dv3k_splitk_reduce(const float *partials, uint32_t rows, uint32_t splits, const float *bias,
                       const float *lambda, uint16_t *x, void *stream) {
  if (!all_aligned(partials, bias, lambda, x)) return bad_args("pointers must be 16-byte aligned");
  if (splits == 0 || splits > 24) return bad_args("splits must be 1..24");
  return launch_status(dv3::launch_splitk_reduce(partials, rows, splits, bias, lambda,
                                                 reinterpret_cast<__half *>(x), nullptr, nullptr,
                                                 nullptr, nullptr, static_cast<cudaStream_t>(stream)),
                       "splitk_reduce");
}

int dv3k_splitk_reduce_layernorm(const float *partials, uint32_t rows, uint32_t splits,
                                 const float *bias, const float *lambda, uint16_t *x,
                                 const float *gamma, const float *beta, uint16_t *h,
                                 float *out_f32, void *stream) {
  if (!all_aligned(partials, bias, lambda, x, gamma, beta, h, out_f32))
    return bad_args("pointers must be 16-byte aligned");
  if (splits == 0 || splits > 24) return bad_args("splits must be 1..24");
  if ((h == nullptr) == (out_f32 == nullptr)) return bad_args("exactly one of h and out_f32");
  return launch_status(dv3::launch_splitk_reduce(partials, rows, splits, bias, lambda,
                                                 reinterpret_cast<__half *>(x), gamma, beta,
                                                 reinterpret_cast<__half *>(h), out_f32,
                                                 static_cast<cudaStream_t>(stream)),
                       "splitk_reduce_layernorm");
}

int dv3k_down_splitk_noalloc(const uint16_t *a, uint32_t rows, const uint16_t *w, uint32_t splits,
                             const float *bias, const float *lambda, uint16_t *x, uint32_t *status,
                             void *stream) {
  if (!all_aligned(a, w, bias, lambda, x)) return bad_args("pointers must be 16-byte aligned");
  if (splits == 0 || (dv3::kMlp / 64) % splits != 0)
    return bad_args("splits must divide 24 (the 64-wide k-blocks of 1536)");
  if (rows == 0) return DV3_OK;
  size_t capacity = 0;
  float *partials = dv3::splitk_scratch(&capacity);
  if (!partials) return fail(DV3_DEVICE, "split-K scratch: no device address");
  if (static_cast<size_t>(splits) * rows * dv3::kHidden > capacity)
    return bad_args("splits x rows exceeds the 6144 partial rows of the no-alloc scratch");
  dv3::GemmMaps maps;
  std::string err;
  if (!dv3::make_gemm_maps(dv3::GemmOp::SplitK1536, a, rows, w, partials, &maps, &err, nullptr,
                           false, splits))
    return bad_args(err.c_str());
  dv3::GemmArgs g;
  g.partials = partials;
  g.splits = splits;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int rc = launch_status(dv3::launch_gemm(dv3::GemmOp::SplitK1536, maps, rows, g, status, s),
                               dv3::gemm_name(dv3::GemmOp::SplitK1536));
  if (rc != DV3_OK) return rc;
  return launch_status(dv3::launch_splitk_reduce(partials, rows, splits, bias, lambda,
                                                 reinterpret_cast<__half *>(x), nullptr, nullptr,
                                                 nullptr, nullptr, s),
                       "splitk_reduce");
}

int dv3k_matmul_resid(const uint16_t *a, uint32_t rows, uint32_t k, const uint16_t *w,
                      const float *bias, const float *lambda, uint16_t *x, uint32_t *status,
                      void *stream) {
  if (!all_aligned(a, w, bias, lambda, x)) return bad_args("pointers must be 16-byte aligned");
  if (k != 384 && k != 1536) return bad_args("k must be 384 or 1536");
  dv3::GemmArgs g;
  g.bias = bias;
  g.lambda = lambda;
  g.out = reinterpret_cast<__half *>(x);
  return gemm_entry(k == 384 ? dv3::GemmOp::Resid384 : dv3::GemmOp::Resid1536, a, rows, w, g, status,
                    stream);
}

int dv3k_matmul_resid_layernorm(const uint16_t *a, uint32_t rows, uint32_t k, const uint16_t *w,
                                const float *bias, const float *lambda, uint16_t *x,
                                const float *gamma, const float *beta, uint16_t *h,
                                float *out_f32, uint32_t *status, void *stream) {
  if (!all_aligned(a, w, bias, lambda, x, gamma, beta, h, out_f32))
    return bad_args("pointers must be 16-byte aligned");
  if (k != 384 && k != 1536) return bad_args("k must be 384 or 1536");
  if ((h == nullptr) == (out_f32 == nullptr)) return bad_args("exactly one of h and out_f32");
  if (rows > 128u * static_cast<uint32_t>(dv3::sm_count(current_device())))
    return bad_args("rows must fit one 128-row tile per SM");
  dv3::GemmArgs g;
  g.bias = bias;
  g.lambda = lambda;
  g.out = reinterpret_cast<__half *>(x);
  g.gamma = gamma;
  g.beta = beta;
  g.ln_out = reinterpret_cast<__half *>(h);
  g.ln_out_f32 = out_f32;
  return gemm_entry(k == 384 ? dv3::GemmOp::ResidLN384 : dv3::GemmOp::ResidLN1536, a, rows, w, g,
                    status, stream);
}

int dv3k_matmul_swiglu(const uint16_t *h, uint32_t rows, const uint16_t *gateup_w,
                       const float *gateup_b, uint16_t *act, uint32_t *status, void *stream) {
  if (!all_aligned(h, gateup_w, gateup_b, act)) return bad_args("pointers must be 16-byte aligned");
  dv3::GemmArgs g;
  g.bias = gateup_b;
  g.out = reinterpret_cast<__half *>(act);
  return gemm_entry(dv3::GemmOp::SwiGLU, h, rows, gateup_w, g, status, stream);
}

int dv3k_matmul_resid_rowstat(const uint16_t *a, uint32_t rows, uint32_t k, const uint16_t *w,
                              const float *bias, const float *lambda, uint16_t *x, float *rowstat,
                              uint16_t *row_aux, uint32_t *status, void *stream) {
  if (!all_aligned(a, w, bias, lambda, x, rowstat, row_aux))
    return bad_args("pointers must be 16-byte aligned");
  if (k != 384 && k != 1536) return bad_args("k must be 384 or 1536");
  if (rowstat == nullptr || row_aux == nullptr) return bad_args("rowstat and row_aux are required");
  if (rows > 128u * static_cast<uint32_t>(dv3::sm_count(current_device())))
    return bad_args("rows must fit one 128-row tile per SM");
  dv3::GemmArgs g;
  g.bias = bias;
  g.lambda = lambda;
  g.out = reinterpret_cast<__half *>(x);
  g.rowstat = reinterpret_cast<float2 *>(rowstat);
  g.row_aux = reinterpret_cast<__half *>(row_aux);
  return gemm_entry(k == 384 ? dv3::GemmOp::ResidStats384 : dv3::GemmOp::ResidStats1536, a, rows,
                    w, g, status, stream);
}

int dv3k_layernorm_rowstat(const uint16_t *x, uint32_t rows, float *rowstat, uint16_t *row_aux,
                           void *stream) {
  if (!all_aligned(x, rowstat, row_aux)) return bad_args("pointers must be 16-byte aligned");
  if (rowstat == nullptr || row_aux == nullptr) return bad_args("rowstat and row_aux are required");
  return launch_status(dv3::launch_layernorm_rowstat(reinterpret_cast<const __half *>(x), rows,
                                                     reinterpret_cast<float2 *>(rowstat),
                                                     reinterpret_cast<__half *>(row_aux),
                                                     static_cast<cudaStream_t>(stream)),
                       "layernorm_rowstat");
}

int dv3k_qkv_rope_folded(const uint16_t *x, uint32_t rows, const uint16_t *wf,
                         const uint16_t *w_aux, const float *rowstat, const uint16_t *row_aux,
                         const float *rope_cos, const float *rope_sin, uint16_t *qkv,
                         uint32_t *status, void *stream) {
  if (!all_aligned(x, wf, w_aux, rowstat, row_aux, rope_cos, rope_sin, qkv))
    return bad_args("pointers must be 16-byte aligned");
  if (w_aux == nullptr || rowstat == nullptr || row_aux == nullptr)
    return bad_args("w_aux, rowstat and row_aux are required");
  dv3::GemmArgs g;
  g.rowstat = reinterpret_cast<float2 *>(const_cast<float *>(rowstat));
  g.row_aux = reinterpret_cast<__half *>(const_cast<uint16_t *>(row_aux));
  g.rope_cos = rope_cos;
  g.rope_sin = rope_sin;
  g.out = reinterpret_cast<__half *>(qkv);
  return gemm_entry(dv3::GemmOp::QkvRopeFold, x, rows, wf, g, status, stream, w_aux);
}

int dv3k_matmul_swiglu_folded(const uint16_t *x, uint32_t rows, const uint16_t *gateup_wf,
                              const uint16_t *w_aux, const float *rowstat,
                              const uint16_t *row_aux, uint16_t *act, uint32_t *status,
                              void *stream) {
  if (!all_aligned(x, gateup_wf, w_aux, rowstat, row_aux, act))
    return bad_args("pointers must be 16-byte aligned");
  if (w_aux == nullptr || rowstat == nullptr || row_aux == nullptr)
    return bad_args("w_aux, rowstat and row_aux are required");
  dv3::GemmArgs g;
  g.rowstat = reinterpret_cast<float2 *>(const_cast<float *>(rowstat));
  g.row_aux = reinterpret_cast<__half *>(const_cast<uint16_t *>(row_aux));
  g.out = reinterpret_cast<__half *>(act);
  return gemm_entry(dv3::GemmOp::SwiGLUFold, x, rows, gateup_wf, g, status, stream, w_aux);
}

uint32_t dv3k_gateup_source_row(uint32_t packed_row) { return dv3::gateup_source_row(packed_row); }

// ------------------------------------------------------------------------------------------
// Packed sequences and the paged cache
// ------------------------------------------------------------------------------------------

}  // extern "C"

namespace {

// A stride of an extent of one row or head is never used: 128 stands for whatever it is.
int64_t used_stride(int64_t stride, uint32_t extent) { return extent > 1 ? stride : 128; }

bool strides_ok(int64_t row, uint32_t rows, int64_t head, uint32_t heads) {
  constexpr int64_t kMost = int64_t{1} << 38;  // a tensor map's strides stay below 2^40 bytes
  if (rows == 0) return true;
  row = used_stride(row, rows);
  head = used_stride(head, heads);
  return row > 0 && head > 0 && row % 8 == 0 && head % 8 == 0 && row < kMost && head < kMost;
}

template <typename... P>
bool words_aligned(P... p) {
  return ((reinterpret_cast<uintptr_t>(p) | ...) & 3u) == 0;
}

// No two (row, head) vectors of `dim` elements share memory.
bool rows_apart(int64_t row, uint32_t rows, int64_t head, uint32_t heads, uint32_t dim) {
  if (rows == 0) return true;
  if (rows > 1 && row < dim) return false;
  if (heads > 1 && head < dim) return false;
  if (rows <= 1 || heads <= 1) return true;
  using wide = __int128;
  return static_cast<wide>(head) * (heads - 1) + dim <= row ||
         static_cast<wide>(row) * (rows - 1) + dim <= head;
}

using dv3::Region;
// A row tensor of 16-bit elements; `n` contiguous bytes.
Region rows_of(const void *p, int64_t row, uint32_t rows, int64_t head, uint32_t heads, uint32_t dim) {
  return {p, row * 2, head * 2, rows, heads, int64_t{dim} * 2};
}
Region bytes_of(const void *p, uint64_t n) { return {p, 1, 1, 1, 1, static_cast<int64_t>(n)}; }
Region cache_of(const void *p, int64_t page, uint32_t pages, uint32_t heads, uint32_t page_size, uint32_t dim) {
  return {p, page * 2, 1, pages, 1, int64_t{heads} * page_size * dim * 2};
}
Region table_of(const int32_t *p, int64_t row, uint32_t rows, uint32_t pages) {
  return {p, row * 4, 1, rows, 1, int64_t{pages} * 4};
}
// Whether the first `outs` of the regions, the outputs, share no memory with one another or with the
// inputs behind them. Ranges that do not meet need no closer look (a call's host time is what bounds it
// for one token: with one for every pair the append's took 3.8 us and not 2.9).
template <size_t kAll>
bool outputs_apart(const Region (&r)[kAll], size_t outs) {
  uintptr_t from[kAll], to[kAll];
  for (size_t i = 0; i < kAll; ++i) {
    from[i] = reinterpret_cast<uintptr_t>(r[i].base);
    const bool none = !r[i].base || !r[i].n_outer || !r[i].n_inner || !r[i].bytes;
    // below 2^31 rows or heads of strides below 2^39 bytes: saturated where that passes 64 bits
    const double far = static_cast<double>(r[i].n_outer - 1) * static_cast<double>(r[i].outer) +
                       static_cast<double>(r[i].n_inner - 1) * static_cast<double>(r[i].inner);
    to[i] = none ? from[i] : far > 9.0e15 ? UINTPTR_MAX
                           : from[i] + static_cast<uintptr_t>(far) + static_cast<uintptr_t>(r[i].bytes);
  }
  for (size_t i = 0; i < outs; ++i)
    for (size_t j = i + 1; j < kAll; ++j)
      if (from[i] < to[j] && from[j] < to[i] && !dv3::apart(r[i], r[j])) return false;
  return true;
}

const char *check_heads(uint32_t q_heads, uint32_t kv_heads, uint32_t head_dim, uint32_t dtype) {
  if (dtype > DV3K_BF16) return "dtype must be DV3K_F16 or DV3K_BF16";
  if (head_dim != 64 && head_dim != 128) return "head_dim must be 64 or 128";
  if (kv_heads == 0 || kv_heads > 65535) return "kv_heads must be 1..65535";
  if (q_heads % kv_heads != 0 || q_heads / kv_heads > 128)
    return "q_heads must be a multiple of kv_heads, at most 128 times it";
  return nullptr;
}

const char *check_pages(uint32_t page_size, uint32_t max_pages) {
  if (page_size == 0 || page_size > 65536) return "page_size must be 1..65536";
  if (static_cast<uint64_t>(max_pages) * page_size > 0x7fffffffull)
    return "max_pages x page_size must be below 2^31";
  return nullptr;
}

constexpr uint32_t kMostRows = 0x7fffff00u;  // rows or sequences of a call

bool paged_rows_ok(const dv3k_paged_attention &a) {
  return static_cast<uint64_t>(a.n_seq) * a.q_heads <= kMostRows;
}
// The packed kernel's search for an item walks the sequences, 32 a turn, while its other roles wait: 2^24
// of them are a quarter of a second at most, where a wait gives up after two.
bool packed_rows_ok(const dv3k_packed_attention &a) {
  return a.total_q <= kMostRows && a.total_k <= kMostRows && a.n_seq <= 1u << 24;
}

const char *check_cache(const void *k, const void *v, int64_t k_page, int64_t v_page,
                        const int32_t *table, int64_t table_stride, uint32_t n_seq,
                        uint32_t max_pages, uint32_t n_pages, uint32_t page_size, uint32_t kv_heads,
                        uint32_t head_dim) {
  if (const char *e = check_pages(page_size, max_pages)) return e;
  if (n_pages > 0x7fffffffu) return "n_pages must be below 2^31";
  if (n_pages > 0 && (!k || !v)) return "null cache";
  if (!all_aligned(k, v)) return "pointers must be 16-byte aligned";
  const int64_t least = static_cast<int64_t>(kv_heads) * page_size * head_dim;
  if (n_pages > 1 && (k_page < least || v_page < least || k_page % 8 != 0 || v_page % 8 != 0))
    return "pages must not overlap, a multiple of 8 elements apart";
  if (n_seq > 0 && max_pages > 0 && !table) return "null page_table";
  if ((reinterpret_cast<uintptr_t>(table) & 3u) != 0) return "page_table must be 4-byte aligned";
  if (n_seq > 1 && table_stride < static_cast<int64_t>(max_pages))
    return "table_stride must be at least max_pages";
  return nullptr;
}

bool scale_ok(float s) { return s > 0.f && s <= 1.0e30f; }

dv3::PagedAttention paged_args(const dv3k_paged_attention &a) {
  dv3::PagedAttention p = {};
  p.q = static_cast<const uint16_t *>(a.q);
  p.k_cache = static_cast<const uint16_t *>(a.k_cache);
  p.v_cache = static_cast<const uint16_t *>(a.v_cache);
  p.out = static_cast<uint16_t *>(a.out);
  p.lse = a.lse;
  p.lens = a.lens;
  p.page_table = a.page_table;
  p.workspace = a.workspace;
  p.q_seq = used_stride(a.q_seq, a.n_seq);
  p.q_head = used_stride(a.q_head, a.q_heads);
  p.out_seq = used_stride(a.out_seq, a.n_seq);
  p.out_head = used_stride(a.out_head, a.q_heads);
  p.k_page = used_stride(a.k_page, a.n_pages);
  p.v_page = used_stride(a.v_page, a.n_pages);
  p.table_stride = used_stride(a.table_stride, a.n_seq);
  p.status = a.status;
  p.page = dv3::page_div(a.page_size);
  p.n_seq = a.n_seq;
  p.max_len = static_cast<uint32_t>(
      std::min<uint64_t>(a.max_len, static_cast<uint64_t>(a.max_pages) * a.page_size));
  p.max_pages = a.max_pages;
  p.n_pages = a.n_pages;
  p.q_heads = a.q_heads;
  p.kv_heads = a.kv_heads;
  p.head_dim = a.head_dim;
  p.scale = a.scale;
  return p;
}

}  // namespace

extern "C" {

int dv3k_attention_packed(const dv3k_packed_attention *a, void *stream) {
  if (!a) return bad_args("null arguments");
  if (const char *e = check_heads(a->q_heads, a->kv_heads, a->head_dim, a->dtype)) return bad_args(e);
  if (a->q_heads == 0) return bad_args("q_heads must be positive");
  if (a->causal > 1 || a->reserved != 0) return bad_args("causal must be 0 or 1, reserved 0");
  if (!scale_ok(a->scale)) return bad_args("scale must be positive and finite");
  if (!packed_rows_ok(*a)) return bad_args("too many rows or sequences");
  if (!strides_ok(a->q_token, a->total_q, a->q_head, a->q_heads) ||
      !strides_ok(a->k_token, a->total_k, a->k_head, a->kv_heads) ||
      !strides_ok(a->v_token, a->total_k, a->v_head, a->kv_heads) ||
      !strides_ok(a->out_token, a->total_q, a->out_head, a->q_heads))
    return bad_args("strides must be positive multiples of 8 elements");
  if (!rows_apart(a->out_token, a->total_q, a->out_head, a->q_heads, a->head_dim))
    return bad_args("rows and heads of out overlap");
  if (a->total_q == 0 || a->n_seq == 0) return DV3_OK;
  if (!a->q || !a->out || !a->cu_q || !a->cu_k || (a->total_k > 0 && (!a->k || !a->v)))
    return bad_args("null tensor");
  if (!all_aligned(a->q, a->k, a->v, a->out, a->workspace))
    return bad_args("pointers must be 16-byte aligned");
  if (!words_aligned(a->lse, a->cu_q, a->cu_k, a->status))
    return bad_args("lse, cu_q, cu_k and status must be 4-byte aligned");
  dv3::PackedAttention p = {};
  p.q = static_cast<const uint16_t *>(a->q);
  p.k = static_cast<const uint16_t *>(a->k);
  p.v = static_cast<const uint16_t *>(a->v);
  p.out = static_cast<uint16_t *>(a->out);
  p.lse = a->lse;
  p.cu_q = a->cu_q;
  p.cu_k = a->cu_k;
  p.q_token = used_stride(a->q_token, a->total_q);
  p.q_head = used_stride(a->q_head, a->q_heads);
  p.k_token = used_stride(a->k_token, a->total_k);
  p.k_head = used_stride(a->k_head, a->total_k ? a->kv_heads : 0);
  p.v_token = used_stride(a->v_token, a->total_k);
  p.v_head = used_stride(a->v_head, a->total_k ? a->kv_heads : 0);
  p.out_token = used_stride(a->out_token, a->total_q);
  p.out_head = used_stride(a->out_head, a->q_heads);
  p.status = a->status;
  p.n_seq = a->n_seq;
  p.total_q = a->total_q;
  p.total_k = a->total_k;
  p.q_heads = a->q_heads;
  p.kv_heads = a->kv_heads;
  p.head_dim = a->head_dim;
  p.causal = a->causal != 0;
  p.scale = a->scale;
  p.workspace = a->workspace;
  const size_t need = dv3::attention_packed_workspace(p);
  if (need > 0 && (!a->workspace || a->workspace_bytes < need))
    return bad_args("workspace must hold dv3k_attention_packed_workspace bytes");
  const uint64_t cu_bytes = 4 * (uint64_t{a->n_seq} + 1);
  const Region all[] = {rows_of(p.out, p.out_token, p.total_q, p.out_head, p.q_heads, p.head_dim),
                        bytes_of(p.lse, 4 * uint64_t{p.total_q} * p.q_heads), bytes_of(p.workspace, need), bytes_of(p.status, 8),
                        rows_of(p.q, p.q_token, p.total_q, p.q_head, p.q_heads, p.head_dim),
                        rows_of(p.k, p.k_token, p.total_k, p.k_head, p.kv_heads, p.head_dim),
                        rows_of(p.v, p.v_token, p.total_k, p.v_head, p.kv_heads, p.head_dim),
                        bytes_of(p.cu_q, cu_bytes), bytes_of(p.cu_k, cu_bytes)};
  if (!outputs_apart(all, 4)) return bad_args("out overlaps an input, or lse, the workspace or status another tensor");
  std::string err;
  const cudaError_t e = dv3::launch_attention_packed(p, a->dtype == DV3K_BF16,
                                                     static_cast<cudaStream_t>(stream), &err);
  if (!err.empty()) return bad_args(err.c_str());
  return launch_status(e, "attention_packed");
}

size_t dv3k_attention_packed_workspace(const dv3k_packed_attention *a) {
  // 0 for what the launch refuses
  if (!a || check_heads(a->q_heads, a->kv_heads, a->head_dim, DV3K_F16) || a->q_heads == 0 || !packed_rows_ok(*a))
    return 0;
  dv3::PackedAttention p = {};
  p.n_seq = a->n_seq;
  p.total_q = a->total_q;
  p.total_k = a->total_k;
  p.q_heads = a->q_heads;
  p.kv_heads = a->kv_heads;
  p.head_dim = a->head_dim;
  return dv3::attention_packed_workspace(p);
}

size_t dv3k_attention_packed_workspace_bound(uint32_t head_dim) {
  return head_dim == 64 || head_dim == 128 ? dv3::attention_packed_workspace_bound(head_dim) : 0;
}

int dv3k_rope_append(const dv3k_rope_append_args *a, void *stream) {
  if (!a) return bad_args("null arguments");
  if (const char *e = check_heads(a->q_heads, a->kv_heads, a->head_dim, a->dtype)) return bad_args(e);
  if (a->reserved != 0) return bad_args("reserved must be 0");
  if ((a->q == nullptr) != (a->q_heads == 0) && a->total > 0)
    return bad_args("q and q_heads go together");
  if (a->rot_dim % 16 != 0 || a->rot_dim > a->head_dim)
    return bad_args("rot_dim must be a multiple of 16 up to head_dim");
  if (a->total > kMostRows || a->n_seq > kMostRows) return bad_args("too many rows or sequences");
  if (!a->cu_new && a->total != a->n_seq)
    return bad_args("without cu_new every sequence has one row: total must equal n_seq");
  if ((a->q_heads > 0 && (!strides_ok(a->q_token, a->total, a->q_head, a->q_heads) ||
                          !strides_ok(a->q_out_token, a->total, a->q_out_head, a->q_heads))) ||
      !strides_ok(a->k_token, a->total, a->k_head, a->kv_heads) ||
      !strides_ok(a->v_token, a->total, a->v_head, a->kv_heads))
    return bad_args("strides must be positive multiples of 8 elements");
  if (a->q_heads > 0 &&
      !rows_apart(a->q_out_token, a->total, a->q_out_head, a->q_heads, a->head_dim))
    return bad_args("rows and heads of q_out overlap");
  if (const char *e = check_cache(a->k_cache, a->v_cache, a->k_page, a->v_page, a->page_table,
                                  a->table_stride, a->n_seq, a->max_pages, a->n_pages,
                                  a->page_size, a->kv_heads, a->head_dim))
    return bad_args(e);
  if (a->total == 0 || a->n_seq == 0) return DV3_OK;
  if (!a->k || !a->v || !a->lens || (a->q_heads > 0 && !a->q_out) ||
      (a->rot_dim > 0 && (!a->cos || !a->sin)))
    return bad_args("null tensor");
  if (!all_aligned(a->q, a->k, a->v, a->q_out, a->cos, a->sin))
    return bad_args("pointers must be 16-byte aligned");
  if (!words_aligned(a->cu_new, a->lens, a->status))
    return bad_args("cu_new, lens and status must be 4-byte aligned");
  dv3::RopeAppend p = {};
  p.q = static_cast<const uint16_t *>(a->q);
  p.k = static_cast<const uint16_t *>(a->k);
  p.v = static_cast<const uint16_t *>(a->v);
  p.q_out = static_cast<uint16_t *>(a->q_out);
  p.k_cache = static_cast<uint16_t *>(a->k_cache);
  p.v_cache = static_cast<uint16_t *>(a->v_cache);
  p.cu_new = a->cu_new;
  p.lens = a->lens;
  p.page_table = a->page_table;
  p.cos = a->cos;
  p.sin = a->sin;
  p.q_token = used_stride(a->q_token, a->total);
  p.q_head = used_stride(a->q_head, a->q_heads);
  p.k_token = used_stride(a->k_token, a->total);
  p.k_head = used_stride(a->k_head, a->kv_heads);
  p.v_token = used_stride(a->v_token, a->total);
  p.v_head = used_stride(a->v_head, a->kv_heads);
  p.qo_token = used_stride(a->q_out_token, a->total);
  p.qo_head = used_stride(a->q_out_head, a->q_heads);
  p.k_page = used_stride(a->k_page, a->n_pages);
  p.v_page = used_stride(a->v_page, a->n_pages);
  p.table_stride = used_stride(a->table_stride, a->n_seq);
  p.status = a->status;
  p.page = dv3::page_div(a->page_size);
  p.n_seq = a->n_seq;
  p.total = a->total;
  p.max_pages = a->max_pages;
  p.n_pages = a->n_pages;
  p.positions = a->positions;
  p.rot_dim = a->rot_dim;
  p.q_heads = a->q_heads;
  p.kv_heads = a->kv_heads;
  p.head_dim = a->head_dim;
  const bool in_place = p.q && p.q == p.q_out;
  if (in_place && (p.q_token != p.qo_token || p.q_head != p.qo_head))
    return bad_args("q_out overlaps q: in place the strides are the same");
  const uint64_t turns = 4 * uint64_t{p.positions} * (p.rot_dim / 2);
  const Region q = rows_of(p.q, p.q_token, p.total, p.q_head, p.q_heads, p.head_dim);
  const Region all[] = {rows_of(p.q_out, p.qo_token, p.total, p.qo_head, p.q_heads, p.head_dim),
                        cache_of(p.k_cache, p.k_page, p.n_pages, p.kv_heads, p.page.size, p.head_dim),
                        cache_of(p.v_cache, p.v_page, p.n_pages, p.kv_heads, p.page.size, p.head_dim), bytes_of(p.status, 8),
                        rows_of(p.k, p.k_token, p.total, p.k_head, p.kv_heads, p.head_dim),
                        rows_of(p.v, p.v_token, p.total, p.v_head, p.kv_heads, p.head_dim),
                        bytes_of(p.cu_new, 4 * (uint64_t{p.n_seq} + 1)), bytes_of(p.lens, 4 * uint64_t{p.n_seq}),
                        table_of(p.page_table, p.table_stride, p.n_seq, p.max_pages), bytes_of(p.cos, turns), bytes_of(p.sin, turns),
                        in_place ? Region{} : q};
  if (!outputs_apart(all, 4)) return bad_args("q_out, a cache or status overlaps another tensor");
  return launch_status(
      dv3::launch_rope_append(p, a->dtype == DV3K_BF16, static_cast<cudaStream_t>(stream)),
      "rope_append");
}

size_t dv3k_attention_paged_workspace(const dv3k_paged_attention *a) {
  // 0 for what the launch refuses
  if (!a || check_heads(a->q_heads, a->kv_heads, a->head_dim, DV3K_F16) || a->q_heads == 0 ||
      a->n_seq == 0 || !paged_rows_ok(*a) || check_pages(a->page_size, a->max_pages))
    return 0;
  return dv3::attention_paged_workspace(paged_args(*a));
}

size_t dv3k_attention_paged_workspace_bound(uint32_t n_seq, uint32_t q_heads, uint32_t kv_heads,
                                            uint32_t head_dim) {
  dv3k_paged_attention a = {};
  a.n_seq = n_seq;
  a.q_heads = q_heads;
  a.kv_heads = kv_heads;
  a.head_dim = head_dim;
  a.page_size = 1;
  if (check_heads(q_heads, kv_heads, head_dim, DV3K_F16) || q_heads == 0 || n_seq == 0 || !paged_rows_ok(a)) return 0;
  return dv3::attention_paged_workspace_bound(paged_args(a));
}

int dv3k_attention_paged(const dv3k_paged_attention *a, void *stream) {
  if (!a) return bad_args("null arguments");
  if (const char *e = check_heads(a->q_heads, a->kv_heads, a->head_dim, a->dtype)) return bad_args(e);
  if (a->q_heads == 0) return bad_args("q_heads must be positive");
  if (!scale_ok(a->scale)) return bad_args("scale must be positive and finite");
  if (!paged_rows_ok(*a)) return bad_args("too many sequences and heads");
  if (!strides_ok(a->q_seq, a->n_seq, a->q_head, a->q_heads) ||
      !strides_ok(a->out_seq, a->n_seq, a->out_head, a->q_heads))
    return bad_args("strides must be positive multiples of 8 elements");
  if (!rows_apart(a->out_seq, a->n_seq, a->out_head, a->q_heads, a->head_dim))
    return bad_args("rows and heads of out overlap");
  if (const char *e = check_cache(a->k_cache, a->v_cache, a->k_page, a->v_page, a->page_table,
                                  a->table_stride, a->n_seq, a->max_pages, a->n_pages,
                                  a->page_size, a->kv_heads, a->head_dim))
    return bad_args(e);
  if (a->n_seq == 0) return DV3_OK;
  if (!a->q || !a->out || !a->lens) return bad_args("null tensor");
  if (!all_aligned(a->q, a->out, a->workspace)) return bad_args("pointers must be 16-byte aligned");
  if (!words_aligned(a->lse, a->lens, a->status))
    return bad_args("lse, lens and status must be 4-byte aligned");
  const dv3::PagedAttention p = paged_args(*a);
  const size_t need = dv3::attention_paged_workspace(p);
  if (need > 0 && (!a->workspace || a->workspace_bytes < need))
    return bad_args("workspace must hold dv3k_attention_paged_workspace bytes");
  const Region all[] = {rows_of(p.out, p.out_seq, p.n_seq, p.out_head, p.q_heads, p.head_dim),
                        bytes_of(p.lse, 4 * uint64_t{p.n_seq} * p.q_heads), bytes_of(p.workspace, need), bytes_of(p.status, 8),
                        rows_of(p.q, p.q_seq, p.n_seq, p.q_head, p.q_heads, p.head_dim),
                        cache_of(p.k_cache, p.k_page, p.n_pages, p.kv_heads, p.page.size, p.head_dim),
                        cache_of(p.v_cache, p.v_page, p.n_pages, p.kv_heads, p.page.size, p.head_dim),
                        bytes_of(p.lens, 4 * uint64_t{p.n_seq}), table_of(p.page_table, p.table_stride, p.n_seq, p.max_pages)};
  if (!outputs_apart(all, 4)) return bad_args("out overlaps an input, or lse, the workspace or status another tensor");
  return launch_status(
      dv3::launch_attention_paged(p, a->dtype == DV3K_BF16, static_cast<cudaStream_t>(stream)),
      "attention_paged");
}

}  // extern "C"
