// Python module `droid_backends` on top of the C ABI of libdroid_hip.so.
//
// Same nine functions, positional signatures, in-place semantics and error convention as the
// reference's pybind module (reference src/droid.cpp:93-259), so droid_slam/depth_video.py:196-222 and
// droid_slam/modules/corr.py:12,19,79,86 call it unchanged.  This file only does what a torch binding
// has to do: contiguity checks (TORCH_CHECK -> RuntimeError, as droid.cpp:89-90), output allocation on
// the inputs' device, workspace allocation through torch's caching allocator, and handing the current
// HIP stream to the C ABI.  No arithmetic happens here, and there is no CPU fallback: CPU tensors are
// rejected.
#include <torch/extension.h>
#include <c10/hip/HIPStream.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <vector>
#include <algorithm>
#include <unordered_set>
#include "../../include/droid_hip.h"

namespace {

#define CHECK_CONTIGUOUS(x) TORCH_CHECK(x.is_contiguous(), #x " must be contiguous")
#define CHECK_DEVICE(x) TORCH_CHECK(x.is_cuda(), #x " must be a ROCm device tensor (droid_backends has no CPU path)")
#define CHECK_INPUT(x) \
  CHECK_DEVICE(x);     \
  CHECK_CONTIGUOUS(x)
#define CHECK_F32(x) TORCH_CHECK(x.scalar_type() == torch::kFloat32, #x " must be float32")
#define CHECK_I64(x) TORCH_CHECK(x.scalar_type() == torch::kInt64, #x " must be int64")

dh_stream_t cur_stream() { return (dh_stream_t)c10::hip::getCurrentHIPStream().stream(); }

void check_status(int rc, const char* what) {
  TORCH_CHECK(rc == DH_OK, what, ": ", dh_status_string(rc));
}

int dtype_code(const torch::Tensor& t, const char* name, bool allow_f64 = false) {
  if (t.scalar_type() == torch::kFloat16) return DH_F16;
  if (t.scalar_type() == torch::kFloat32) return DH_F32;
  if (allow_f64 && t.scalar_type() == torch::kFloat64) return DH_F64;
  TORCH_CHECK(false, name, allow_f64 ? " must be float16, float32 or float64" : " must be float16 or float32");
  return -1;
}

// ---- ba (droid.cpp:93-122) --------------------------------------------------------------------
std::vector<torch::Tensor> ba_impl(torch::Tensor poses, torch::Tensor disps, torch::Tensor intrinsics,
                                   torch::Tensor disps_sens, c10::optional<torch::Tensor> alpha, torch::Tensor targets,
                                   torch::Tensor weights, torch::Tensor eta, torch::Tensor ii, torch::Tensor jj, const int t0,
                                   const int t1, const int iterations, const float lm, const float ep, const bool motion_only) {
  CHECK_INPUT(targets); CHECK_INPUT(weights); CHECK_INPUT(poses); CHECK_INPUT(disps);
  CHECK_INPUT(intrinsics); CHECK_INPUT(disps_sens); CHECK_INPUT(ii); CHECK_INPUT(jj);
  CHECK_DEVICE(eta);
  CHECK_F32(poses); CHECK_F32(disps); CHECK_F32(intrinsics); CHECK_F32(disps_sens);
  CHECK_F32(targets); CHECK_F32(weights); CHECK_F32(eta); CHECK_I64(ii); CHECK_I64(jj);
  eta = eta.contiguous();                           // the reference does not check eta (droid.cpp:110-117)
  const int F = (int)disps.size(0), ht = (int)disps.size(1), wd = (int)disps.size(2);
  const int E = (int)ii.size(0);
  TORCH_CHECK(poses.size(0) >= F && disps_sens.size(0) >= F, "poses / disps_sens shorter than disps");
  TORCH_CHECK(jj.size(0) == E && targets.size(0) == E && weights.size(0) == E, "edge count mismatch");
  const int HW = ht * wd;
  const int K = HW > 0 ? (int)(eta.numel() / HW) : 0;
  const int P = t1 - t0;
  auto fopts = poses.options();
  torch::Tensor dx = torch::zeros({P > 0 ? P : 0, 6}, fopts);
  torch::Tensor dz = torch::zeros({K, HW}, fopts);
  const size_t wsb = dh_ba_workspace_bytes(F, E, ht, wd, t0, t1, motion_only ? 1 : 0);
  TORCH_CHECK(wsb > 0, "ba: invalid arguments (t0/t1/buffer sizes)");
  torch::Tensor ws = torch::empty({(int64_t)wsb}, poses.options().dtype(torch::kUInt8));
  const float* al = nullptr;
  if (alpha.has_value()) {
    const torch::Tensor& a = *alpha;
    CHECK_INPUT(a); CHECK_F32(a);
    TORCH_CHECK(a.numel() == disps.numel(), "ba_ex: alpha must have the shape of disps");
    al = a.data_ptr<float>();
  }
  const int rc = dh_ba_ex(poses.data_ptr<float>(), disps.data_ptr<float>(), intrinsics.data_ptr<float>(),
                       disps_sens.data_ptr<float>(), al, targets.data_ptr<float>(), weights.data_ptr<float>(),
                       eta.data_ptr<float>(), ii.data_ptr<int64_t>(), jj.data_ptr<int64_t>(),
                       F, E, K, ht, wd, t0, t1, iterations, lm, ep, motion_only ? 1 : 0,
                       dx.data_ptr<float>(), motion_only ? nullptr : dz.data_ptr<float>(),
                       ws.data_ptr(), wsb, cur_stream());
  check_status(rc, "ba");
  return {dx, dz};
}


std::vector<torch::Tensor> ba(torch::Tensor poses, torch::Tensor disps, torch::Tensor intrinsics,
                              torch::Tensor disps_sens, torch::Tensor targets, torch::Tensor weights,
                              torch::Tensor eta, torch::Tensor ii, torch::Tensor jj, const int t0, const int t1,
                              const int iterations, const float lm, const float ep, const bool motion_only) {
  return ba_impl(poses, disps, intrinsics, disps_sens, c10::nullopt, targets, weights, eta, ii, jj, t0, t1, iterations, lm, ep, motion_only);
}

// ba with a per-pixel depth-prior weight alpha [buf,ht,wd] (MI355X extension, include/droid_hip.h dh_ba_ex)
std::vector<torch::Tensor> ba_ex(torch::Tensor poses, torch::Tensor disps, torch::Tensor intrinsics,
                                 torch::Tensor disps_sens, torch::Tensor alpha, torch::Tensor targets, torch::Tensor weights,
                                 torch::Tensor eta, torch::Tensor ii, torch::Tensor jj, const int t0, const int t1,
                                 const int iterations, const float lm, const float ep, const bool motion_only) {
  return ba_impl(poses, disps, intrinsics, disps_sens, alpha, targets, weights, eta, ii, jj, t0, t1, iterations, lm, ep, motion_only);
}


// ---- split BA for the edge-sharded multi-GPU solver: build -> (all-reduce of `system`) -> finish ------
// returns {workspace (opaque, keeps everything alive), system [(npad+48), npad] f64 view into it}: rows
// 0..npad-1 = reduced camera matrix (6P x 6P in the top-left corner), row npad = right-hand side.
static std::vector<torch::Tensor> ba_build_any(bool shard, torch::Tensor poses, torch::Tensor disps, torch::Tensor intrinsics,
                                               torch::Tensor disps_sens, c10::optional<torch::Tensor> alpha,
                                               torch::Tensor targets, torch::Tensor weights,
                                               torch::Tensor eta, torch::Tensor ii, torch::Tensor jj, const int t0, const int t1,
                                               const bool motion_only) {
  CHECK_INPUT(targets); CHECK_INPUT(weights); CHECK_INPUT(poses); CHECK_INPUT(disps);
  CHECK_INPUT(intrinsics); CHECK_INPUT(disps_sens); CHECK_INPUT(ii); CHECK_INPUT(jj); CHECK_INPUT(eta);
  CHECK_F32(poses); CHECK_F32(disps); CHECK_F32(intrinsics); CHECK_F32(disps_sens);
  CHECK_F32(targets); CHECK_F32(weights); CHECK_F32(eta); CHECK_I64(ii); CHECK_I64(jj);
  const int F = (int)disps.size(0), ht = (int)disps.size(1), wd = (int)disps.size(2);
  const int E = (int)ii.size(0), HW = ht * wd;
  const int K = HW > 0 ? (int)(eta.numel() / HW) : 0;
  const size_t wsb = dh_ba_workspace_bytes(F, E, ht, wd, t0, t1, motion_only ? 1 : 0);
  TORCH_CHECK(wsb > 0, "ba_build: invalid arguments");
  torch::Tensor ws = torch::empty({(int64_t)wsb}, poses.options().dtype(torch::kUInt8));
  double* H = nullptr; double* b = nullptr;
  const float* al = nullptr;
  if (alpha.has_value()) {
    const torch::Tensor& a = *alpha;
    CHECK_INPUT(a); CHECK_F32(a);
    TORCH_CHECK(shard, "ba_build: the per-pixel prior weight exists on ba_ex and ba_build_shard_ex");
    TORCH_CHECK(a.numel() == disps.numel(), "ba_build_shard_ex: alpha must have the shape of disps");
    al = a.data_ptr<float>();
  }
  if (shard)
    check_status(dh_ba_build_shard_ex(poses.data_ptr<float>(), disps.data_ptr<float>(), intrinsics.data_ptr<float>(),
                                      disps_sens.data_ptr<float>(), al, targets.data_ptr<float>(), weights.data_ptr<float>(),
                                      eta.data_ptr<float>(), ii.data_ptr<int64_t>(), jj.data_ptr<int64_t>(), F, E, K, ht, wd,
                                      t0, t1, motion_only ? 1 : 0, &H, &b, ws.data_ptr(), wsb, cur_stream()),
                 "ba_build_shard");
  else
    check_status(dh_ba_build(poses.data_ptr<float>(), disps.data_ptr<float>(), intrinsics.data_ptr<float>(),
                             disps_sens.data_ptr<float>(), targets.data_ptr<float>(), weights.data_ptr<float>(),
                             eta.data_ptr<float>(), ii.data_ptr<int64_t>(), jj.data_ptr<int64_t>(), F, E, K, ht, wd,
                             t0, t1, motion_only ? 1 : 0, &H, &b, ws.data_ptr(), wsb, cur_stream()),
                 "ba_build");
  int rows = 0, cols = 0;
  check_status(dh_ba_system_shape(t0, t1, &rows, &cols), "ba_system_shape");
  torch::Tensor sys = torch::from_blob(H, {rows, cols}, poses.options().dtype(torch::kFloat64));
  return {ws, sys};
}

std::vector<torch::Tensor> ba_build(torch::Tensor poses, torch::Tensor disps, torch::Tensor intrinsics,
                                    torch::Tensor disps_sens, torch::Tensor targets, torch::Tensor weights,
                                    torch::Tensor eta, torch::Tensor ii, torch::Tensor jj, const int t0, const int t1,
                                    const bool motion_only) {
  return ba_build_any(false, poses, disps, intrinsics, disps_sens, c10::nullopt, targets, weights, eta, ii, jj, t0, t1, motion_only);
}

// the edge-sharded solver's build (dh_ba_build_shard): no host synchronisation, the argument flag travels with the exchange
std::vector<torch::Tensor> ba_build_shard(torch::Tensor poses, torch::Tensor disps, torch::Tensor intrinsics,
                                          torch::Tensor disps_sens, torch::Tensor targets, torch::Tensor weights,
                                          torch::Tensor eta, torch::Tensor ii, torch::Tensor jj, const int t0, const int t1,
                                          const bool motion_only) {
  return ba_build_any(true, poses, disps, intrinsics, disps_sens, c10::nullopt, targets, weights, eta, ii, jj, t0, t1, motion_only);
}

// ba_build_shard with ba_ex's per-pixel depth-prior weight alpha [buf,ht,wd] (dh_ba_build_shard_ex; BASELINE configs[4] on the sharded path)
std::vector<torch::Tensor> ba_build_shard_ex(torch::Tensor poses, torch::Tensor disps, torch::Tensor intrinsics,
                                             torch::Tensor disps_sens, torch::Tensor alpha, torch::Tensor targets, torch::Tensor weights,
                                             torch::Tensor eta, torch::Tensor ii, torch::Tensor jj, const int t0, const int t1,
                                             const bool motion_only) {
  return ba_build_any(true, poses, disps, intrinsics, disps_sens, alpha, targets, weights, eta, ii, jj, t0, t1, motion_only);
}

static std::vector<torch::Tensor> ba_finish_any(torch::Tensor poses, torch::Tensor disps, torch::Tensor jj, torch::Tensor ws,
                                                const int n_eta_rows, const int t0, const int t1, const float lm, const float ep,
                                                const bool motion_only, const int own_lo, const int own_hi) {
  CHECK_INPUT(poses); CHECK_INPUT(disps); CHECK_INPUT(jj); CHECK_INPUT(ws); CHECK_F32(poses); CHECK_F32(disps);
  CHECK_I64(jj);
  const int F = (int)disps.size(0), ht = (int)disps.size(1), wd = (int)disps.size(2), E = (int)jj.size(0);
  const int P = t1 - t0;
  torch::Tensor dx = torch::zeros({P > 0 ? P : 0, 6}, poses.options());
  torch::Tensor dz = torch::zeros({F, ht * wd}, poses.options());
  check_status(dh_ba_finish_owned(poses.data_ptr<float>(), disps.data_ptr<float>(), jj.data_ptr<int64_t>(), F, E, ht, wd,
                                  t0, t1, lm, ep, motion_only ? 1 : 0, own_lo, own_hi, dx.data_ptr<float>(),
                                  motion_only ? nullptr : dz.data_ptr<float>(), ws.data_ptr(), (size_t)ws.numel(),
                                  cur_stream()),
               "ba_finish");
  return {dx, dz.narrow(0, 0, std::min(n_eta_rows, F))};
}

std::vector<torch::Tensor> ba_finish(torch::Tensor poses, torch::Tensor disps, torch::Tensor jj, torch::Tensor ws,
                                     const int n_eta_rows, const int t0, const int t1, const float lm, const float ep,
                                     const bool motion_only) {
  return ba_finish_any(poses, disps, jj, ws, n_eta_rows, t0, t1, lm, ep, motion_only, 0, 1 << 30);
}

std::vector<torch::Tensor> ba_finish_owned(torch::Tensor poses, torch::Tensor disps, torch::Tensor jj, torch::Tensor ws,
                                           const int n_eta_rows, const int t0, const int t1, const float lm, const float ep,
                                           const bool motion_only, const int own_lo, const int own_hi) {
  return ba_finish_any(poses, disps, jj, ws, n_eta_rows, t0, t1, lm, ep, motion_only, own_lo, own_hi);
}

// {Qinv [F,HW], w [F,HW] f32 (rows < K valid, ordered like kx), kx [F] int32, K [1] int32}: views into the workspace of ba_build
std::vector<torch::Tensor> ba_depth_blocks(torch::Tensor ws, torch::Tensor disps, torch::Tensor jj, const int t0, const int t1) {
  CHECK_INPUT(ws); CHECK_INPUT(disps); CHECK_INPUT(jj);
  const int F = (int)disps.size(0), ht = (int)disps.size(1), wd = (int)disps.size(2), E = (int)jj.size(0);
  const float *q = nullptr, *w = nullptr; const int *kx = nullptr, *K = nullptr;
  check_status(dh_ba_depth_blocks(ws.data_ptr(), (size_t)ws.numel(), F, E, ht, wd, t0, t1, &q, &w, &kx, &K), "ba_depth_blocks");
  auto f32 = disps.options().dtype(torch::kFloat32), i32 = disps.options().dtype(torch::kInt32);
  return {torch::from_blob((void*)q, {F, (int64_t)ht * wd}, f32), torch::from_blob((void*)w, {F, (int64_t)ht * wd}, f32),
          torch::from_blob((void*)kx, {F}, i32), torch::from_blob((void*)K, {1}, i32)};
}

// packed exchange of the co-visible 6x6 blocks (dh_ba_pack_blocks / dh_ba_unpack_blocks): `packed` f64
// [36 * n_blocks + 6 (t1 - t0) + 2], bp / bq int32 block rows / columns; disps / jj only give the sizes
void ba_pack_blocks(torch::Tensor ws, torch::Tensor disps, torch::Tensor jj, const int t0, const int t1, const bool motion_only,
                    torch::Tensor bp, torch::Tensor bq, const int host_flags, torch::Tensor packed) {
  CHECK_INPUT(ws); CHECK_INPUT(bp); CHECK_INPUT(bq); CHECK_INPUT(packed);
  TORCH_CHECK(bp.scalar_type() == torch::kInt32 && bq.scalar_type() == torch::kInt32 && bp.numel() == bq.numel(), "ba_pack_blocks: bp / bq int32, same length");
  TORCH_CHECK(packed.scalar_type() == torch::kFloat64 && (size_t)packed.numel() >= dh_ba_packed_len((int)bp.numel(), t0, t1), "ba_pack_blocks: packed buffer");
  check_status(dh_ba_pack_blocks(ws.data_ptr(), (size_t)ws.numel(), (int)disps.size(0), (int)jj.size(0), (int)disps.size(1), (int)disps.size(2),
                                 t0, t1, motion_only ? 1 : 0, bp.data_ptr<int32_t>(), bq.data_ptr<int32_t>(), (int)bp.numel(), host_flags,
                                 packed.data_ptr<double>(), cur_stream()),
               "ba_pack_blocks");
}

void ba_unpack_blocks(torch::Tensor ws, torch::Tensor disps, torch::Tensor jj, const int t0, const int t1, const bool motion_only,
                      torch::Tensor bp, torch::Tensor bq, torch::Tensor packed) {
  CHECK_INPUT(ws); CHECK_INPUT(bp); CHECK_INPUT(bq); CHECK_INPUT(packed);
  TORCH_CHECK(bp.scalar_type() == torch::kInt32 && bq.scalar_type() == torch::kInt32 && bp.numel() == bq.numel(), "ba_unpack_blocks: bp / bq int32, same length");
  TORCH_CHECK(packed.scalar_type() == torch::kFloat64 && (size_t)packed.numel() >= dh_ba_packed_len((int)bp.numel(), t0, t1), "ba_unpack_blocks: packed buffer");
  check_status(dh_ba_unpack_blocks(ws.data_ptr(), (size_t)ws.numel(), (int)disps.size(0), (int)jj.size(0), (int)disps.size(1), (int)disps.size(2),
                                   t0, t1, motion_only ? 1 : 0, bp.data_ptr<int32_t>(), bq.data_ptr<int32_t>(), (int)bp.numel(),
                                   packed.data_ptr<double>(), cur_stream()),
               "ba_unpack_blocks");
}

// dense exchange: status f64 [2]; set = false reads this rank's flags into it, set = true applies the all-reduced ones
void ba_exchange_flags(torch::Tensor ws, torch::Tensor disps, torch::Tensor jj, const int t0, const int t1, const bool motion_only,
                       const int host_flags, torch::Tensor status, const bool set) {
  CHECK_INPUT(ws); CHECK_INPUT(status);
  TORCH_CHECK(status.scalar_type() == torch::kFloat64 && status.numel() >= 2, "ba_exchange_flags: status f64 [2]");
  check_status(dh_ba_exchange_flags(ws.data_ptr(), (size_t)ws.numel(), (int)disps.size(0), (int)jj.size(0), (int)disps.size(1), (int)disps.size(2),
                                    t0, t1, motion_only ? 1 : 0, host_flags, status.data_ptr<double>(), set ? 1 : 0, cur_stream()),
               "ba_exchange_flags");
}

// ---- geometry (droid.cpp:125-171, 228-242) ------------------------------------------------------
torch::Tensor frame_distance(torch::Tensor poses, torch::Tensor disps, torch::Tensor intrinsics,
                             torch::Tensor ii, torch::Tensor jj, const float beta) {
  CHECK_INPUT(poses); CHECK_INPUT(disps); CHECK_INPUT(intrinsics); CHECK_INPUT(ii); CHECK_INPUT(jj);
  CHECK_F32(poses); CHECK_F32(disps); CHECK_F32(intrinsics); CHECK_I64(ii); CHECK_I64(jj);
  const int M = (int)ii.size(0);
  torch::Tensor dist = torch::zeros({M}, poses.options());
  check_status(dh_frame_distance(poses.data_ptr<float>(), disps.data_ptr<float>(), intrinsics.data_ptr<float>(),
                                 ii.data_ptr<int64_t>(), jj.data_ptr<int64_t>(), dist.data_ptr<float>(), M,
                                 (int)disps.size(1), (int)disps.size(2), beta, cur_stream()),
               "frame_distance");
  return dist;
}

std::vector<torch::Tensor> projmap(torch::Tensor poses, torch::Tensor disps, torch::Tensor intrinsics,
                                   torch::Tensor ii, torch::Tensor jj) {
  CHECK_INPUT(poses); CHECK_INPUT(disps); CHECK_INPUT(intrinsics); CHECK_INPUT(ii); CHECK_INPUT(jj);
  CHECK_F32(poses); CHECK_F32(disps); CHECK_F32(intrinsics); CHECK_I64(ii); CHECK_I64(jj);
  const int M = (int)ii.size(0), ht = (int)disps.size(1), wd = (int)disps.size(2);
  torch::Tensor coords = torch::empty({M, ht, wd, 3}, poses.options());
  torch::Tensor valid = torch::empty({M, ht, wd, 1}, poses.options());
  check_status(dh_projmap(poses.data_ptr<float>(), disps.data_ptr<float>(), intrinsics.data_ptr<float>(),
                          ii.data_ptr<int64_t>(), jj.data_ptr<int64_t>(), coords.data_ptr<float>(),
                          valid.data_ptr<float>(), M, ht, wd, cur_stream()),
               "projmap");
  return {coords, valid};
}

torch::Tensor iproj(torch::Tensor poses, torch::Tensor disps, torch::Tensor intrinsics) {
  CHECK_INPUT(poses); CHECK_INPUT(disps); CHECK_INPUT(intrinsics);
  CHECK_F32(poses); CHECK_F32(disps); CHECK_F32(intrinsics);
  const int N = (int)disps.size(0), ht = (int)disps.size(1), wd = (int)disps.size(2);
  torch::Tensor points = torch::empty({N, ht, wd, 3}, disps.options());
  check_status(dh_iproj(poses.data_ptr<float>(), disps.data_ptr<float>(), intrinsics.data_ptr<float>(),
                        points.data_ptr<float>(), N, ht, wd, cur_stream()),
               "iproj");
  return points;
}

torch::Tensor depth_filter(torch::Tensor poses, torch::Tensor disps, torch::Tensor intrinsics,
                           torch::Tensor ix, torch::Tensor thresh) {
  CHECK_INPUT(poses); CHECK_INPUT(disps); CHECK_INPUT(intrinsics); CHECK_INPUT(ix); CHECK_INPUT(thresh);
  CHECK_F32(poses); CHECK_F32(disps); CHECK_F32(intrinsics); CHECK_I64(ix); CHECK_F32(thresh);
  const int M = (int)ix.size(0), N = (int)disps.size(0), ht = (int)disps.size(1), wd = (int)disps.size(2);
  torch::Tensor counter = torch::empty({M, ht, wd}, disps.options());
  check_status(dh_depth_filter(poses.data_ptr<float>(), disps.data_ptr<float>(), intrinsics.data_ptr<float>(),
                               ix.data_ptr<int64_t>(), thresh.data_ptr<float>(), counter.data_ptr<float>(), M, N,
                               ht, wd, cur_stream()),
               "depth_filter");
  return counter;
}

// ---- correlation (droid.cpp:175-226) -------------------------------------------------------------
std::vector<torch::Tensor> corr_index_forward(torch::Tensor volume, torch::Tensor coords, int radius) {
  CHECK_INPUT(volume); CHECK_INPUT(coords); CHECK_F32(coords);
  TORCH_CHECK(volume.dim() == 5 && coords.dim() == 4, "corr_index_forward: volume [N,h1,w1,h2,w2], coords [N,2,h1,w1]");
  const int N = (int)volume.size(0), h1 = (int)volume.size(1), w1 = (int)volume.size(2);
  torch::Tensor corr = torch::empty({N, 2 * radius + 1, 2 * radius + 1, h1, w1}, volume.options());
  check_status(dh_corr_index_fwd(volume.data_ptr(), coords.data_ptr<float>(), corr.data_ptr(),
                                 dtype_code(volume, "volume", true), N, h1, w1, (int)volume.size(3), (int)volume.size(4),
                                 radius, cur_stream()),
               "corr_index_forward");
  return {corr};
}

std::vector<torch::Tensor> corr_index_backward(torch::Tensor volume, torch::Tensor coords,
                                               torch::Tensor corr_grad, int radius) {
  CHECK_INPUT(volume); CHECK_INPUT(coords); CHECK_INPUT(corr_grad); CHECK_F32(coords);
  TORCH_CHECK(corr_grad.scalar_type() == volume.scalar_type(), "corr_grad dtype must match volume");
  torch::Tensor volume_grad = torch::empty_like(volume);
  check_status(dh_corr_index_bwd(coords.data_ptr<float>(), corr_grad.data_ptr(), volume_grad.data_ptr(),
                                 dtype_code(volume, "volume", true), (int)volume.size(0), (int)volume.size(1),
                                 (int)volume.size(2), (int)volume.size(3), (int)volume.size(4), radius, cur_stream()),
               "corr_index_backward");
  return {volume_grad};
}

// ---- reference-layout volume + pooling for any image size (droid_amd.corr.CorrBlockRef) ----------------------
torch::Tensor corr_volume_build(torch::Tensor fmap1, torch::Tensor fmap2) {
  CHECK_INPUT(fmap1); CHECK_INPUT(fmap2);
  TORCH_CHECK(fmap1.dim() == 4 && fmap1.sizes() == fmap2.sizes() && fmap1.scalar_type() == fmap2.scalar_type(),
              "corr_volume_build: fmaps [E,C,h,w] of equal shape and dtype");
  const int E = (int)fmap1.size(0), C = (int)fmap1.size(1), h = (int)fmap1.size(2), w = (int)fmap1.size(3);
  torch::Tensor vol = torch::empty({E, h, w, h, w}, fmap1.options());
  check_status(dh_corr_volume_build(fmap1.data_ptr(), fmap2.data_ptr(), vol.data_ptr(), dtype_code(fmap1, "fmap1"), E, C, h, w, cur_stream()),
               "corr_volume_build");
  return vol;
}

torch::Tensor corr_volume_pool(torch::Tensor vol) {
  CHECK_INPUT(vol);
  TORCH_CHECK(vol.dim() >= 3, "corr_volume_pool: volume [..., h2, w2]");
  const int h2 = (int)vol.size(-2), w2 = (int)vol.size(-1);
  std::vector<int64_t> shape(vol.sizes().begin(), vol.sizes().end());
  shape[shape.size() - 2] = h2 / 2; shape[shape.size() - 1] = w2 / 2;
  torch::Tensor out = torch::empty(shape, vol.options());
  const long n = h2 * w2 > 0 ? vol.numel() / ((long)h2 * w2) : 0;
  check_status(dh_corr_volume_pool(vol.data_ptr(), out.data_ptr(), dtype_code(vol, "volume"), n, h2, w2, cur_stream()), "corr_volume_pool");
  return out;
}

std::vector<torch::Tensor> altcorr_forward(torch::Tensor fmap1, torch::Tensor fmap2, torch::Tensor coords,
                                           torch::Tensor ii, torch::Tensor jj, int radius) {
  CHECK_INPUT(fmap1); CHECK_INPUT(fmap2); CHECK_INPUT(coords); CHECK_DEVICE(ii); CHECK_DEVICE(jj);
  CHECK_F32(coords); CHECK_I64(ii); CHECK_I64(jj);
  TORCH_CHECK(fmap1.scalar_type() == fmap2.scalar_type(), "fmap dtypes differ");
  ii = ii.contiguous(); jj = jj.contiguous();
  const int B = (int)coords.size(0), M = (int)coords.size(1), H = (int)coords.size(3), W = (int)coords.size(4);
  const int rd = 2 * radius + 1;
  torch::Tensor corr = torch::empty({B, M, rd, rd, H, W}, fmap1.options());
  check_status(dh_altcorr_fwd(fmap1.data_ptr(), fmap2.data_ptr(), coords.data_ptr<float>(), ii.data_ptr<int64_t>(),
                              jj.data_ptr<int64_t>(), corr.data_ptr(), dtype_code(fmap1, "fmap1"), B,
                              (int)fmap1.size(1), (int)fmap2.size(1), (int)fmap1.size(2), H, W, (int)fmap2.size(3),
                              (int)fmap2.size(4), M, radius, cur_stream()),
               "altcorr_forward");
  return {corr};
}

// argument order follows the definition the reference actually links (droid.cpp:212-226)
std::vector<torch::Tensor> altcorr_backward(torch::Tensor fmap1, torch::Tensor fmap2, torch::Tensor coords,
                                            torch::Tensor corr_grad, torch::Tensor ii, torch::Tensor jj, int radius) {
  CHECK_INPUT(fmap1); CHECK_INPUT(fmap2); CHECK_INPUT(coords); CHECK_INPUT(corr_grad);
  CHECK_DEVICE(ii); CHECK_DEVICE(jj); CHECK_F32(coords); CHECK_I64(ii); CHECK_I64(jj);
  ii = ii.contiguous(); jj = jj.contiguous();
  torch::Tensor g = corr_grad.to(torch::kFloat32).contiguous();
  torch::Tensor g1 = torch::zeros(fmap1.sizes(), fmap1.options().dtype(torch::kFloat32));
  torch::Tensor g2 = torch::zeros(fmap2.sizes(), fmap2.options().dtype(torch::kFloat32));
  const int B = (int)coords.size(0), M = (int)coords.size(1), H = (int)coords.size(3), W = (int)coords.size(4);
  check_status(dh_altcorr_bwd(fmap1.data_ptr(), fmap2.data_ptr(), coords.data_ptr<float>(), ii.data_ptr<int64_t>(),
                              jj.data_ptr<int64_t>(), g.data_ptr<float>(), g1.data_ptr<float>(),
                              g2.data_ptr<float>(), dtype_code(fmap1, "fmap1"), B, (int)fmap1.size(1),
                              (int)fmap2.size(1), (int)fmap1.size(2), H, W, (int)fmap2.size(3), (int)fmap2.size(4),
                              M, radius, cur_stream()),
               "altcorr_backward");
  return {g1.to(fmap1.scalar_type()), g2.to(fmap2.scalar_type())};
}


// channel-last MFMA variant (droid_amd.corr.AltCorrBlock): fmap1 [N1,H,W,128], fmap2 [N2,H2,W2,128] f16, coords [M,2,H,W]
torch::Tensor altcorr_forward_nhwc(torch::Tensor fmap1, torch::Tensor fmap2, torch::Tensor coords, torch::Tensor ii,
                                   torch::Tensor jj) {
  CHECK_INPUT(fmap1); CHECK_INPUT(fmap2); CHECK_INPUT(coords); CHECK_INPUT(ii); CHECK_INPUT(jj);
  CHECK_F32(coords); CHECK_I64(ii); CHECK_I64(jj);
  TORCH_CHECK(fmap1.scalar_type() == torch::kFloat16 && fmap2.scalar_type() == torch::kFloat16, "fmaps must be float16");
  TORCH_CHECK(fmap1.dim() == 4 && fmap2.dim() == 4 && coords.dim() == 4 && coords.size(1) == 2, "altcorr_forward_nhwc: shapes");
  const int N1 = (int)fmap1.size(0), H = (int)fmap1.size(1), W = (int)fmap1.size(2), C = (int)fmap1.size(3);
  const int N2 = (int)fmap2.size(0), H2 = (int)fmap2.size(1), W2 = (int)fmap2.size(2), M = (int)ii.size(0);
  TORCH_CHECK(coords.size(0) == M && coords.size(2) == H && coords.size(3) == W && fmap2.size(3) == C, "altcorr_forward_nhwc: shapes");
  torch::Tensor out = torch::empty({M, 7, 7, H, W}, fmap1.options());
  check_status(dh_altcorr_fwd_nhwc(fmap1.data_ptr(), fmap2.data_ptr(), coords.data_ptr<float>(), ii.data_ptr<int64_t>(),
                                   jj.data_ptr<int64_t>(), out.data_ptr(), N1, N2, C, H, W, H2, W2, M, cur_stream()),
               "altcorr_forward_nhwc");
  return out;
}

// all levels of AltCorrBlock.__call__ into one [M, 49 * levels, H, W] tensor (no per-level stack copies)
torch::Tensor altcorr_forward_nhwc_levels(torch::Tensor fmap1, std::vector<torch::Tensor> fmap2_levels, torch::Tensor coords,
                                          torch::Tensor ii, torch::Tensor jj) {
  CHECK_INPUT(fmap1); CHECK_INPUT(coords); CHECK_INPUT(ii); CHECK_INPUT(jj);
  CHECK_F32(coords); CHECK_I64(ii); CHECK_I64(jj);
  TORCH_CHECK(fmap1.scalar_type() == torch::kFloat16 && fmap1.dim() == 4 && coords.dim() == 4 && coords.size(1) == 2, "altcorr_forward_nhwc_levels: shapes");
  const int N1 = (int)fmap1.size(0), H = (int)fmap1.size(1), W = (int)fmap1.size(2), C = (int)fmap1.size(3), M = (int)ii.size(0);
  const int L = (int)fmap2_levels.size();
  TORCH_CHECK(coords.size(0) == M && coords.size(2) == H && coords.size(3) == W && L >= 1, "altcorr_forward_nhwc_levels: shapes");
  torch::Tensor out = torch::empty({M, 49 * L, H, W}, fmap1.options());
  for (int l = 0; l < L; ++l) {
    const torch::Tensor& f2 = fmap2_levels[l];
    CHECK_INPUT(f2);
    TORCH_CHECK(f2.scalar_type() == torch::kFloat16 && f2.dim() == 4 && f2.size(3) == C, "altcorr_forward_nhwc_levels: level features [N2,h,w,C] float16");
    check_status(dh_altcorr_fwd_nhwc_level(fmap1.data_ptr(), f2.data_ptr(), coords.data_ptr<float>(), ii.data_ptr<int64_t>(), jj.data_ptr<int64_t>(),
                                           (char*)out.data_ptr() + (size_t)l * 49 * H * W * 2, N1, (int)f2.size(0), C, H, W, (int)f2.size(1), (int)f2.size(2), M,
                                           l, (long)49 * L * H * W, cur_stream()), "altcorr_forward_nhwc_levels");
  }
  return out;
}

// ---- MI355X-native correlation pyramid (own layout; droid_amd.corr.CorrBlock) ----------------------------
// h_real / w_real > 0: the features are an h_real x w_real image, zero-padded to the canvas size of the tensors
// (dh_corr_pyramid_build_canvas); 0 = the tensors ARE the image
// out: optional pre-allocated pyramid storage (float16, contiguous, at least E records) -- the caller's ARENA: a 105 GB hipMalloc
// costs seconds on a cold device, so callers that rebuild pyramids of the same graph (FactorGraph.update_lowmem) keep the storage
torch::Tensor corr_pyramid_build(torch::Tensor fmap1, torch::Tensor fmap2, const int h_real, const int w_real,
                                 const c10::optional<torch::Tensor>& out) {
  CHECK_INPUT(fmap1); CHECK_INPUT(fmap2);
  TORCH_CHECK(fmap1.scalar_type() == torch::kFloat16 && fmap2.scalar_type() == torch::kFloat16, "fmaps must be float16");
  TORCH_CHECK(fmap1.dim() == 4 && fmap1.sizes() == fmap2.sizes(), "corr_pyramid_build: fmaps [E,C,h,w] of equal shape");
  const int E = (int)fmap1.size(0), C = (int)fmap1.size(1), h = (int)fmap1.size(2), w = (int)fmap1.size(3);
  const size_t bytes1 = dh_corr_pyramid_bytes(1, h, w);
  TORCH_CHECK(bytes1 > 0, "corr_pyramid_build: unsupported image size (need h % 8 == 0 and w in {16,32,64})");
  torch::Tensor pyr;
  if (out.has_value() && out->defined()) {
    CHECK_INPUT((*out));
    TORCH_CHECK(out->scalar_type() == torch::kFloat16 && out->dim() == 2 && out->size(0) >= E && (size_t)out->size(1) * 2 == bytes1,
                "corr_pyramid_build: out must be float16 [>= E, record elements] for this image size");
    pyr = out->narrow(0, 0, E);
  } else {
    pyr = torch::empty({E, (int64_t)(bytes1 / 2)}, fmap1.options());
  }
  const int chunk = 256;                                  // bounds the channel-last scratch copies
  const size_t wsb = dh_corr_pyramid_workspace_bytes(std::min(E, chunk), h, w);
  torch::Tensor ws = torch::empty({(int64_t)wsb}, fmap1.options().dtype(torch::kUInt8));
  for (int s = 0; s < E; s += chunk) {
    const int n = std::min(chunk, E - s);
    check_status(dh_corr_pyramid_build_canvas(fmap1[s].data_ptr(), fmap2[s].data_ptr(), pyr[s].data_ptr(), ws.data_ptr(), wsb,
                                              n, C, h, w, h_real > 0 ? h_real : h, w_real > 0 ? w_real : w, cur_stream()),
                 "corr_pyramid_build");
  }
  return pyr;
}

// frame-level build: prepared = corr_pyramid_prepare_frames(fmaps [F,C,h,w] f16 (canvas-sized), h_real, w_real) -> [F, T, C] f16;
// corr_pyramid_build_indexed(prepared, idx1 [E] i64, idx2 [E] i64, h, w, out=None) -> pyramid [E, record elements]
torch::Tensor corr_pyramid_prepare_frames(torch::Tensor fmaps, const int h_real, const int w_real) {
  CHECK_INPUT(fmaps);
  TORCH_CHECK(fmaps.scalar_type() == torch::kFloat16 && fmaps.dim() == 4, "corr_pyramid_prepare_frames: fmaps [F,C,h,w] float16");
  const int F = (int)fmaps.size(0), C = (int)fmaps.size(1), h = (int)fmaps.size(2), w = (int)fmaps.size(3);
  const size_t bytes = dh_corr_pyramid_prepared_bytes(F, h, w);
  TORCH_CHECK(F == 0 || bytes > 0, "corr_pyramid_prepare_frames: unsupported image size (need h % 8 == 0 and w in {16,32,64})");
  torch::Tensor prep = torch::empty({F, F > 0 ? (int64_t)(bytes / 2 / F / C) : 0, C}, fmaps.options());
  check_status(dh_corr_pyramid_prepare_frames(fmaps.data_ptr(), prep.data_ptr(), F, C, h, w, h_real > 0 ? h_real : h, w_real > 0 ? w_real : w,
                                              cur_stream()), "corr_pyramid_prepare_frames");
  return prep;
}

torch::Tensor corr_pyramid_build_indexed(torch::Tensor prepared, torch::Tensor idx1, torch::Tensor idx2, const int h, const int w,
                                         const c10::optional<torch::Tensor>& out) {
  CHECK_INPUT(prepared); CHECK_INPUT(idx1); CHECK_INPUT(idx2); CHECK_I64(idx1); CHECK_I64(idx2);
  TORCH_CHECK(prepared.scalar_type() == torch::kFloat16 && prepared.dim() == 3 && prepared.size(2) == 128, "corr_pyramid_build_indexed: prepared [F,T,128] float16");
  const int F = (int)prepared.size(0), E = (int)idx1.size(0);
  TORCH_CHECK(idx2.size(0) == E, "corr_pyramid_build_indexed: idx1 / idx2 of equal length");
  const size_t bytes1 = dh_corr_pyramid_bytes(1, h, w);
  TORCH_CHECK(bytes1 > 0 && (size_t)prepared.size(1) * 128 * 2 * (size_t)std::max(F, 1) == dh_corr_pyramid_prepared_bytes(std::max(F, 1), h, w),
              "corr_pyramid_build_indexed: prepared does not belong to this image size");
  if (E > 0) {                                            // one read-back for the four bounds (an index outside the tensor would be a wild read)
    torch::Tensor b = torch::stack({idx1.min(), idx1.max(), idx2.min(), idx2.max()}).cpu();
    const int64_t* bp = b.data_ptr<int64_t>();
    TORCH_CHECK(bp[0] >= 0 && bp[1] < F && bp[2] >= 0 && bp[3] < F, "corr_pyramid_build_indexed: frame index out of range");
  }
  torch::Tensor pyr;
  if (out.has_value() && out->defined()) {
    CHECK_INPUT((*out));
    TORCH_CHECK(out->scalar_type() == torch::kFloat16 && out->dim() == 2 && out->size(0) >= E && (size_t)out->size(1) * 2 == bytes1,
                "corr_pyramid_build_indexed: out must be float16 [>= E, record elements] for this image size");
    pyr = out->narrow(0, 0, E);
  } else {
    pyr = torch::empty({E, (int64_t)(bytes1 / 2)}, prepared.options());
  }
  check_status(dh_corr_pyramid_build_indexed(prepared.data_ptr(), idx1.data_ptr<int64_t>(), idx2.data_ptr<int64_t>(), pyr.data_ptr(), F, E, h, w,
                                             cur_stream()), "corr_pyramid_build_indexed");
  return pyr;
}

torch::Tensor corr_pyramid_lookup(torch::Tensor pyramid, torch::Tensor coords) {
  CHECK_INPUT(pyramid); CHECK_INPUT(coords); CHECK_F32(coords);
  TORCH_CHECK(pyramid.scalar_type() == torch::kFloat16, "pyramid must be float16");
  TORCH_CHECK(coords.dim() == 4 && coords.size(3) == 2, "corr_pyramid_lookup: coords [E,h,w,2]");
  const int E = (int)coords.size(0), h = (int)coords.size(1), w = (int)coords.size(2);
  TORCH_CHECK(pyramid.size(0) == E && (size_t)pyramid.size(1) * 2 == dh_corr_pyramid_bytes(1, h, w),
              "corr_pyramid_lookup: pyramid does not match coords");
  torch::Tensor out = torch::empty({E, 4 * 49, h, w}, pyramid.options());
  check_status(dh_corr_pyramid_lookup(pyramid.data_ptr(), coords.data_ptr<float>(), out.data_ptr(), E, h, w, cur_stream()),
               "corr_pyramid_lookup");
  return out;
}

torch::Tensor corr_pyramid_lookup_nhwc(torch::Tensor pyramid, torch::Tensor coords) {
  CHECK_INPUT(pyramid); CHECK_INPUT(coords); CHECK_F32(coords);
  TORCH_CHECK(pyramid.scalar_type() == torch::kFloat16, "pyramid must be float16");
  TORCH_CHECK(coords.dim() == 4 && coords.size(3) == 2, "corr_pyramid_lookup_nhwc: coords [E,h,w,2]");
  const int E = (int)coords.size(0), h = (int)coords.size(1), w = (int)coords.size(2);
  TORCH_CHECK(pyramid.size(0) == E && (size_t)pyramid.size(1) * 2 == dh_corr_pyramid_bytes(1, h, w),
              "corr_pyramid_lookup_nhwc: pyramid does not match coords");
  torch::Tensor out = torch::empty({4, E, h, w, 56}, pyramid.options());
  check_status(dh_corr_pyramid_lookup_nhwc(pyramid.data_ptr(), coords.data_ptr<float>(), out.data_ptr(), E, h, w, cur_stream()),
               "corr_pyramid_lookup_nhwc");
  return out;
}

torch::Tensor corr_pyramid_lookup_corr0(torch::Tensor pyramid, torch::Tensor coords, torch::Tensor wpk, torch::Tensor bias) {
  CHECK_INPUT(pyramid); CHECK_INPUT(coords); CHECK_F32(coords); CHECK_INPUT(wpk); CHECK_INPUT(bias);
  TORCH_CHECK(pyramid.scalar_type() == torch::kFloat16, "pyramid must be float16");
  TORCH_CHECK(coords.dim() == 4 && coords.size(3) == 2, "corr_pyramid_lookup_corr0: coords [E,h,w,2]");
  TORCH_CHECK(wpk.scalar_type() == torch::kFloat16 && wpk.numel() == 13 * 128 * 16, "corr_pyramid_lookup_corr0: wpk [13,128,16] float16");
  TORCH_CHECK(bias.scalar_type() == torch::kFloat32 && bias.numel() == 128, "corr_pyramid_lookup_corr0: bias [128] float32");
  const int E = (int)coords.size(0), h = (int)coords.size(1), w = (int)coords.size(2);
  TORCH_CHECK(pyramid.size(0) == E && (size_t)pyramid.size(1) * 2 == dh_corr_pyramid_bytes(1, h, w),
              "corr_pyramid_lookup_corr0: pyramid does not match coords");
  torch::Tensor out = torch::empty({E, h, w, 128}, pyramid.options());
  check_status(dh_corr_pyramid_lookup_corr0(pyramid.data_ptr(), coords.data_ptr<float>(), wpk.data_ptr(), bias.data_ptr<float>(),
                                            out.data_ptr(), E, h, w, cur_stream()), "corr_pyramid_lookup_corr0");
  return out;
}

torch::Tensor corr0_nchw(torch::Tensor x, torch::Tensor wp, torch::Tensor bias) {
  CHECK_INPUT(x); CHECK_INPUT(wp); CHECK_INPUT(bias);
  TORCH_CHECK(x.scalar_type() == torch::kFloat16 && x.dim() == 4 && x.size(1) == 196, "corr0_nchw: x [E,196,h,w] float16");
  TORCH_CHECK(wp.scalar_type() == torch::kFloat16 && wp.dim() == 2 && wp.size(0) == 128 && wp.size(1) == 208, "corr0_nchw: wp [128,208] float16");
  TORCH_CHECK(bias.scalar_type() == torch::kFloat32 && bias.numel() == 128, "corr0_nchw: bias [128] float32");
  const int64_t E = x.size(0), h = x.size(2), w = x.size(3);
  torch::Tensor out = torch::empty({E, h, w, 128}, x.options());
  check_status(dh_corr0_nchw_f16(x.data_ptr(), wp.data_ptr(), bias.data_ptr<float>(), out.data_ptr(), (int)E, (int)(h * w), cur_stream()),
               "corr0_nchw");
  return out;
}

torch::Tensor glo_gemv(torch::Tensor red, torch::Tensor wt, torch::Tensor bias, double scale) {
  CHECK_INPUT(red); CHECK_INPUT(wt); CHECK_INPUT(bias);
  TORCH_CHECK(red.scalar_type() == torch::kFloat32 && red.dim() == 2 && red.size(1) == 128, "glo_gemv: red [E,128] float32");
  TORCH_CHECK(wt.scalar_type() == torch::kFloat32 && wt.dim() == 2 && wt.size(0) == 128, "glo_gemv: wt [128,N] float32");
  const int64_t E = red.size(0), N = wt.size(1);
  TORCH_CHECK(bias.scalar_type() == torch::kFloat32 && bias.numel() == N && N <= 384, "glo_gemv: bias [N], N <= 384");
  torch::Tensor out = torch::empty({E, N}, red.options());
  check_status(dh_glo_gemv(red.data_ptr<float>(), wt.data_ptr<float>(), bias.data_ptr<float>(), out.data_ptr<float>(), (int)E, (int)N,
                           (float)scale, cur_stream()), "glo_gemv");
  return out;
}

torch::Tensor segment_mean(torch::Tensor x, torch::Tensor order, torch::Tensor seg_off) {
  CHECK_INPUT(x); CHECK_INPUT(order); CHECK_INPUT(seg_off); CHECK_I64(order); CHECK_I64(seg_off);
  TORCH_CHECK(x.scalar_type() == torch::kFloat16 && x.dim() >= 2, "segment_mean: x [E,...] float16");
  const int64_t E = x.size(0), K = seg_off.numel() - 1;
  TORCH_CHECK(order.numel() == E && K >= 0, "segment_mean: order [E], seg_off [K+1]");
  const int64_t row = E > 0 ? x.numel() / E : 0;
  auto sizes = x.sizes().vec(); sizes[0] = K;
  torch::Tensor out = torch::empty(sizes, x.options());
  if (E > 0) check_status(dh_segment_mean_f16(x.data_ptr(), order.data_ptr<int64_t>(), seg_off.data_ptr<int64_t>(), out.data_ptr(),
                                              (int)K, (long)row, cur_stream()), "segment_mean");
  return out;
}

// ---- implicit-GEMM convolution with fused epilogues (droid_amd.update.UpdateModule) ----------------------
// stride-2 "same" convolution of one dense NHWC input (dh_conv2d_s2_nhwc_f16: the encoders' down-sampling layers) -> [N,H/2,W/2,Cout] f16
torch::Tensor conv2d_s2_nhwc(torch::Tensor input, torch::Tensor weight, torch::Tensor bias, int64_t KH, int64_t KW, int64_t Cout, int64_t epilogue) {
  CHECK_INPUT(input); CHECK_INPUT(weight); CHECK_INPUT(bias); CHECK_F32(bias);
  TORCH_CHECK(input.scalar_type() == torch::kFloat16 && input.dim() == 4, "conv2d_s2_nhwc: input [N,H,W,C] float16, dense");
  TORCH_CHECK(weight.scalar_type() == torch::kFloat16 && weight.dim() == 2, "conv2d_s2_nhwc: packed weight [CoutPad,Kpad] float16");
  const int N = (int)input.size(0), H = (int)input.size(1), W = (int)input.size(2), C = (int)input.size(3);
  TORCH_CHECK(H % 2 == 0 && W % 2 == 0, "conv2d_s2_nhwc: even image size");
  torch::Tensor out = torch::empty({N, H / 2, W / 2, Cout}, input.options());
  check_status(dh_conv2d_s2_nhwc_f16(input.data_ptr(), C, C, weight.data_ptr(), bias.data_ptr<float>(), N, H, W, (int)KH, (int)KW, (int)Cout,
                                     (int)weight.size(0), (int)weight.size(1), (int)epilogue, out.data_ptr(), (int)Cout, cur_stream()),
               "conv2d_s2_nhwc");
  return out;
}

void conv2d_nhwc(std::vector<torch::Tensor> inputs, torch::Tensor weight, c10::optional<torch::Tensor> weight_halo,
                 torch::Tensor bias, int64_t KH, int64_t KW,
                 int64_t Cout, int64_t epilogue, c10::optional<torch::Tensor> out, int64_t out_stride,
                 c10::optional<torch::Tensor> gterm, c10::optional<torch::Tensor> aux0, c10::optional<torch::Tensor> aux1,
                 c10::optional<torch::Tensor> red, c10::optional<torch::Tensor> cinit, c10::optional<torch::Tensor> cinit_idx,
                 int64_t cinit_off, bool out_raw_f32, int64_t weights_layout, bool out_tiled, bool cinit_tiled,
                 c10::optional<torch::Tensor> glo_weight, c10::optional<torch::Tensor> glo_bias, c10::optional<torch::Tensor> glo_red) {
  TORCH_CHECK(!inputs.empty() && inputs.size() <= 4, "conv2d_nhwc: 1..4 inputs");
  const void* ptrs[4]; int chans[4], strides[4];
  const int64_t N = inputs[0].size(0), H = inputs[0].size(1), W = inputs[0].size(2);
  for (size_t i = 0; i < inputs.size(); ++i) {
    const torch::Tensor& t = inputs[i];
    TORCH_CHECK(t.is_cuda() && t.scalar_type() == torch::kFloat16 && t.dim() == 4, "conv2d_nhwc: inputs [N,H,W,C] float16 device tensors");
    TORCH_CHECK(t.size(0) == N && t.size(1) == H && t.size(2) == W, "conv2d_nhwc: input shapes differ");
    // dense NHWC or a channel slice of one: stride(3) == 1, pixels equally spaced
    // (the stride of a size-1 dimension is arbitrary in torch: only dimensions that are actually stepped through count)
    TORCH_CHECK(t.stride(3) == 1 && (H == 1 || t.stride(1) == t.stride(2) * W) && (N == 1 || t.stride(0) == t.stride(2) * W * H),
                "conv2d_nhwc: input must be NHWC (channel slices allowed)");
    ptrs[i] = t.data_ptr(); chans[i] = (int)t.size(3); strides[i] = (int)t.stride(2);
  }
  CHECK_INPUT(weight); CHECK_INPUT(bias); CHECK_F32(bias);
  TORCH_CHECK(weight.scalar_type() == torch::kFloat16 && weight.dim() == 2, "conv2d_nhwc: packed weight [CoutPad,Kpad] float16");
  auto opt_ptr = [](const c10::optional<torch::Tensor>& t) -> void* { return t.has_value() ? t->data_ptr() : nullptr; };
  auto last = [](const c10::optional<torch::Tensor>& t) -> int { return t.has_value() ? (int)t->stride(2) : 0; };   // pixel stride
  const bool out_f32 = out.has_value() && out->scalar_type() == torch::kFloat32;
  if (gterm.has_value()) { const torch::Tensor& gt = *gterm; CHECK_INPUT(gt); CHECK_F32(gt); }
  if (red.has_value()) { const torch::Tensor& rt = *red; CHECK_INPUT(rt); CHECK_F32(rt); }
  const float* ci = nullptr; const int64_t* cidx = nullptr; int cstride = 0;
  if (cinit.has_value()) {
    const torch::Tensor& ct = *cinit;
    TORCH_CHECK(cinit_idx.has_value(), "conv2d_nhwc: cinit needs cinit_idx");
    const torch::Tensor& it = *cinit_idx;
    CHECK_INPUT(ct); CHECK_F32(ct); CHECK_INPUT(it); CHECK_I64(it);
    if (cinit_tiled) {      // accumulator-tile layout (include/droid_hip.h): [K, H*W/256 pixel tiles, C/128 cout tiles, 32768 floats per tile]
      TORCH_CHECK(ct.dim() == 4 && ct.size(1) * 256 == H * W && ct.size(3) == 32768 && it.numel() == N,
                  "conv2d_nhwc: tiled cinit [K, H*W/256, C/128, 32768] f32, cinit_idx [N] i64");
      cstride = -(int)ct.size(2) * 128;
    } else {
      TORCH_CHECK(ct.dim() == 4 && ct.size(1) == H && ct.size(2) == W && it.numel() == N, "conv2d_nhwc: cinit [K,H,W,C] f32, cinit_idx [N] i64");
      cstride = (int)ct.size(3);
    }
    ci = ct.data_ptr<float>(); cidx = it.data_ptr<int64_t>();
  }
  TORCH_CHECK(!out_raw_f32 || out_f32, "conv2d_nhwc: out_raw_f32 needs a float32 output");
  TORCH_CHECK(!out_tiled || (out_f32 && out_raw_f32), "conv2d_nhwc: out_tiled needs a raw float32 output");
  const void* gw = nullptr; const float* gb = nullptr; float* gr = nullptr;
  if (glo_red.has_value()) {          // the next iteration's global-context reduction behind the q gate (dh_conv2d_nhwc_f16_ex3)
    TORCH_CHECK(glo_weight.has_value() && glo_bias.has_value(), "conv2d_nhwc: glo_red needs glo_weight and glo_bias");
    const torch::Tensor& w = *glo_weight; const torch::Tensor& b = *glo_bias; const torch::Tensor& r = *glo_red;
    CHECK_INPUT(w); CHECK_INPUT(b); CHECK_F32(b); CHECK_INPUT(r); CHECK_F32(r);
    TORCH_CHECK(w.scalar_type() == torch::kFloat16 && w.dim() == 2 && w.size(0) == 128 && w.size(1) == 128 && b.numel() == 128 &&
                r.dim() == 2 && r.size(0) == N && r.size(1) == 128, "conv2d_nhwc: glo_weight [128,128] f16, glo_bias [128] f32, glo_red [N,128] f32");
    gw = w.data_ptr(); gb = b.data_ptr<float>(); gr = r.data_ptr<float>();
  }
  check_status(dh_conv2d_nhwc_f16_ex3(ptrs, chans, strides, (int)inputs.size(), weight.data_ptr(), opt_ptr(weight_halo), (int)weights_layout, bias.data_ptr<float>(),
                                     (int)N, (int)H, (int)W, (int)KH, (int)KW, (int)Cout, (int)weight.size(0), (int)weight.size(1),
                                     (int)epilogue, opt_ptr(out), out_f32 ? (out_tiled ? 3 : out_raw_f32 ? 2 : 1) : 0, (int)out_stride,
                                     gterm.has_value() ? gterm->data_ptr<float>() : nullptr,
                                     opt_ptr(aux0), last(aux0), opt_ptr(aux1), last(aux1),
                                     red.has_value() ? red->data_ptr<float>() : nullptr, ci, cidx, cstride, (int)cinit_off,
                                     gw, gb, gr, cur_stream()),
               "conv2d_nhwc");
}

// ---- factor-graph side kernels (droid_amd.factor_graph / droid_amd.depth_video) ---------------------------------
// zero the canvas pixels outside the h x w image, in place (dh_canvas_mask_f16)
void canvas_mask_(torch::Tensor x, const int h, const int w) {
  CHECK_INPUT(x);
  TORCH_CHECK(x.scalar_type() == torch::kFloat16 && x.dim() == 4, "canvas_mask_: [N,Hc,Wc,C] float16");
  check_status(dh_canvas_mask_f16(x.data_ptr(), (int)x.size(0), (int)x.size(1), (int)x.size(2), (int)x.size(3), h, w, cur_stream()), "canvas_mask_");
}

torch::Tensor motion_features(torch::Tensor coords1, torch::Tensor target) {
  CHECK_INPUT(coords1); CHECK_INPUT(target); CHECK_F32(coords1); CHECK_F32(target);
  TORCH_CHECK(coords1.dim() == 4 && coords1.size(3) == 2 && target.sizes() == coords1.sizes(), "motion_features: [E,h,w,2]");
  const int E = (int)coords1.size(0), ht = (int)coords1.size(1), wd = (int)coords1.size(2);
  torch::Tensor flow = torch::empty({E, ht, wd, 8}, coords1.options().dtype(torch::kFloat16));
  check_status(dh_motion_features(coords1.data_ptr<float>(), target.data_ptr<float>(), flow.data_ptr(), E, ht, wd, cur_stream()), "motion_features");
  return flow;
}

// -> {target [E,h,w,2], weight [E,h,w,2], target_ba [E,2,h,w], weight_ba [E,2,h,w]}
std::vector<torch::Tensor> ba_inputs(torch::Tensor coords1, torch::Tensor dw) {
  CHECK_INPUT(coords1); CHECK_INPUT(dw); CHECK_F32(coords1); CHECK_F32(dw);
  TORCH_CHECK(coords1.dim() == 4 && coords1.size(3) == 2 && dw.dim() == 4 && dw.size(3) == 4 && dw.size(0) == coords1.size(0), "ba_inputs: shapes");
  const int E = (int)coords1.size(0), ht = (int)coords1.size(1), wd = (int)coords1.size(2);
  torch::Tensor target = torch::empty({E, ht, wd, 2}, coords1.options()), weight = torch::empty({E, ht, wd, 2}, coords1.options());
  torch::Tensor tb = torch::empty({E, 2, ht, wd}, coords1.options()), wb = torch::empty({E, 2, ht, wd}, coords1.options());
  check_status(dh_ba_inputs(coords1.data_ptr<float>(), dw.data_ptr<float>(), target.data_ptr<float>(), weight.data_ptr<float>(),
                            tb.data_ptr<float>(), wb.data_ptr<float>(), E, ht, wd, cur_stream()), "ba_inputs");
  return {target, weight, tb, wb};
}

torch::Tensor cvx_upsample(torch::Tensor disp, torch::Tensor mask) {
  CHECK_INPUT(disp); CHECK_INPUT(mask); CHECK_F32(disp);
  TORCH_CHECK(mask.scalar_type() == torch::kFloat16 && mask.dim() == 4 && mask.size(3) == 576 && disp.dim() == 3 &&
              mask.size(0) == disp.size(0) && mask.size(1) == disp.size(1) && mask.size(2) == disp.size(2),
              "cvx_upsample: disp [K,h,w] f32, mask [K,h,w,576] f16");
  const int K = (int)disp.size(0), ht = (int)disp.size(1), wd = (int)disp.size(2);
  torch::Tensor out = torch::empty({K, 8 * ht, 8 * wd}, disp.options());
  check_status(dh_cvx_upsample(disp.data_ptr<float>(), mask.data_ptr(), out.data_ptr<float>(), K, ht, wd, cur_stream()), "cvx_upsample");
  return out;
}

// dist [(t-t0)*(t-t1)] f32 (modified), edges_i/j: existing edges; returns {new_edges [2*max_new,2] i64, count [1] i32} (device)
std::vector<torch::Tensor> proximity_nms(torch::Tensor dist, torch::Tensor edges_i, torch::Tensor edges_j, int64_t t0, int64_t t1,
                                         int64_t t, int64_t rad, int64_t nms, double thresh, int64_t max_factors, int64_t n_es0,
                                         bool stereo, int64_t max_new) {
  CHECK_INPUT(dist); CHECK_F32(dist); CHECK_INPUT(edges_i); CHECK_INPUT(edges_j); CHECK_I64(edges_i); CHECK_I64(edges_j);
  TORCH_CHECK(dist.numel() == (t - t0) * (t - t1) && edges_i.numel() == edges_j.numel(), "proximity_nms: shapes");
  const int ne = (int)edges_i.numel();
  check_status(dh_proximity_nms(dist.data_ptr<float>(), nullptr, nullptr, edges_i.data_ptr<int64_t>(), edges_j.data_ptr<int64_t>(), ne, (int)t0,
                                (int)t1, (int)t, (int)rad, (int)nms, (float)thresh, (int)max_factors, (int)n_es0, stereo ? 1 : 0,
                                nullptr, 0, nullptr, 0, cur_stream()), "proximity_nms (mask)");
  auto srt = torch::sort(dist.view({-1}), /*stable=*/true, 0, false);
  torch::Tensor sorted = std::get<0>(srt).contiguous(), order = std::get<1>(srt).contiguous();
  torch::Tensor out = torch::zeros({2 * max_new, 2}, edges_i.options());
  torch::Tensor count = torch::zeros({1}, dist.options().dtype(torch::kInt32));
  check_status(dh_proximity_nms(dist.data_ptr<float>(), sorted.data_ptr<float>(), order.data_ptr<int64_t>(), nullptr, nullptr, 0, (int)t0, (int)t1, (int)t, (int)rad,
                                (int)nms, (float)thresh, (int)max_factors, (int)n_es0, stereo ? 1 : 0, out.data_ptr<int64_t>(),
                                (int)max_new, count.data_ptr<int>(), 1, cur_stream()), "proximity_nms (walk)");
  return {out, count};
}

torch::Tensor heads_gather(torch::Tensor partials, torch::Tensor bias4, int64_t H, int64_t W, int64_t mode) {
  CHECK_INPUT(partials); CHECK_INPUT(bias4); CHECK_F32(partials); CHECK_F32(bias4);
  TORCH_CHECK(partials.dim() == 5 && partials.size(2) == 6 && partials.size(3) == 64 && partials.size(4) == 4 && bias4.numel() >= 4 && W == 64 &&
              H % 4 == 0 && (partials.size(1) * 4) % H == 0,
              "heads_gather: partials [cout tiles, N*H/4 pixel tiles, 6, 64, 4] f32 of images with 64 columns");
  const int N = (int)(partials.size(1) * 4 / H);
  // mode 1: GraphAgg's eta head (one output, 0.01 * softplus) -> [N,H,W]
  torch::Tensor dw = mode == 1 ? torch::empty({N, H, W}, partials.options()) : torch::empty({N, H, W, 4}, partials.options());
  check_status(dh_heads_gather_ex(partials.data_ptr<float>(), bias4.data_ptr<float>(), dw.data_ptr<float>(), N, (int)H, (int)W,
                                  (int)partials.size(0), (int)mode, cur_stream()), "heads_gather");
  return dw;
}

// ---- encoder glue (droid_amd.encoder) ---------------------------------------------------------------------------------
torch::Tensor norm_act(torch::Tensor x, c10::optional<torch::Tensor> residual, bool normalize, bool relu) {
  CHECK_INPUT(x);
  TORCH_CHECK(x.scalar_type() == torch::kFloat16 && x.dim() == 4, "norm_act: x [N,H,W,C] float16");
  const int N = (int)x.size(0), HW = (int)(x.size(1) * x.size(2)), C = (int)x.size(3);
  const void* r = nullptr;
  if (residual.has_value()) {
    const torch::Tensor& rt = *residual; CHECK_INPUT(rt);
    TORCH_CHECK(rt.scalar_type() == torch::kFloat16 && rt.sizes() == x.sizes(), "norm_act: residual must match x");
    r = rt.data_ptr();
  }
  torch::Tensor y = torch::empty_like(x);
  torch::Tensor ws = torch::empty({normalize ? (int64_t)N * C * 2 : 1}, x.options().dtype(torch::kFloat32));
  check_status(dh_norm_act_nhwc_f16(x.data_ptr(), r, y.data_ptr(), ws.data_ptr<float>(), N, HW, C, normalize ? 1 : 0, relu ? 1 : 0,
                                    cur_stream()), "norm_act");
  return y;
}

// ---- extensions beyond the reference module (used by droid_amd / lietorch compat) ----------------
std::vector<torch::Tensor> reproject(torch::Tensor poses, torch::Tensor disps, torch::Tensor intrinsics,
                                     torch::Tensor ii, torch::Tensor jj) {
  CHECK_INPUT(poses); CHECK_INPUT(disps); CHECK_INPUT(intrinsics); CHECK_INPUT(ii); CHECK_INPUT(jj);
  CHECK_F32(poses); CHECK_F32(disps); CHECK_F32(intrinsics); CHECK_I64(ii); CHECK_I64(jj);
  const int E = (int)ii.size(0), ht = (int)disps.size(1), wd = (int)disps.size(2);
  torch::Tensor coords = torch::empty({E, ht, wd, 2}, poses.options());
  torch::Tensor valid = torch::empty({E, ht, wd, 1}, poses.options());
  // intrinsics [4]: one camera; [frames,4]: per frame (source frame's for the back-projection, target frame's for the projection)
  const int per_frame = intrinsics.dim() == 2 ? 1 : 0;
  TORCH_CHECK(intrinsics.size(-1) == 4 && (!per_frame || intrinsics.size(0) >= disps.size(0)),
              "reproject: intrinsics must be [4] or [frames,4] with one row per frame of disps");
  check_status(dh_reproject_ex(poses.data_ptr<float>(), disps.data_ptr<float>(), intrinsics.data_ptr<float>(), per_frame,
                               ii.data_ptr<int64_t>(), jj.data_ptr<int64_t>(), coords.data_ptr<float>(),
                               valid.data_ptr<float>(), E, ht, wd, cur_stream()),
               "reproject");
  return {coords, valid};
}

torch::Tensor se3_op(const std::string& op, torch::Tensor a, torch::Tensor b) {
  CHECK_INPUT(a); CHECK_F32(a);
  const bool two = (op == "mul" || op == "retr");
  if (two) { CHECK_INPUT(b); CHECK_F32(b); }
  const int64_t n = (op == "exp" || op == "retr") ? a.numel() / 6 : a.numel() / 7;
  auto shape = a.sizes().vec();
  shape.back() = (op == "log") ? 6 : 7;
  torch::Tensor out = torch::empty(shape, a.options());
  int rc;
  if (op == "log") rc = dh_se3_log(a.data_ptr<float>(), out.data_ptr<float>(), (int)n, cur_stream());
  else if (op == "inv") rc = dh_se3_inv(a.data_ptr<float>(), out.data_ptr<float>(), (int)n, cur_stream());
  else if (op == "mul") rc = dh_se3_mul(a.data_ptr<float>(), b.data_ptr<float>(), out.data_ptr<float>(), (int)n, cur_stream());
  else if (op == "exp") rc = dh_se3_exp(a.data_ptr<float>(), out.data_ptr<float>(), (int)n, cur_stream());
  else if (op == "retr") rc = dh_se3_retr(a.data_ptr<float>(), b.data_ptr<float>(), out.data_ptr<float>(), (int)n, cur_stream());
  else { TORCH_CHECK(false, "se3_op: unknown op ", op); rc = DH_ERR_ARG; }
  check_status(rc, "se3_op");
  return out;
}

// a [n,7], X [n,npts,D] with D = 4 (act) or 6 (adjT)
torch::Tensor se3_map(const std::string& op, torch::Tensor a, torch::Tensor X) {
  CHECK_INPUT(a); CHECK_INPUT(X); CHECK_F32(a); CHECK_F32(X);
  const int n = (int)(a.numel() / 7);
  const int D = (op == "act4") ? 4 : 6;
  TORCH_CHECK(X.size(-1) == D, "se3_map: last dim must be ", D);
  const int npts = n > 0 ? (int)(X.numel() / D / n) : 0;
  torch::Tensor Y = torch::empty_like(X);
  int rc = (op == "act4") ? dh_se3_act4(a.data_ptr<float>(), X.data_ptr<float>(), Y.data_ptr<float>(), n, npts, cur_stream())
                          : dh_se3_adjT(a.data_ptr<float>(), X.data_ptr<float>(), Y.data_ptr<float>(), n, npts, cur_stream());
  check_status(rc, "se3_map");
  return Y;
}

// ---- token operators: packed attention, norm + rotation of query / key heads (include/droid_hip.h dh_attn_*, dh_qk_norm_rope_*) ------
// These entry points take strided views, run on the tensors' own device (whatever the current one is) and on that device's current stream.
dh_stream_t stream_of(const torch::Tensor& t) { return (dh_stream_t)c10::hip::getCurrentHIPStream(t.get_device()).stream(); }

int token_dtype(const torch::Tensor& t, const char* name, bool allow_f32) {
  if (t.scalar_type() == torch::kFloat16) return DH_F16;
  if (t.scalar_type() == torch::kBFloat16) return DH_BF16;
  if (allow_f32 && t.scalar_type() == torch::kFloat32) return DH_F32;
  TORCH_CHECK(false, name, allow_f32 ? " must be float16, bfloat16 or float32" : " must be float16 or bfloat16");
  return -1;
}
// (a tangent would be dropped in silence)
void check_no_tangents(std::initializer_list<const torch::Tensor*> tensors) {
  for (const torch::Tensor* t : tensors) TORCH_CHECK(!t || !t->defined() || !t->_fw_grad(0).defined(), "an input carries a tangent: the token operators have no forward-mode derivative");
}
void check_heads(const torch::Tensor& t, const char* name, const torch::Tensor& like) {
  TORCH_CHECK(t.is_cuda(), name, " must be a ROCm device tensor (droid_backends has no CPU path)");
  TORCH_CHECK(t.dim() == 3, name, " must be [rows, heads, head_dim]");
  TORCH_CHECK(t.device() == like.device(), name, " is on another device");
  TORCH_CHECK(t.scalar_type() == like.scalar_type(), name, " has another type");
}
int64_t row_stride(const torch::Tensor& t) { return t.size(0) > 1 ? t.stride(0) : 0; }
int64_t head_stride(const torch::Tensor& t) { return t.size(1) > 1 ? t.stride(1) : 0; }
#define TOKEN_VIEW(t) t.data_ptr(), row_stride(t), head_stride(t)
// what dh_attn_* can read in place: adjacent channels, 16-byte pieces, offsets of a tile below 2^31
bool attn_view(const torch::Tensor& t) {
  return t.stride(2) == 1 && ((uintptr_t)t.data_ptr() & 15) == 0 && row_stride(t) % 8 == 0 && head_stride(t) % 8 == 0 &&
         row_stride(t) < (1ll << 24) && 128 * row_stride(t) + 32 * head_stride(t) + t.size(2) < (1ll << 30);
}
torch::Tensor attn_input(const torch::Tensor& t, bool keys = false) {
  const bool ok = t.numel() == 0 || (attn_view(t) && !(keys && t.size(0) > 1 && t.stride(0) < t.size(2)));        // rows of keys must not overlap
  return ok ? t : t.clone(at::MemoryFormat::Contiguous);
}

// What a view [rows, heads, channels] with adjacent channels covers: rows x heads pieces of `width` bytes.  at::get_overlap_status decides nothing for
// views that are not dense, and heads sliced from one projection are not.
struct Pieces { int64_t p, rows, st, heads, sh, width; };
Pieces pieces_of(const torch::Tensor& t) {
  const int64_t size = t.element_size();
  if (t.numel() == 0) return {0, 0, 0, 0, 0, 0};
  if (t.dim() != 3) return {(int64_t)t.data_ptr(), 1, 0, 1, 0, t.numel() * size};                      // positions, frequencies, weights: contiguous
  return {(int64_t)t.data_ptr(), t.size(0), t.size(0) > 1 ? t.stride(0) * size : 0, t.size(1), t.size(1) > 1 ? t.stride(1) * size : 0, t.size(2) * size};
}
// is there an m of [lo, hi] with -before < x + m step < behind
bool hits(int64_t x, int64_t step, int64_t lo, int64_t hi, int64_t before, int64_t behind) {
  if (step == 0) return lo <= hi && x > -before && x < behind;
  const int64_t y = -before - x, m = std::max(lo, (y >= 0 ? y / step : -((-y + step - 1) / step)) + 1);
  return m <= hi && x + m * step < behind;
}
constexpr int64_t MOST_PAIRS = 1 << 20;
// Do two of them share a byte?  Exact where the row strides agree (one row agrees with any) or there are up to 2^20 pairs of rows and heads to look
// at; otherwise yes as soon as the memory between their ends does.
bool overlap(Pieces a, Pieces b) {
  if (!a.rows || !b.rows || !a.heads || !b.heads) return false;
  const auto end = [](const Pieces& x) { return x.p + (x.rows - 1) * x.st + (x.heads - 1) * x.sh + x.width; };
  if (end(a) <= b.p || end(b) <= a.p) return false;
  if (a.rows == 1) a.st = b.st;
  if (b.rows == 1) b.st = a.st;
  if (a.heads == 1) a.sh = b.sh;
  if (b.heads == 1) b.sh = a.sh;
  const bool rows_alike = a.st == b.st, heads_alike = a.sh == b.sh;
  if (a.rows > b.rows && !rows_alike) std::swap(a, b);                       // the fewer rows one by one
  const int64_t n = (rows_alike ? 1 : a.rows) * (heads_alike ? a.heads + b.heads - 1 : std::min(a.heads * b.heads, MOST_PAIRS + 1));
  if (n > MOST_PAIRS) return true;
  for (int64_t r = 0; r < (rows_alike ? 1 : a.rows); ++r) {
    const int64_t x = b.p - (a.p + r * a.st), lo = rows_alike ? -(a.rows - 1) : 0;
    if (heads_alike) {
      for (int64_t h = -(a.heads - 1); h < b.heads; ++h)
        if (hits(x + h * a.sh, b.st, lo, b.rows - 1, b.width, a.width)) return true;
    } else {
      for (int64_t g = 0; g < a.heads; ++g)
        for (int64_t h = 0; h < b.heads; ++h)
          if (hits(x + h * b.sh - g * a.sh, b.st, lo, b.rows - 1, b.width, a.width)) return true;
    }
  }
  return false;
}
// do two elements of one view share their place?
bool overlaps_itself(const Pieces& a) {
  if (a.rows > 1 && a.st < a.width) return a.heads > 0;
  for (int64_t h = 1; h < a.heads; ++h)
    if (hits(h * a.sh, a.st, -(a.rows - 1), a.rows - 1, a.width, a.width)) return true;
  return false;
}
bool same_pieces(const Pieces& a, const Pieces& b) {
  return a.p == b.p && a.rows == b.rows && a.st == b.st && a.heads == b.heads && a.sh == b.sh && a.width == b.width;
}
// (an input whose channels are not adjacent is copied before anything is written)
void check_out(const torch::Tensor& out, const char* name) {
  TORCH_CHECK(!overlaps_itself(pieces_of(out)), name, ": several of its elements lie at the same place");
  TORCH_CHECK(!(at::GradMode::is_enabled() && out.requires_grad()) && !out._fw_grad(0).defined(), name, " wants a gradient or carries a tangent: what is written to it has none");
}
// written in place: autograd has to see that a tensor which it kept for a backward pass is another one now
void mark_written(const torch::Tensor& out) {
  if (!out.is_inference()) out.unsafeGetTensorImpl()->bump_version();
}
void check_apart(const torch::Tensor& out, const char* name, const torch::Tensor& in, const char* in_name, bool may_be_same = false) {
  if (out.numel() == 0 || in.numel() == 0 || (in.dim() == 3 && in.stride(2) != 1)) return;
  const Pieces a = pieces_of(out), b = pieces_of(in);
  TORCH_CHECK((may_be_same && same_pieces(a, b)) || !overlap(a, b), name, " overlaps ", in_name, may_be_same ? " without being it" : "");
}

dh_attn_info attn_info(const torch::Tensor& info) {
  TORCH_CHECK(info.device().is_cpu() && info.scalar_type() == torch::kInt64 && info.is_contiguous() && info.numel() * 8 == (int64_t)sizeof(dh_attn_info),
              "info must be what attention_plan returned");
  dh_attn_info i;
  memcpy(&i, info.data_ptr<int64_t>(), sizeof i);
  return i;
}

// (plan int32 on the host, info int64 on the host)
std::vector<torch::Tensor> attention_plan(const std::vector<int64_t>& q_len, const std::vector<int64_t>& k_len, c10::optional<std::vector<int64_t>> k_start,
                                          int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t causal_block) {
  TORCH_CHECK(q_len.size() == k_len.size() && (!k_start || k_start->size() == q_len.size()), "attention_plan: one key length (and start) for each sequence");
  TORCH_CHECK(heads > 0 && kv_heads > 0 && heads % kv_heads == 0 && heads / kv_heads <= 32 && heads < 65536, "attention_plan: heads must be a multiple (up to 32) of kv_heads");
  TORCH_CHECK(head_dim >= 8 && head_dim <= 128 && head_dim % 8 == 0, "attention_plan: head_dim must be a multiple of 8 up to 128");
  TORCH_CHECK(causal_block >= 0, "attention_plan: causal_block must not be negative");
  dh_attn_info i;
  const int64_t* ks = k_start ? k_start->data() : nullptr;
  check_status(dh_attn_plan(q_len.data(), k_len.data(), ks, (int64_t)q_len.size(), (int)heads, (int)kv_heads, (int)head_dim, causal_block, nullptr, 0, &i),
               "attention_plan (lengths and starts must not be negative, rows at most 2^30, work items a launch's)");
  torch::Tensor plan = torch::empty({i.ints}, torch::kInt32), info = torch::empty({(int64_t)(sizeof i / 8)}, torch::kInt64);
  check_status(dh_attn_plan(q_len.data(), k_len.data(), ks, (int64_t)q_len.size(), (int)heads, (int)kv_heads, (int)head_dim, causal_block,
                            plan.data_ptr<int32_t>(), i.ints, &i), "attention_plan");
  memcpy(info.data_ptr<int64_t>(), &i, sizeof i);
  return {plan, info};
}

void check_attn(const torch::Tensor& q, const torch::Tensor& k, const torch::Tensor& v, const torch::Tensor& plan, const dh_attn_info& i, const char* what) {
  check_no_tangents({&q, &k, &v});
  check_heads(q, "q", q); check_heads(k, "k", q); check_heads(v, "v", q);
  TORCH_CHECK(q.size(1) == i.heads && k.size(1) == i.kv_heads && q.size(2) == i.head_dim && k.size(2) == i.head_dim && v.sizes() == k.sizes(), what,
              ": q must be [rows, ", i.heads, ", ", i.head_dim, "], k and v [rows, ", i.kv_heads, ", ", i.head_dim, "] as the plan says");
  TORCH_CHECK(q.size(0) >= i.q_rows, what, ": the plan has ", i.q_rows, " query rows, q has ", q.size(0));
  TORCH_CHECK(k.size(0) >= i.k_rows, what, ": the plan has ", i.k_rows, " key rows, k has ", k.size(0));
  TORCH_CHECK(plan.device() == q.device() && plan.scalar_type() == torch::kInt32 && plan.is_contiguous() && plan.numel() == i.ints, what, ": the plan is on another device");
  plan.record_stream(c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(q.get_device()).unwrap());       // the caller may drop a plan while its work is queued, on any stream
}

// {o [rows, heads, head_dim], lse [rows, heads] f32, o_low (for_backward: what the rounding of o left behind; else None)}; rows behind the last sequence are 0 / -inf, or left alone in an `out` of the caller's
std::vector<torch::Tensor> attention_forward(torch::Tensor q, torch::Tensor k, torch::Tensor v, torch::Tensor plan, torch::Tensor info, double scale,
                                             c10::optional<torch::Tensor> out, bool for_backward) {
  const dh_attn_info i = attn_info(info);
  check_attn(q, k, v, plan, i, "attention_forward");
  const int dt = token_dtype(q, "q", false);
  TORCH_CHECK(scale > 0 && scale < 1e30, "attention_forward: scale must be positive");
  const c10::DeviceGuard guard(q.device());
  torch::Tensor o = out ? *out : torch::empty(q.sizes(), q.options());
  torch::Tensor lse = torch::empty({q.size(0), q.size(1)}, q.options().dtype(torch::kFloat32));
  torch::Tensor low = for_backward ? torch::empty(q.sizes(), q.options()) : torch::Tensor();
  if (out) {
    check_heads(o, "out", q);
    TORCH_CHECK(o.sizes() == q.sizes() && attn_view(o), "out must have q's shape, adjacent channels and 16-byte aligned heads");
    check_out(o, "out");
    check_apart(o, "out", q, "q"); check_apart(o, "out", k, "k"); check_apart(o, "out", v, "v");
  }
  q = attn_input(q); k = attn_input(k, true); v = attn_input(v, true);
  const size_t wsb = dh_attn_fwd_workspace_bytes(&i);
  torch::Tensor ws;
  if (wsb) ws = torch::empty({(int64_t)wsb}, q.options().dtype(torch::kUInt8));
  check_status(dh_attn_fwd(TOKEN_VIEW(q), TOKEN_VIEW(k), TOKEN_VIEW(v), TOKEN_VIEW(o), for_backward ? low.data_ptr() : nullptr, lse.data_ptr<float>(),
                           plan.data_ptr<int32_t>(), &i, dt, q.size(0), k.size(0), (float)scale, !out, wsb ? ws.data_ptr() : nullptr, wsb, stream_of(q)), "attention_forward");
  if (out) mark_written(o);
  if (out && q.size(0) > i.q_rows) lse.narrow(0, i.q_rows, q.size(0) - i.q_rows).fill_(-std::numeric_limits<float>::infinity());
  return {o, lse, low};
}

// {dq, dk, dv}, zero in rows that belong to no sequence
std::vector<torch::Tensor> attention_backward(torch::Tensor grad, torch::Tensor q, torch::Tensor k, torch::Tensor v, torch::Tensor o, torch::Tensor lse,
                                              c10::optional<torch::Tensor> low, torch::Tensor plan, torch::Tensor info, double scale) {
  const dh_attn_info i = attn_info(info);
  check_attn(q, k, v, plan, i, "attention_backward");
  check_no_tangents({&grad});
  check_heads(o, "o", q); check_heads(grad, "grad", q);
  TORCH_CHECK(o.sizes() == q.sizes() && grad.sizes() == q.sizes(), "attention_backward: o and grad must have q's shape");
  TORCH_CHECK(lse.device() == q.device() && lse.scalar_type() == torch::kFloat32 && lse.is_contiguous() && lse.dim() == 2 && lse.size(0) == q.size(0) && lse.size(1) == q.size(1),
              "attention_backward: lse must be what attention_forward returned");
  if (low) check_heads(*low, "o_low", q);
  TORCH_CHECK(!low || (low->sizes() == q.sizes() && low->is_contiguous()), "attention_backward: o_low must be what attention_forward returned");
  TORCH_CHECK(!i.keys_shared, "attention_backward: two sequences of the plan share keys");
  const int dt = token_dtype(q, "q", false);
  TORCH_CHECK(scale > 0 && scale < 1e30, "attention_backward: scale must be positive");
  const c10::DeviceGuard guard(q.device());
  q = attn_input(q); k = attn_input(k, true); v = attn_input(v, true); o = attn_input(o); grad = attn_input(grad);
  const bool gaps = i.k_total < i.k_rows;
  torch::Tensor dq = torch::empty(q.sizes(), q.options());
  torch::Tensor dk = gaps ? torch::zeros(k.sizes(), k.options()) : torch::empty(k.sizes(), k.options());
  torch::Tensor dv = gaps ? torch::zeros(k.sizes(), k.options()) : torch::empty(k.sizes(), k.options());
  const size_t wsb = dh_attn_bwd_workspace_bytes(&i);
  torch::Tensor ws = torch::empty({(int64_t)wsb}, q.options().dtype(torch::kUInt8));
  check_status(dh_attn_bwd(TOKEN_VIEW(grad), TOKEN_VIEW(q), TOKEN_VIEW(k), TOKEN_VIEW(v), TOKEN_VIEW(o), low ? low->data_ptr() : nullptr, lse.data_ptr<float>(), TOKEN_VIEW(dq), TOKEN_VIEW(dk), TOKEN_VIEW(dv),
                           plan.data_ptr<int32_t>(), &i, dt, q.size(0), k.size(0), (float)scale, 1, ws.data_ptr(), wsb, stream_of(q)), "attention_backward");
  return {dq, dk, dv};
}

// A leaf keeps the stream that its gradient was first wanted on for as long as a graph of it lives; autograd would join that stream into a
// capture, which ends the process.  Refused instead, before anything is recorded, for every leaf that the inputs come from.
void refuse_leaves_of_other_streams(std::initializer_list<const torch::Tensor*> inputs, const char* what) {
  if (!(*inputs.begin())->is_cuda()) return;                                 // (refused further on)
  const c10::DeviceGuard guard((*inputs.begin())->device());
  if (c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None) return;
  std::vector<torch::autograd::Node*> todo;
  std::unordered_set<torch::autograd::Node*> seen;
  const auto visit = [&](torch::autograd::Node* n) { if (n && seen.insert(n).second) todo.push_back(n); };
  std::vector<std::shared_ptr<torch::autograd::Node>> held;                  // (what the tensors give may be theirs alone)
  for (const torch::Tensor* t : inputs) {
    if (!t || !t->defined() || !t->requires_grad()) continue;
    held.push_back(t->is_leaf() ? torch::autograd::impl::try_get_grad_accumulator(*t) : t->grad_fn());
    visit(held.back().get());
  }
  while (!todo.empty()) {
    torch::autograd::Node* n = todo.back();
    todo.pop_back();
    if (n->next_edges().empty()) {                                           // the end of a path: a leaf's accumulator, or a node without inputs that want a gradient
      const auto stream = n->stream();
      TORCH_CHECK(!stream || *stream == c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(stream->device_index()).unwrap(), what,
                  ": this stream is being captured, and a graph of the same leaves lives on another one; drop it first");
    }
    for (const auto& e : n->next_edges()) visit(e.function.get());
  }
}

// the same with a gradient (once): what droid_amd.attention.packed_attention calls where one is wanted
struct PackedAttention : public torch::autograd::Function<PackedAttention> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, torch::Tensor q, torch::Tensor k, torch::Tensor v, torch::Tensor plan, torch::Tensor info,
                                                double scale) {
    auto r = attention_forward(q, k, v, plan, info, scale, c10::nullopt, true);
    ctx->save_for_backward({q, k, v, r[0], r[1], r[2], plan, info});
    ctx->saved_data["scale"] = scale;
    ctx->mark_non_differentiable({r[1]});
    return {r[0], r[1]};
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    TORCH_CHECK(!at::GradMode::is_enabled(), "packed_attention is differentiable once (create_graph is not supported)");
    const auto s = ctx->get_saved_variables();
    auto r = attention_backward(grads[0], s[0], s[1], s[2], s[3], s[4], s[5], s[6], s[7], ctx->saved_data["scale"].toDouble());
    return {r[0], r[1], r[2], torch::Tensor(), torch::Tensor(), torch::Tensor()};
  }
};
std::vector<torch::Tensor> packed_attention(torch::Tensor q, torch::Tensor k, torch::Tensor v, torch::Tensor plan, torch::Tensor info, double scale) {
  refuse_leaves_of_other_streams({&q, &k, &v}, "packed_attention");
  return PackedAttention::apply(q, k, v, plan, info, scale);
}

struct RopeArgs { std::vector<int> sections; int pos_type, w_dtype; const void *qw, *kw; };
RopeArgs rope_args(const torch::Tensor& q, const torch::Tensor& k, const torch::Tensor& positions, const torch::Tensor& inv_freq, const std::vector<int64_t>& sections,
                   const c10::optional<torch::Tensor>& q_weight, const c10::optional<torch::Tensor>& k_weight, bool normalize, double eps) {
  check_no_tangents({&q, &k, &positions, &inv_freq, q_weight ? &*q_weight : nullptr, k_weight ? &*k_weight : nullptr});
  check_heads(q, "q", q); check_heads(k, "k", q);
  TORCH_CHECK(k.size(0) == q.size(0) && k.size(2) == q.size(2), "q and k must have the same tokens and head_dim");
  const int64_t d = q.size(2);
  TORCH_CHECK(d >= 2 && d <= 256 && d % 2 == 0, "head_dim must be even and at most 256");
  TORCH_CHECK(!sections.empty() && sections.size() <= 4, "one to four sections");
  RopeArgs a{{}, 0, DH_F32, nullptr, nullptr};
  int64_t pairs = 0;
  for (const int64_t s : sections) {
    TORCH_CHECK(s >= 0 && s <= d, "sections must not be negative");
    a.sections.push_back((int)s);
    pairs += s;
  }
  TORCH_CHECK(pairs <= d / 2, "the sections have ", pairs, " pairs, a head has ", d / 2);
  TORCH_CHECK(positions.device() == q.device() && positions.is_contiguous() && positions.numel() == q.size(0) * (int64_t)sections.size() && positions.dim() <= 2 &&
              positions.dim() >= 1 && positions.size(0) == q.size(0), "positions must be contiguous [tokens, axes] on q's device");
  a.pos_type = positions.scalar_type() == torch::kInt32 ? 0 : positions.scalar_type() == torch::kInt64 ? 1 : positions.scalar_type() == torch::kFloat32 ? 2 : -1;
  TORCH_CHECK(a.pos_type >= 0, "positions must be int32, int64 or float32");
  TORCH_CHECK(inv_freq.device() == q.device() && inv_freq.scalar_type() == torch::kFloat32 && inv_freq.is_contiguous() && inv_freq.numel() == pairs,
              "inv_freq must be contiguous float32 with one value for each pair of the sections, on q's device");
  TORCH_CHECK(normalize || (!q_weight && !k_weight), "weights need normalize");
  TORCH_CHECK(eps >= 0, "eps must not be negative");
  const torch::Tensor* first = nullptr;
  for (const auto* w : {&q_weight, &k_weight})
    if (*w) {
      const torch::Tensor& t = **w;
      TORCH_CHECK(t.device() == q.device() && t.dim() == 1 && t.size(0) == d && t.is_contiguous(), "weights must be contiguous [head_dim] on q's device");
      TORCH_CHECK(!first || first->scalar_type() == t.scalar_type(), "q_weight and k_weight must have one type");
      a.w_dtype = token_dtype(t, "weights", true);
      first = &t;
      (w == &q_weight ? a.qw : a.kw) = t.data_ptr();
    }
  return a;
}
torch::Tensor rope_input(const torch::Tensor& t) { return t.numel() == 0 || t.stride(2) == 1 ? t : t.contiguous(); }

void rope_status(int rc, const char* what) {
  TORCH_CHECK(rc != DH_ERR_UNSUPPORTED, what, ": a head of more than 128 channels needs even halves (pairs, resting channels, strides)");
  check_status(rc, what);
}

std::vector<torch::Tensor> qk_norm_rope_forward(torch::Tensor q, torch::Tensor k, torch::Tensor positions, torch::Tensor inv_freq, const std::vector<int64_t>& sections,
                                                c10::optional<torch::Tensor> q_weight, c10::optional<torch::Tensor> k_weight, bool normalize, double eps, bool interleaved,
                                                c10::optional<torch::Tensor> q_out, c10::optional<torch::Tensor> k_out) {
  const RopeArgs a = rope_args(q, k, positions, inv_freq, sections, q_weight, k_weight, normalize, eps);
  const int dt = token_dtype(q, "q", true);
  const c10::DeviceGuard guard(q.device());
  torch::Tensor qo = q_out ? *q_out : torch::empty(q.sizes(), q.options()), ko = k_out ? *k_out : torch::empty(k.sizes(), k.options());
  check_heads(qo, "q_out", q); check_heads(ko, "k_out", q);
  TORCH_CHECK(qo.sizes() == q.sizes() && ko.sizes() == k.sizes() && (qo.numel() == 0 || qo.stride(2) == 1) && (ko.numel() == 0 || ko.stride(2) == 1),
              "q_out / k_out must have the shapes of q / k and adjacent channels");
  if (q_out || k_out) {
    check_out(qo, "q_out"); check_out(ko, "k_out");
    check_apart(qo, "q_out", q, "q", true); check_apart(ko, "k_out", k, "k", true);
    check_apart(qo, "q_out", k, "k"); check_apart(ko, "k_out", q, "q"); check_apart(qo, "q_out", ko, "k_out");
    for (const torch::Tensor* t : {&positions, &inv_freq, q_weight ? &*q_weight : nullptr, k_weight ? &*k_weight : nullptr})
      if (t) { check_apart(qo, "q_out", *t, "another input"); check_apart(ko, "k_out", *t, "another input"); }
  }
  q = rope_input(q); k = rope_input(k);
  rope_status(dh_qk_norm_rope_fwd(TOKEN_VIEW(q), TOKEN_VIEW(k), TOKEN_VIEW(qo), TOKEN_VIEW(ko), positions.data_ptr(), a.pos_type,
                                  inv_freq.data_ptr<float>(), a.sections.data(), (int)a.sections.size(), a.qw, a.kw, a.w_dtype, dt, q.size(0), (int)q.size(1), (int)k.size(1),
                                  (int)q.size(2), normalize, (float)eps, interleaved, stream_of(q)), "qk_norm_rope_forward");
  if (q_out) mark_written(qo);
  if (k_out) mark_written(ko);
  return {qo, ko};
}

// {dq, dk, dq_weight, dk_weight}; the weights' gradients are None where there is no weight
std::vector<torch::Tensor> qk_norm_rope_backward(torch::Tensor dq_out, torch::Tensor dk_out, torch::Tensor q, torch::Tensor k, torch::Tensor positions, torch::Tensor inv_freq,
                                                 const std::vector<int64_t>& sections, c10::optional<torch::Tensor> q_weight, c10::optional<torch::Tensor> k_weight,
                                                 bool normalize, double eps, bool interleaved) {
  const RopeArgs a = rope_args(q, k, positions, inv_freq, sections, q_weight, k_weight, normalize, eps);
  check_no_tangents({&dq_out, &dk_out});
  check_heads(dq_out, "dq_out", q); check_heads(dk_out, "dk_out", q);
  TORCH_CHECK(dq_out.sizes() == q.sizes() && dk_out.sizes() == k.sizes(), "the gradients must have the shapes of q and k");
  const int dt = token_dtype(q, "q", true);
  const c10::DeviceGuard guard(q.device());
  q = rope_input(q); k = rope_input(k); dq_out = rope_input(dq_out); dk_out = rope_input(dk_out);
  torch::Tensor dq = torch::empty(q.sizes(), q.options()), dk = torch::empty(k.sizes(), k.options());
  torch::Tensor dqw, dkw, ws;
  if (q_weight) dqw = torch::empty_like(*q_weight);
  if (k_weight) dkw = torch::empty_like(*k_weight);
  const size_t wsb = q_weight || k_weight ? dh_qk_norm_rope_bwd_workspace_bytes((int)q.size(2)) : 0;
  if (wsb) ws = torch::empty({(int64_t)wsb}, q.options().dtype(torch::kUInt8));
  rope_status(dh_qk_norm_rope_bwd(TOKEN_VIEW(dq_out), TOKEN_VIEW(dk_out), TOKEN_VIEW(q), TOKEN_VIEW(k), TOKEN_VIEW(dq), TOKEN_VIEW(dk), q_weight ? dqw.data_ptr() : nullptr,
                                  k_weight ? dkw.data_ptr() : nullptr, positions.data_ptr(), a.pos_type, inv_freq.data_ptr<float>(), a.sections.data(), (int)a.sections.size(),
                                  a.qw, a.kw, a.w_dtype, dt, q.size(0), (int)q.size(1), (int)k.size(1), (int)q.size(2), normalize, (float)eps, interleaved, wsb ? ws.data_ptr() : nullptr, wsb,
                                  stream_of(q)), "qk_norm_rope_backward");
  return {dq, dk, dqw, dkw};
}

struct QkNormRope : public torch::autograd::Function<QkNormRope> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, torch::Tensor q, torch::Tensor k, torch::Tensor positions, torch::Tensor inv_freq,
                                                c10::optional<torch::Tensor> q_weight, c10::optional<torch::Tensor> k_weight, std::vector<int64_t> sections, bool normalize,
                                                double eps, bool interleaved) {
    auto r = qk_norm_rope_forward(q, k, positions, inv_freq, sections, q_weight, k_weight, normalize, eps, interleaved, c10::nullopt, c10::nullopt);
    // (a rotation alone needs no input for its gradient)
    ctx->save_for_backward({normalize ? q : torch::Tensor(), normalize ? k : torch::Tensor(), positions, inv_freq, q_weight.value_or(torch::Tensor()), k_weight.value_or(torch::Tensor())});
    ctx->saved_data["sections"] = sections;
    ctx->saved_data["normalize"] = normalize;
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["interleaved"] = interleaved;
    return {r[0], r[1]};
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    TORCH_CHECK(!at::GradMode::is_enabled(), "qk_norm_rope is differentiable once (create_graph is not supported)");
    const auto s = ctx->get_saved_variables();
    const bool normalize = ctx->saved_data["normalize"].toBool();
    const auto opt = [](const torch::Tensor& t) { return t.defined() ? c10::optional<torch::Tensor>(t) : c10::nullopt; };
    auto r = qk_norm_rope_backward(grads[0], grads[1], normalize ? s[0] : grads[0], normalize ? s[1] : grads[1], s[2], s[3], ctx->saved_data["sections"].toIntVector(), opt(s[4]),
                                   opt(s[5]), normalize, ctx->saved_data["eps"].toDouble(), ctx->saved_data["interleaved"].toBool());
    const torch::Tensor none;
    return {r[0], r[1], none, none, s[4].defined() ? r[2] : none, s[5].defined() ? r[3] : none, none, none, none, none};
  }
};
std::vector<torch::Tensor> qk_norm_rope(torch::Tensor q, torch::Tensor k, torch::Tensor positions, torch::Tensor inv_freq, const std::vector<int64_t>& sections,
                                        c10::optional<torch::Tensor> q_weight, c10::optional<torch::Tensor> k_weight, bool normalize, double eps, bool interleaved) {
  refuse_leaves_of_other_streams({&q, &k, q_weight ? &*q_weight : nullptr, k_weight ? &*k_weight : nullptr}, "qk_norm_rope");
  return QkNormRope::apply(q, k, positions, inv_freq, q_weight, k_weight, sections, normalize, eps, interleaved);
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  // bundle adjustment kernels (names and order as reference src/droid.cpp:246-259)
  m.def("ba", &ba, "bundle adjustment");
  m.def("frame_distance", &frame_distance, "frame_distance");
  m.def("projmap", &projmap, "projmap");
  m.def("depth_filter", &depth_filter, "depth_filter");
  m.def("iproj", &iproj, "back projection");
  // correlation volume kernels
  m.def("altcorr_forward", &altcorr_forward, "ALTCORR forward");
  m.def("altcorr_backward", &altcorr_backward, "ALTCORR backward");
  m.def("corr_index_forward", &corr_index_forward, "INDEX forward");
  m.def("corr_index_backward", &corr_index_backward, "INDEX backward");
  // MI355X extensions (not in the reference module)
  m.def("ba_ex", &ba_ex, "bundle adjustment with a per-pixel depth-prior weight");
  m.def("ba_build", &ba_build, "per-rank reduced camera system (split BA)");
  m.def("ba_depth_blocks", &ba_depth_blocks, "views of Qinv = 1/C, w, kx, K in the workspace of ba_build (the keep-alive is the caller's: hold `ws`)");
  m.def("ba_finish", &ba_finish, "damp + solve + back-substitute + retract (split BA)");
  m.def("ba_build_shard", &ba_build_shard, "ba_build without a host synchronisation (edge-sharded BA)");
  m.def("ba_build_shard_ex", &ba_build_shard_ex, "ba_build_shard with a per-pixel depth-prior weight");
  m.def("ba_finish_owned", &ba_finish_owned, "ba_finish that only moves the depths of frames [own_lo, own_hi)");
  m.def("ba_pack_blocks", &ba_pack_blocks, "co-visible 6x6 blocks + rhs + flags -> one contiguous f64 buffer");
  m.def("ba_unpack_blocks", &ba_unpack_blocks, "all-reduced buffer -> system + flags");
  m.def("ba_exchange_flags", &ba_exchange_flags, "argument / pattern flags of the dense exchange");
  m.def("altcorr_forward_nhwc_levels", &altcorr_forward_nhwc_levels, "all pyramid levels of the on-the-fly correlation into one [M,49L,H,W] tensor");
  m.def("altcorr_forward_nhwc", &altcorr_forward_nhwc, "on-the-fly correlation on the fp16 MFMA, channel-last features");
  m.def("corr_volume_build", &corr_volume_build, "all-pairs volume in the reference layout (any image size)");
  m.def("corr_volume_pool", &corr_volume_pool, "2x2 average pooling of the last two dims of a reference-layout volume");
  m.def("corr_pyramid_build", &corr_pyramid_build, "all-pairs correlation pyramid, MI355X layout", py::arg("fmap1"), py::arg("fmap2"),
        py::arg("h_real") = 0, py::arg("w_real") = 0, py::arg("out") = py::none());
  m.def("corr_pyramid_prepare_frames", &corr_pyramid_prepare_frames, "channel-last transpose + pooled levels once per frame", py::arg("fmaps"),
        py::arg("h_real") = 0, py::arg("w_real") = 0);
  m.def("corr_pyramid_build_indexed", &corr_pyramid_build_indexed, "pyramid of edges (idx1[e], idx2[e]) from prepared frames", py::arg("prepared"),
        py::arg("idx1"), py::arg("idx2"), py::arg("h"), py::arg("w"), py::arg("out") = py::none());
  m.def("corr_pyramid_lookup", &corr_pyramid_lookup, "fused 4-level lookup on the MI355X pyramid");
  m.def("corr_pyramid_lookup_nhwc", &corr_pyramid_lookup_nhwc, "fused 4-level lookup, channel-last output for the update operator");
  m.def("corr_pyramid_lookup_corr0", &corr_pyramid_lookup_corr0, "4-level lookup fused with the correlation encoder's first layer (1x1, 196 -> 128, ReLU)");
  m.def("corr0_nchw", &corr0_nchw, "corr_encoder.0 (1x1, 196 -> 128, relu) on the reference-layout lookup output [E,196,h,w] -> [E,h,w,128]");
  m.def("glo_gemv", &glo_gemv, "global-context GEMV of the ConvGRU gates: fp16(bias + fp16(red * scale) wt)");
  m.def("segment_mean", &segment_mean, "mean over row segments (GraphAgg scatter_mean)");
  m.def("conv2d_s2_nhwc", &conv2d_s2_nhwc, "stride-2 same convolution (encoders' down-sampling layers)");
  m.def("conv2d_nhwc", &conv2d_nhwc, "implicit-GEMM NHWC convolution on the fp16 MFMA with fused epilogues",
        py::arg("inputs"), py::arg("weight"), py::arg("weight_halo"), py::arg("bias"), py::arg("KH"), py::arg("KW"), py::arg("Cout"),
        py::arg("epilogue"), py::arg("out"), py::arg("out_stride"), py::arg("gterm"), py::arg("aux0"), py::arg("aux1"), py::arg("red"),
        py::arg("cinit") = py::none(), py::arg("cinit_idx") = py::none(), py::arg("cinit_off") = 0, py::arg("out_raw_f32") = false,
        py::arg("weights_layout") = 0, py::arg("out_tiled") = false, py::arg("cinit_tiled") = false,
        py::arg("glo_weight") = py::none(), py::arg("glo_bias") = py::none(), py::arg("glo_red") = py::none());
  m.def("conv_set_timestamps", [](c10::optional<torch::Tensor> buf) {
    if (buf.has_value() && buf->defined()) {
      CHECK_INPUT((*buf));
      TORCH_CHECK(buf->scalar_type() == torch::kInt64 && buf->dim() == 2 && buf->size(1) == 8, "conv_set_timestamps: int64 [workgroups, 8]");
      check_status(dh_conv_set_timestamps(buf->data_ptr(), (long)buf->size(0)), "conv_set_timestamps");
    } else {
      check_status(dh_conv_set_timestamps(nullptr, 0), "conv_set_timestamps");
    }
  }, "-DDH_ABLATION builds: phase timestamps of the 3x3 convolution kernels into an int64 [workgroups, 8] tensor (None = off)");
  m.def("canvas_mask_", &canvas_mask_, "zero the canvas pixels outside the h x w image (fp16 NHWC, in place)");
  m.def("motion_features", &motion_features, "cat(coords1 - coords0, target - coords1).clamp(-64, 64) as fp16 NHWC");
  m.def("ba_inputs", &ba_inputs, "target = coords1 + delta, weight; also in ba's [E,2,h,w] layout");
  m.def("cvx_upsample", &cvx_upsample, "convex 8x upsampling of depth maps");
  m.def("proximity_nms", &proximity_nms, "candidate masking + greedy NMS of add_proximity_factors on the device");
  m.def("heads_gather", &heads_gather, "second head layer from the fused first layer's partial products",
        py::arg("partials"), py::arg("bias4"), py::arg("H"), py::arg("W"), py::arg("mode") = 0);
  m.def("norm_act", &norm_act, "instance norm / residual add + activation on channel-last fp16 (encoders)");
  m.def("reproject", &reproject, "fused reprojection (Python thresholds)");
  m.def("se3_op", &se3_op, "SE3 inv/mul/exp/retr");
  m.def("se3_map", &se3_map, "SE3 act4/adjT");
  m.def("_token_views_overlap", [](const torch::Tensor& a, const torch::Tensor& b) { return overlap(pieces_of(a), pieces_of(b)); }, "what out= is checked with");
  m.def("_token_view_overlaps_itself", [](const torch::Tensor& a) { return overlaps_itself(pieces_of(a)); }, "what out= is checked with");
  m.def("attention_plan", &attention_plan, "work items of packed attention for one set of lengths", py::arg("q_lengths"), py::arg("k_lengths"), py::arg("k_starts"),
        py::arg("heads"), py::arg("kv_heads"), py::arg("head_dim"), py::arg("causal_block") = 0);
  m.def("attention_forward", &attention_forward, "packed softmax attention: {o, lse, o_low}", py::arg("q"), py::arg("k"), py::arg("v"), py::arg("plan"), py::arg("info"),
        py::arg("scale"), py::arg("out") = py::none(), py::arg("for_backward") = false);
  m.def("attention_backward", &attention_backward, "gradients of packed softmax attention: {dq, dk, dv}");
  m.def("packed_attention", &packed_attention, "attention_forward with a gradient: {o, lse}");
  m.def("qk_norm_rope", &qk_norm_rope, "qk_norm_rope_forward with a gradient: {q, k}");
  m.def("qk_norm_rope_forward", &qk_norm_rope_forward, "norm of query / key heads and rotation by position: {q, k}", py::arg("q"), py::arg("k"), py::arg("positions"),
        py::arg("inv_freq"), py::arg("sections"), py::arg("q_weight") = py::none(), py::arg("k_weight") = py::none(), py::arg("normalize") = true, py::arg("eps") = 1e-6,
        py::arg("interleaved") = false, py::arg("q_out") = py::none(), py::arg("k_out") = py::none());
  m.def("qk_norm_rope_backward", &qk_norm_rope_backward, "gradients of qk_norm_rope_forward: {dq, dk, dq_weight, dk_weight}", py::arg("dq_out"), py::arg("dk_out"),
        py::arg("q"), py::arg("k"), py::arg("positions"), py::arg("inv_freq"), py::arg("sections"), py::arg("q_weight") = py::none(), py::arg("k_weight") = py::none(),
        py::arg("normalize") = true, py::arg("eps") = 1e-6, py::arg("interleaved") = false);
  m.def("version", []() { return std::string(dh_version()); });
  m.def("set_option", [](const std::string& name, int value) { check_status(dh_set_option(name.c_str(), value), "set_option"); });
  m.def("options_epoch", []() { return dh_options_epoch(); });
  m.def("get_option", [](const std::string& name) { int v = 0; check_status(dh_get_option(name.c_str(), &v), "get_option"); return v; });
}
