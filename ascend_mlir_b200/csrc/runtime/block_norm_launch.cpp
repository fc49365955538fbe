#include "runtime/block_norm_launch.h"

#include <algorithm>
#include <cstring>

#include "kernels/block_norm.h"

namespace afir {
namespace {

// Sizes beyond these are refused, so that every product of them, times an element's bytes, fits 63 bits.
constexpr int64_t kMaxRows = 1ll << 36, kMaxRowLength = 1ll << 24;

int elemTypeOf(DType t, bool &ok) {
  ok = true;
  switch (t) {
  case DType::F32: return kernels::kF32;
  case DType::F16: return kernels::kF16;
  case DType::BF16: return kernels::kBF16;
  default: ok = false; return 0;
  }
}

struct Sizes { int64_t rows = 0, cols = 0, outCols = 0, groupRows = 1, groups = 0; };

Status evalSizes(const LaunchDescriptor &d, const std::map<std::string, int64_t> &tiling, Sizes &s) {
  if (Status e = evalDim(d.op.rows, tiling, s.rows); !e) return e;
  if (Status e = evalDim(d.op.cols, tiling, s.cols); !e) return e;
  if (d.kernelClass == KernelClass::CheckpointGrad)
    if (Status e = evalDim(d.op.outCols, tiling, s.outCols); !e) return e;
  if (Status e = evalDim(d.op.groupRows, tiling, s.groupRows); !e) return e;
  if (s.rows > kMaxRows) return Status::error("more than " + std::to_string(kMaxRows) + " rows");
  if (s.cols < 1) return Status::error("rows need at least one column");
  const int64_t most = d.kernelClass == KernelClass::BlockNorm ? kernels::kMaxNormCols : kMaxRowLength;
  if (s.cols > most) return Status::error("rows of " + std::to_string(s.cols) + " columns: at most " + std::to_string(most) + " are supported");
  if (s.outCols > kMaxRowLength) return Status::error("rows of " + std::to_string(s.outCols) + " columns: at most " + std::to_string(kMaxRowLength) + " are supported");
  if (s.groupRows < 1) return Status::error("a gate row serves at least one row");
  s.groups = (s.rows + s.groupRows - 1) / s.groupRows;
  return Status::success();
}

// One argument as a kernel sees it, and the bytes it covers (for the check that outputs keep clear of everything else).
struct Region {
  std::string name;
  char *base = nullptr;
  int64_t rows = 0, width = 0, pitch = 0;  // bytes
  int64_t ld = 0;                          // elements
  bool output = false;
  bool rowTensor = false;  // [rows, cols] of the rows' own type
};

bool overlaps(const Region &a, const Region &b) {
  if (!a.rows || !a.width || !b.rows || !b.width) return false;
  const char *aEnd = a.base + (a.rows - 1) * a.pitch + a.width, *bEnd = b.base + (b.rows - 1) * b.pitch + b.width;
  if (aEnd <= b.base || bEnd <= a.base) return false;
  if (a.pitch == b.pitch && a.pitch > 0) {  // two column ranges of one wide tensor
    int64_t shift = (b.base - a.base) % a.pitch;
    if (shift < 0) shift += a.pitch;
    if (shift >= a.width && shift + b.width <= a.pitch) return false;
  }
  return true;
}

class Binder {
public:
  Binder(const LaunchDescriptor &d, const std::map<std::string, int64_t> &tiling, const LaunchArgs &args) : d_(d), tiling_(tiling), args_(args) {}

  bool has(const char *role) const { return d_.op.roles.count(role) != 0; }

  // The argument in `role` as `rows` rows of `cols` elements of type t (a vector: rows = 1).  Absent and optional: a null region.
  Status bind(const char *role, int64_t rows, int64_t cols, DType t, bool output, bool required, Region &out, bool vector = false) {
    out = Region();
    out.name = role;
    auto it = d_.op.roles.find(role);
    if (it == d_.op.roles.end()) return required ? Status::error(std::string("operator needs an argument in the role '") + role + "'") : Status::success();
    ++bound_;
    const ViewSpec &v = it->second;
    const std::string what = std::string(role) + " (argument " + std::to_string(v.arg) + ")";
    if (v.dtype != t) return Status::error(what + " is declared " + dtypeName(v.dtype) + ", the operator takes " + dtypeName(t));
    if (output != (v.arg >= d_.numInputs)) return Status::error(what + (output ? " must be an output" : " must be an input"));
    const size_t rank = vector ? 1 : 2;
    if (v.shape.size() != rank) return Status::error(what + " must have " + std::to_string(rank) + (vector ? " dim" : " dims"));
    int64_t shape[2] = {1, 1}, offset[2] = {0, 0};
    for (size_t i = 0; i < rank; ++i) {
      const size_t at = vector ? 1 : i;
      if (Status s = evalDim(v.shape[i], tiling_, shape[at]); !s) return s;
      if (!v.offset.empty())
        if (Status s = evalDim(v.offset[i], tiling_, offset[at]); !s) return s;
      const int64_t limit = at == 0 ? kMaxRows : (vector ? kMaxRows : kMaxRowLength);
      if (shape[at] > limit || offset[at] > limit) return Status::error(what + ": a dim is too large");
    }
    if (offset[0] + rows > shape[0] || offset[1] + cols > shape[1])
      return Status::error("[cuda:bindings] " + what + ": " + std::to_string(rows) + " x " + std::to_string(cols) + " from (" + std::to_string(offset[0]) + ", " +
                           std::to_string(offset[1]) + ") exceeds its shape " + std::to_string(shape[0]) + " x " + std::to_string(shape[1]));
    const size_t eb = dtypeBytes(t);
    const unsigned __int128 want = static_cast<unsigned __int128>(shape[0]) * static_cast<unsigned __int128>(shape[1]) * eb;
    const size_t given = args_.argBytes[static_cast<size_t>(v.arg)];
    if (want != given)
      return Status::error("[cuda:bindings] " + what + " is " + std::to_string(given) + " bytes, the tiling dims imply " +
                           std::to_string(static_cast<unsigned long long>(want)));
    out.base = static_cast<char *>(args_.argPtrs[static_cast<size_t>(v.arg)]);
    if (!out.base && rows && cols) return Status::error("[cuda:bindings] " + what + " is null");
    if (reinterpret_cast<uintptr_t>(out.base) % eb) return Status::error("[cuda:bindings] " + what + " is not aligned to its elements");
    if (out.base) out.base += (static_cast<size_t>(offset[0]) * static_cast<size_t>(shape[1]) + static_cast<size_t>(offset[1])) * eb;
    out.rows = rows;
    out.width = cols * static_cast<int64_t>(eb);
    out.ld = shape[1];
    out.pitch = shape[1] * static_cast<int64_t>(eb);
    out.output = output;
    regions_.push_back(out);
    return Status::success();
  }
  Status rowsOf(const char *role, int64_t rows, int64_t cols, bool output, bool required, Region &out) {
    if (Status s = bind(role, rows, cols, d_.dtype, output, required, out); !s) return s;
    if (has(role)) regions_.back().rowTensor = true;
    return Status::success();
  }
  Status vector(const char *role, int64_t n, DType t, bool output, bool required, Region &out) { return bind(role, 1, n, t, output, required, out, true); }

  // Outputs keep clear of every other argument, except that a row tensor may be written in the place of one that is
  // read (same start, same row length: each thread reads its columns of a row before it writes them).
  Status finish(bool inPlace = true) const {
    if (bound_ != d_.op.roles.size()) return Status::error("an argument has a role that this operator does not take");
    for (size_t i = 0; i < regions_.size(); ++i)
      for (size_t j = 0; j < regions_.size(); ++j) {
        const Region &a = regions_[i], &b = regions_[j];
        if (i == j || !a.output || (b.output && j < i) || !overlaps(a, b)) continue;
        const bool same = a.base == b.base && a.pitch == b.pitch && a.width == b.width;
        if (inPlace && same && !b.output && a.rowTensor && b.rowTensor) continue;
        return Status::error("[cuda:bindings] " + a.name + " overlaps " + b.name);
      }
    return Status::success();
  }

private:
  const LaunchDescriptor &d_;
  const std::map<std::string, int64_t> &tiling_;
  const LaunchArgs &args_;
  std::vector<Region> regions_;
  size_t bound_ = 0;
};

kernels::RowsIn rowsIn(const Region &r) { return {r.base, r.ld}; }
kernels::RowsOut rowsOut(const Region &r) { return {r.base, r.ld}; }
float *f32Of(const Region &r) { return reinterpret_cast<float *>(r.base); }
int64_t checkpointBlocks(int64_t cols) { return (cols + kernels::kCheckpointBlock - 1) / kernels::kCheckpointBlock; }

Status bindCheckpoint(Binder &b, const Sizes &s, bool output, bool required, Region &codes, Region &exps) {
  if (b.has("codes") != b.has("exps")) return Status::error("a checkpoint is its codes and its exps");
  if (Status e = b.bind("codes", s.rows, s.cols, DType::U8, output, required, codes); !e) return e;
  return b.bind("exps", s.rows, checkpointBlocks(s.cols), DType::U8, output, required, exps);
}

Status kernelStatus(int code, const char *what) {
  if (code == 0) return Status::success();
  return Status::error(std::string(what) + ": " + kernels::cudaErrorText(code));
}

// Scratch behind the status block.
Status scratch(const LaunchArgs &args, size_t need, void *&at, size_t &bytes) {
  at = nullptr;
  bytes = 0;
  if (!args.workspace || args.workspaceBytes < kWorkspaceStatusBytes + need)
    return Status::error("needs " + std::to_string(kWorkspaceStatusBytes + need) + " workspace bytes, " + std::to_string(args.workspaceBytes) + " given");
  if (reinterpret_cast<uintptr_t>(args.workspace) % 16) return Status::error("[cuda:memory] the workspace must be 16-byte aligned");
  at = static_cast<char *>(args.workspace) + kWorkspaceStatusBytes;
  bytes = args.workspaceBytes - kWorkspaceStatusBytes;
  return Status::success();
}

// `rstd` and, for a layer norm, `mean`: both or neither where they are optional.
Status bindStats(Binder &b, const std::string &prefix, const Sizes &s, bool layer, bool output, bool required, Region &rstd, Region &mean) {
  const std::string r = prefix + "rstd", m = prefix + "mean";
  if (Status e = b.vector(r.c_str(), s.rows, DType::F32, output, required, rstd); !e) return e;
  if (!layer) return Status::success();
  if (b.has(r.c_str()) != b.has(m.c_str())) return Status::error("a layer norm's statistics are " + r + " and " + m);
  return b.vector(m.c_str(), s.rows, DType::F32, output, required, mean);
}

Status launchNormForward(const LaunchDescriptor &d, const Sizes &s, const std::map<std::string, int64_t> &tiling, const LaunchArgs &args, LaunchInfo &info) {
  const OperatorSpec &o = d.op;
  bool ok1, ok2;
  kernels::BlockNormLaunch l = {};
  l.elemType = elemTypeOf(d.dtype, ok1);
  l.paramType = elemTypeOf(o.paramType, ok2);
  if (!ok1 || !ok2) return Status::error("block norms take f32, f16 or bf16");
  if (o.paramType != d.dtype && o.paramType != DType::F32) return Status::error("parameters are f32 or of the rows' type");
  const bool layer = o.kind == kernels::kLayerNorm, post = o.pass != kernels::kPre, pre = o.pass != kernels::kPost;
  Binder b(d, tiling, args);
  Region x, y, w, bias, gate, scale, nw, nb, out, h, rstd, mean, nrstd, nmean, codes, exps;
  if (Status e = b.rowsOf("x", s.rows, s.cols, false, true, x); !e) return e;
  if (Status e = b.vector("weight", s.cols, o.paramType, false, true, w); !e) return e;
  if (layer)
    if (Status e = b.vector("bias", s.cols, o.paramType, false, true, bias); !e) return e;
  if (post) {
    if (Status e = b.rowsOf("y", s.rows, s.cols, false, true, y); !e) return e;
    if (Status e = b.rowsOf("out", s.rows, s.cols, true, true, out); !e) return e;
    if (o.gateForm == kernels::kGateToken)
      if (Status e = b.rowsOf("gate", s.rows, s.cols, false, true, gate); !e) return e;
    if (o.gateForm == kernels::kGateGroup)
      if (Status e = b.bind("gate", s.groups, s.cols, d.dtype, false, true, gate); !e) return e;
    if (Status e = b.vector("scale", s.cols, o.paramType, false, false, scale); !e) return e;
  }
  if (pre)
    if (Status e = b.rowsOf("h", s.rows, s.cols, true, true, h); !e) return e;
  if (post && pre) {
    if (Status e = b.vector("next_weight", s.cols, o.paramType, false, true, nw); !e) return e;
    if (layer)
      if (Status e = b.vector("next_bias", s.cols, o.paramType, false, true, nb); !e) return e;
    if (Status e = bindStats(b, "next_", s, layer, true, false, nrstd, nmean); !e) return e;
  }
  if (Status e = bindStats(b, "", s, layer, true, false, rstd, mean); !e) return e;
  if (Status e = bindCheckpoint(b, s, true, false, codes, exps); !e) return e;
  if (Status e = b.finish(); !e) return e;

  l.pass = o.pass;
  l.kind = o.kind;
  l.rows = s.rows;
  l.cols = s.cols;
  l.x = rowsIn(x);
  l.y = rowsIn(y);
  l.out = rowsOut(out);
  l.h = rowsOut(h);
  const kernels::NormVectors first = {w.base, bias.base};
  const kernels::NormStatsOut firstStats = {f32Of(rstd), f32Of(mean)};
  if (post) {
    l.a = first;
    l.statsA = firstStats;
    l.b = {nw.base, nb.base};
    l.statsB = {f32Of(nrstd), f32Of(nmean)};
    l.epsA = static_cast<float>(o.eps);
    l.epsB = static_cast<float>(o.nextEps);
  } else {
    l.b = first;
    l.statsB = firstStats;
    l.epsB = static_cast<float>(o.eps);
  }
  l.gateForm = o.gateForm;
  l.gateAct = o.gateAct;
  l.gate = rowsIn(gate);
  l.groupRows = s.groupRows;
  l.scale = scale.base;
  l.alpha = static_cast<float>(o.alpha);
  l.checkpoint = {reinterpret_cast<uint8_t *>(codes.base), codes.ld, reinterpret_cast<uint8_t *>(exps.base), exps.ld};
  return kernelStatus(kernels::launchBlockNorm(l, args.stream, &info.kernelsLaunched), "block norm launch");
}

Status launchNormGrad(const LaunchDescriptor &d, const Sizes &s, const std::map<std::string, int64_t> &tiling, const LaunchArgs &args, LaunchInfo &info) {
  const OperatorSpec &o = d.op;
  bool ok1, ok2;
  kernels::BlockNormGradLaunch l = {};
  l.elemType = elemTypeOf(d.dtype, ok1);
  l.paramType = elemTypeOf(o.paramType, ok2);
  if (!ok1 || !ok2) return Status::error("block norms take f32, f16 or bf16");
  if (o.paramType != d.dtype && o.paramType != DType::F32) return Status::error("parameters are f32 or of the rows' type");
  const bool layer = o.kind == kernels::kLayerNorm, post = o.pass != kernels::kPre, pre = o.pass != kernels::kPost;
  Binder b(d, tiling, args);
  Region dout, dh, source, y, w, bias, gate, scale, nw, rstd, mean, nrstd, nmean, codes, exps;
  Region dx, dy, dw, db, dgate, dscale, dnw, dnb;
  const bool packed = b.has("codes");
  if (Status e = b.rowsOf("dout", s.rows, s.cols, false, o.pass == kernels::kPost, dout); !e) return e;
  if (Status e = b.rowsOf("dx", s.rows, s.cols, true, true, dx); !e) return e;
  if (pre)
    if (Status e = b.rowsOf("dh", s.rows, s.cols, false, true, dh); !e) return e;
  if (Status e = bindCheckpoint(b, s, false, false, codes, exps); !e) return e;
  if (!post && !packed)
    if (Status e = b.rowsOf("x", s.rows, s.cols, false, true, source); !e) return e;
  if (Status e = b.vector("weight", s.cols, o.paramType, false, true, w); !e) return e;
  if (Status e = b.vector("dweight", s.cols, DType::F32, true, true, dw); !e) return e;
  if (layer)
    if (Status e = b.vector("dbias", s.cols, DType::F32, true, true, db); !e) return e;
  if (Status e = bindStats(b, "", s, layer, false, true, rstd, mean); !e) return e;
  if (post) {
    if (!packed)
      if (Status e = b.rowsOf("y", s.rows, s.cols, false, true, y); !e) return e;
    if (Status e = b.rowsOf("dy", s.rows, s.cols, true, true, dy); !e) return e;
    if (layer)
      if (Status e = b.vector("bias", s.cols, o.paramType, false, true, bias); !e) return e;
    if (o.gateForm == kernels::kGateToken) {
      if (Status e = b.rowsOf("gate", s.rows, s.cols, false, true, gate); !e) return e;
      if (Status e = b.rowsOf("dgate", s.rows, s.cols, true, true, dgate); !e) return e;
    }
    if (o.gateForm == kernels::kGateGroup) {
      if (Status e = b.bind("gate", s.groups, s.cols, d.dtype, false, true, gate); !e) return e;
      if (Status e = b.bind("dgate", s.groups, s.cols, DType::F32, true, true, dgate); !e) return e;
    }
    if (b.has("scale") != b.has("dscale")) return Status::error("a residual scale has a gradient: 'scale' and 'dscale' come together");
    if (Status e = b.vector("scale", s.cols, o.paramType, false, false, scale); !e) return e;
    if (Status e = b.vector("dscale", s.cols, DType::F32, true, false, dscale); !e) return e;
  }
  if (post && pre) {
    if (Status e = b.rowsOf("out", s.rows, s.cols, false, true, source); !e) return e;
    if (Status e = b.vector("next_weight", s.cols, o.paramType, false, true, nw); !e) return e;
    if (Status e = bindStats(b, "next_", s, layer, false, true, nrstd, nmean); !e) return e;
    if (Status e = b.vector("dnext_weight", s.cols, DType::F32, true, true, dnw); !e) return e;
    if (layer)
      if (Status e = b.vector("dnext_bias", s.cols, DType::F32, true, true, dnb); !e) return e;
  }
  if (Status e = b.finish(); !e) return e;

  l.pass = o.pass;
  l.kind = o.kind;
  l.rows = s.rows;
  l.cols = s.cols;
  l.dout = rowsIn(dout);
  l.dh = rowsIn(dh);
  l.source = rowsIn(source);
  l.y = rowsIn(y);
  l.checkpoint = {reinterpret_cast<const uint8_t *>(codes.base), codes.ld, reinterpret_cast<const uint8_t *>(exps.base), exps.ld};
  const kernels::NormVectors first = {w.base, bias.base};
  const kernels::NormStatsIn firstStats = {f32Of(rstd), f32Of(mean)};
  const kernels::NormSums firstSums = {f32Of(dw), f32Of(db)};
  if (post) {
    l.a = first;
    l.statsA = firstStats;
    l.da = firstSums;
    l.b = {nw.base, nullptr};
    l.statsB = {f32Of(nrstd), f32Of(nmean)};
    l.db = {f32Of(dnw), f32Of(dnb)};
  } else {
    l.b = first;
    l.statsB = firstStats;
    l.db = firstSums;
  }
  l.gateForm = o.gateForm;
  l.gateAct = o.gateAct;
  l.gate = rowsIn(gate);
  l.groupRows = s.groupRows;
  l.scale = scale.base;
  l.alpha = static_cast<float>(o.alpha);
  l.dx = rowsOut(dx);
  l.dy = rowsOut(dy);
  l.dgate = rowsOut(dgate);
  l.dscale = f32Of(dscale);
  size_t need = 0;
  if (Status e = operatorWorkspaceBytes(d, tiling, args.device, need); !e) return e;
  if (Status e = scratch(args, need - kWorkspaceStatusBytes, l.workspace, l.workspaceBytes); !e) return e;
  return kernelStatus(kernels::launchBlockNormGrad(l, args.stream, &info.kernelsLaunched), "block norm gradient launch");
}

Status launchCheckpoint(const LaunchDescriptor &d, const Sizes &s, const std::map<std::string, int64_t> &tiling, const LaunchArgs &args, LaunchInfo &info) {
  bool ok;
  const int elemType = elemTypeOf(d.dtype, ok);
  if (!ok) return Status::error("checkpoints hold f32, f16 or bf16");
  Binder b(d, tiling, args);
  Region x, codes, exps;
  if (Status e = b.rowsOf("x", s.rows, s.cols, d.op.gradient, true, x); !e) return e;
  if (Status e = bindCheckpoint(b, s, !d.op.gradient, true, codes, exps); !e) return e;
  if (Status e = b.finish(); !e) return e;
  if (d.op.gradient) {
    kernels::CheckpointRestoreLaunch l = {};
    l.elemType = elemType;
    l.rows = s.rows;
    l.cols = s.cols;
    l.in = {reinterpret_cast<const uint8_t *>(codes.base), codes.ld, reinterpret_cast<const uint8_t *>(exps.base), exps.ld};
    l.out = rowsOut(x);
    return kernelStatus(kernels::launchCheckpointRestore(l, args.stream, &info.kernelsLaunched), "checkpoint restore launch");
  }
  kernels::CheckpointPackLaunch l = {};
  l.elemType = elemType;
  l.rows = s.rows;
  l.cols = s.cols;
  l.x = rowsIn(x);
  l.out = {reinterpret_cast<uint8_t *>(codes.base), codes.ld, reinterpret_cast<uint8_t *>(exps.base), exps.ld};
  return kernelStatus(kernels::launchCheckpointPack(l, args.stream, &info.kernelsLaunched), "checkpoint pack launch");
}

} // namespace

Status operatorWorkspaceBytes(const LaunchDescriptor &d, const std::map<std::string, int64_t> &tiling, int device, size_t &bytes) {
  bytes = kWorkspaceStatusBytes;
  Sizes s;
  if (Status e = evalSizes(d, tiling, s); !e) return e;
  const int sms = kernels::deviceSmCount(device);
  if (d.kernelClass == KernelClass::BlockNorm && d.op.gradient)
    bytes += kernels::blockNormGradWorkspaceBytes(d.op.pass, d.op.kind, d.op.gateForm, s.rows, s.cols, s.groupRows, sms);
  return Status::success();
}

Status launchOperator(const LaunchDescriptor &d, const std::map<std::string, int64_t> &tiling, const LaunchArgs &args, LaunchInfo &info) {
  if (args.rowEnd >= 0) return Status::error("operator kernels do not take a row range");
  Sizes s;
  if (Status e = evalSizes(d, tiling, s); !e) return e;
  if (d.kernelClass == KernelClass::BlockNorm)
    return d.op.gradient ? launchNormGrad(d, s, tiling, args, info) : launchNormForward(d, s, tiling, args, info);
  if (d.kernelClass == KernelClass::Checkpoint) return launchCheckpoint(d, s, tiling, args, info);
  return Status::error("unsupported kernel class");
}

} // namespace afir
