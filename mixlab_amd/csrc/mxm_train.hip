// C ABI of the handles around the MoE op's training step (declared in
// include/mixmoe.h): residual norms and gradient sets.  Same conventions as
// the op's handles (mxm_abi.hip): int64 handles, status codes, an exception
// fence around every entry point; every argument is checked before the device
// is touched.
#include <algorithm>
#include <cmath>
#include <map>
#include <mutex>
#include <vector>

#include "../../include/mixmoe.h"
#include "mxm_host.h"
#include "mxm_train.h"

namespace {

struct TrainHandle {
  std::shared_ptr<StreamRef> stream_ref;
  int n_cu = 256;
  virtual ~TrainHandle() = default;
  hipStream_t stream() const { return stream_ref->stream; }
};

struct ResNorm : TrainHandle {
  ResNormArgs base{};  // what every call shares
  int64_t max_rows = 0;
  bool backward = false;
  DevBuf part, gate_part;
  // (the destructor's wait keeps the workspace until the calls that use it end)
  ~ResNorm() override {
    if (stream_ref) (void)hipStreamSynchronize(stream());
  }
};

struct GradSet : TrainHandle {
  struct Tensor {
    int64_t n;
    bool bf16;
    float decay;
  };
  std::vector<Tensor> tensors;
  GradArgs base{};
  DevBuf chunks, partial, small;  // small: ticket, then the scalars at byte 64
  bool bound = false, has_params = false;
  ~GradSet() override {
    if (stream_ref) (void)hipStreamSynchronize(stream());
  }
};

std::mutex g_train_mu;
std::map<int64_t, std::shared_ptr<TrainHandle>> g_train;

std::shared_ptr<TrainHandle> find(int64_t h) {
  std::lock_guard<std::mutex> lk(g_train_mu);
  const auto it = g_train.find(h);
  return it == g_train.end() ? nullptr : it->second;
}
template <class T>
std::shared_ptr<T> get(int64_t h) {
  return std::dynamic_pointer_cast<T>(find(h));
}

std::shared_ptr<StreamRef> stream_of_handle(int64_t h) {
  if (auto s = mxm_op_stream(h)) return s;
  const auto t = find(h);
  return t ? t->stream_ref : nullptr;
}

// Makes `dev` current for a call and puts the caller's device back.
struct DeviceGuard {
  int prev = -1;
  bool moved = false;
  explicit DeviceGuard(int dev) {
    HIPCK(hipGetDevice(&prev));
    if (prev != dev) {
      HIPCK(hipSetDevice(dev));
      moved = true;
    }
  }
  ~DeviceGuard() {
    if (moved) (void)hipSetDevice(prev);
  }
};

int64_t keep(std::shared_ptr<TrainHandle> t) {
  const int64_t h = mxm_new_handle();
  std::lock_guard<std::mutex> lk(g_train_mu);
  g_train[h] = std::move(t);
  return h;
}

template <class T>
int destroy(int64_t h, const char* what) {
  return fenced([&] {
    std::shared_ptr<TrainHandle> victim;
    {
      std::lock_guard<std::mutex> lk(g_train_mu);
      const auto it = g_train.find(h);
      if (it == g_train.end() || !dynamic_cast<T*>(it->second.get())) {
        g_last_error = std::string(what) + " invalid handle";
        return MXM_ERR_OP;
      }
      victim = std::move(it->second);
      g_train.erase(it);
    }
    return MXM_OK;
  });
}

#define HANDLE_OR_RETURN(T, var, h, what)          \
  const std::shared_ptr<T> var = get<T>(h);        \
  if (!var) {                                      \
    g_last_error = what " invalid handle";         \
    return MXM_ERR_OP;                             \
  }

bool float_dtype(int64_t t) { return t == MXM_DTYPE_F32 || t == MXM_DTYPE_BF16; }

void check_pointer(const char* what, const char* name, const void* p, bool bf16, bool required) {
  if (!p && required) fail("%s %s must be non-NULL", what, name);
  if (reinterpret_cast<uintptr_t>(p) % (bf16 ? 2 : 4) != 0)
    fail("%s %s is not aligned to its elements", what, name);
}

enum : unsigned { ROWS = 1, POST = 2, SCALE = 4, GATE = 8, NORM = 16 };

// Where a call's tensors lie.  An output may be one of the inputs that it is
// computed beside, element for element (`in_place`, a mask of kinds), and rows of
// results may take each other's place (the thread that stores both leaves the
// later one); every other overlap of an output is refused.
struct Tensors {
  struct One {
    const char* name;
    uintptr_t from, to;
    int item;
    unsigned kind;
    unsigned in_place;  // of an output: kinds of inputs
  };
  One all[14];
  int n = 0;
  void add(const char* name, const void* p, int64_t elements, bool bf16, unsigned kind, unsigned in_place) {
    if (!p || elements <= 0) return;
    const uintptr_t from = reinterpret_cast<uintptr_t>(p);
    const int item = bf16 ? 2 : 4;
    all[n++] = {name, from, from + (uintptr_t)elements * item, item, kind, in_place};
  }
  void in(const char* name, const void* p, int64_t elements, bool bf16, unsigned kind) {
    add(name, p, elements, bf16, kind, 0);
  }
  void out(const char* name, const void* p, int64_t elements, bool bf16, unsigned in_place) {
    add(name, p, elements, bf16, in_place & ROWS, in_place);
  }
  void check(const char* what) const {
    for (int i = 0; i < n; ++i) {
      const One& o = all[i];
      if (!o.in_place) continue;
      for (int j = 0; j < n; ++j) {
        const One& t = all[j];
        if (i == j || t.from >= o.to || o.from >= t.to) continue;
        if ((o.in_place & t.kind) && t.from == o.from && t.to == o.to && t.item == o.item) continue;
        fail("%s %s overlaps %s", what, o.name, t.name);
      }
    }
  }
};
// The stream of `stream_of`, or a new one on the current device.
std::shared_ptr<StreamRef> choose_stream(std::shared_ptr<StreamRef> shared) {
  if (shared) return shared;
  int dev = 0;
  HIPCK(hipGetDevice(&dev));
  return std::make_shared<StreamRef>(dev);
}

std::shared_ptr<StreamRef> shared_stream(const char* what, int64_t stream_of) {
  if (stream_of == 0) return nullptr;
  auto s = stream_of_handle(stream_of);
  if (!s) fail("%s stream_of %lld is not a live handle", what, (long long)stream_of);
  return s;
}

int64_t gate_elements(const ResNormArgs& a, int64_t rows) {
  return a.gate ? (rows + a.gate_rows - 1) / a.gate_rows * (a.gate == 2 ? a.D : 1) : 0;
}

int cu_count(int device) {
  int n = 0;
  HIPCK(hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, device));
  return n;
}

#define RESNORM "RESIDUAL_NORM"
#define GRADSET "GRADIENT_SET"

}  // namespace

extern "C" {

int64_t mxm_resnorm_create(const int64_t* params, int n_params, float eps, int64_t stream_of) {
  int64_t handle = 0;
  const int rc = fenced([&] {
    if (!params || n_params < 10)
      fail(RESNORM " requires D,maxRows,streamDtype,branchDtype,outDtype,scaleDtype,gradDtype,"
                   "flags,gate,gateRows");
    const int64_t D = params[0], rows = params[1], flags = params[7], gate = params[8],
                  gate_rows = params[9];
    if (D < 1 || D > MXM_RESNORM_MAX_D || rows < 0 || rows > ((int64_t)1 << 30))
      fail(RESNORM " invalid dimensions (D in [1,%d], maxRows in [0,2^30])", MXM_RESNORM_MAX_D);
    for (int i = 2; i < 7; ++i)
      if (!float_dtype(params[i]))
        fail(RESNORM " dtype %lld unsupported (want fp32 or bf16)", (long long)params[i]);
    const int64_t all = MXM_RESNORM_BRANCH | MXM_RESNORM_POST_NORM | MXM_RESNORM_NORM |
                        MXM_RESNORM_GATE_SIGMOID | MXM_RESNORM_BACKWARD;
    if (flags & ~all) fail(RESNORM " unknown flags 0x%llx", (unsigned long long)(flags & ~all));
    const bool branch = flags & MXM_RESNORM_BRANCH, post = flags & MXM_RESNORM_POST_NORM;
    if (!branch && !(flags & MXM_RESNORM_NORM))
      fail(RESNORM " needs MXM_RESNORM_BRANCH or MXM_RESNORM_NORM");
    if (!branch && (post || gate != MXM_GATE_NONE))
      fail(RESNORM " post norm and gate need MXM_RESNORM_BRANCH");
    if (gate < MXM_GATE_NONE || gate > MXM_GATE_CHANNEL) fail(RESNORM " unsupported gate kind");
    if (gate == MXM_GATE_NONE && (flags & MXM_RESNORM_GATE_SIGMOID))
      fail(RESNORM " MXM_RESNORM_GATE_SIGMOID needs a gate");
    if (gate != MXM_GATE_NONE && (gate_rows < 1 || gate_rows > ((int64_t)1 << 30)))
      fail(RESNORM " gateRows must be in [1,2^30]");
    if (!(eps >= 0.0f) || !std::isfinite(eps)) fail(RESNORM " eps must be finite and >= 0");
    auto shared = shared_stream(RESNORM, stream_of);

    auto r = std::make_shared<ResNorm>();
    const DeviceGuard guard(shared ? shared->device : [] {
      int dev = 0;
      HIPCK(hipGetDevice(&dev));
      return dev;
    }());
    r->stream_ref = choose_stream(shared);
    r->n_cu = cu_count(r->stream_ref->device);
    r->max_rows = rows;
    r->backward = (flags & MXM_RESNORM_BACKWARD) != 0;
    ResNormArgs& a = r->base;
    a.D = (int)D;
    a.eps = eps;
    a.inv_d = (float)(1.0 / (double)D);
    a.n_cu = r->n_cu;
    a.branch = branch;
    a.post_norm = post;
    a.norm = (flags & MXM_RESNORM_NORM) != 0;
    a.sigmoid = (flags & MXM_RESNORM_GATE_SIGMOID) != 0;
    a.x_bf16 = params[2] == MXM_DTYPE_BF16;
    a.delta_bf16 = params[3] == MXM_DTYPE_BF16;
    a.y_bf16 = params[4] == MXM_DTYPE_BF16;
    a.p_bf16 = params[5] == MXM_DTYPE_BF16;
    a.g_bf16 = params[6] == MXM_DTYPE_BF16;
    a.gate = (int)gate;
    a.gate_rows = gate == MXM_GATE_NONE ? 1 : (int)gate_rows;
    if (r->backward) {
      a.max_parts = (int)mxm_resnorm_max_parts(rows, a.D, a.x_bf16 && a.g_bf16, a.gate_rows > 1,
                                               a.n_cu);
      const size_t parts = (size_t)a.max_parts;
      r->part.alloc(2 * parts * (size_t)D * 4);
      if (a.gate && a.gate_rows > 1)
        r->gate_part.alloc(parts * (size_t)(gate == MXM_GATE_CHANNEL ? D : 1) * 4);
      a.part = r->part.as<float>();
      a.gate_part = r->gate_part.as<float>();
    }
    handle = keep(std::move(r));
    return MXM_OK;
  });
  return rc == MXM_OK ? handle : 0;
}

int mxm_resnorm_destroy(int64_t h) { return destroy<ResNorm>(h, RESNORM); }

int mxm_resnorm_forward(int64_t h, int64_t rows, const void* x, const void* delta,
                        const void* post_scale, const void* branch_scale, const void* gate,
                        const void* norm_scale, void* h_out, void* y) {
  HANDLE_OR_RETURN(ResNorm, r, h, RESNORM);
  return fenced([&] {
    ResNormArgs a = r->base;
    if (rows < 0 || rows > r->max_rows)
      fail(RESNORM " rows %lld out of range [0,%lld]", (long long)rows, (long long)r->max_rows);
    const bool any = rows > 0;
    check_pointer(RESNORM, "x", x, a.x_bf16, any);
    check_pointer(RESNORM, "delta", delta, a.delta_bf16, any && a.branch);
    check_pointer(RESNORM, "h", h_out, a.x_bf16, any && a.branch);
    check_pointer(RESNORM, "y", y, a.y_bf16, any && a.norm);
    check_pointer(RESNORM, "gate", gate, a.p_bf16, any && a.gate != 0);
    check_pointer(RESNORM, "post_scale", post_scale, a.p_bf16, false);
    check_pointer(RESNORM, "branch_scale", branch_scale, a.p_bf16, false);
    check_pointer(RESNORM, "norm_scale", norm_scale, a.p_bf16, false);
    if (post_scale && !a.post_norm) fail(RESNORM " post_scale given without MXM_RESNORM_POST_NORM");
    if (branch_scale && !a.branch) fail(RESNORM " branch_scale given without MXM_RESNORM_BRANCH");
    if (norm_scale && !a.norm) fail(RESNORM " norm_scale given without MXM_RESNORM_NORM");
    const int64_t n = rows * a.D, gates = gate_elements(a, rows);
    Tensors t;
    t.in("x", x, n, a.x_bf16, ROWS);
    if (a.branch) t.in("delta", delta, n, a.delta_bf16, ROWS);
    t.in("post_scale", post_scale, a.D, a.p_bf16, POST);
    t.in("branch_scale", branch_scale, a.D, a.p_bf16, SCALE);
    t.in("norm_scale", norm_scale, a.D, a.p_bf16, NORM);
    t.in("gate", gate, gates, a.p_bf16, GATE);
    if (a.branch) t.out("h", h_out, n, a.x_bf16, ROWS);
    if (a.norm) t.out("y", y, n, a.y_bf16, ROWS);
    t.check(RESNORM);
    const DeviceGuard guard(r->stream_ref->device);
    a.N = (int)rows;
    a.x = x;
    a.delta = delta;
    a.post = post_scale;
    a.scale = branch_scale;
    a.gatep = gate;
    a.w = norm_scale;
    a.h = h_out;
    a.y = y;
    mxm_launch_resnorm(a, r->stream());
    HIPCK(hipGetLastError());
    return MXM_OK;
  });
}

int mxm_resnorm_backward(int64_t h, int64_t rows, const void* h_in, const void* delta,
                         const void* post_scale, const void* branch_scale, const void* gate,
                         const void* norm_scale, const void* dh, const void* dy, void* dx,
                         void* d_delta, float* d_post_scale, float* d_branch_scale, float* d_gate,
                         float* d_norm_scale) {
  HANDLE_OR_RETURN(ResNorm, r, h, RESNORM);
  return fenced([&] {
    ResNormArgs a = r->base;
    if (!r->backward) fail(RESNORM " backward needs a handle created with MXM_RESNORM_BACKWARD");
    if (rows < 0 || rows > r->max_rows)
      fail(RESNORM " rows %lld out of range [0,%lld]", (long long)rows, (long long)r->max_rows);
    const bool any = rows > 0;
    check_pointer(RESNORM, "h", h_in, a.x_bf16, any && a.norm);
    check_pointer(RESNORM, "delta", delta, a.delta_bf16, any && a.branch);
    check_pointer(RESNORM, "dh", dh, a.g_bf16, any && !a.norm);
    check_pointer(RESNORM, "dy", dy, a.g_bf16, any && a.norm);
    check_pointer(RESNORM, "dx", dx, a.g_bf16, any && (a.norm || !a.branch));
    check_pointer(RESNORM, "d_delta", d_delta, a.g_bf16, any && a.branch);
    check_pointer(RESNORM, "gate", gate, a.p_bf16, any && a.gate != 0);
    check_pointer(RESNORM, "post_scale", post_scale, a.p_bf16, false);
    check_pointer(RESNORM, "branch_scale", branch_scale, a.p_bf16, false);
    check_pointer(RESNORM, "norm_scale", norm_scale, a.p_bf16, false);
    check_pointer(RESNORM, "d_post_scale", d_post_scale, false, false);
    check_pointer(RESNORM, "d_branch_scale", d_branch_scale, false, false);
    check_pointer(RESNORM, "d_gate", d_gate, false, false);
    check_pointer(RESNORM, "d_norm_scale", d_norm_scale, false, false);
    if ((post_scale || d_post_scale) && !a.post_norm)
      fail(RESNORM " post_scale given without MXM_RESNORM_POST_NORM");
    if ((branch_scale || d_branch_scale) && !a.branch)
      fail(RESNORM " branch_scale given without MXM_RESNORM_BRANCH");
    if ((norm_scale || d_norm_scale) && !a.norm)
      fail(RESNORM " norm_scale given without MXM_RESNORM_NORM");
    if (d_gate && !a.gate) fail(RESNORM " d_gate given without a gate");
    const int64_t n = rows * a.D, gates = gate_elements(a, rows);
    Tensors t;
    if (a.norm) t.in("h", h_in, n, a.x_bf16, ROWS);
    if (a.branch) t.in("delta", delta, n, a.delta_bf16, ROWS);
    t.in("dh", dh, n, a.g_bf16, ROWS);
    if (a.norm) t.in("dy", dy, n, a.g_bf16, ROWS);
    t.in("post_scale", post_scale, a.D, a.p_bf16, POST);
    t.in("branch_scale", branch_scale, a.D, a.p_bf16, SCALE);
    t.in("norm_scale", norm_scale, a.D, a.p_bf16, NORM);
    t.in("gate", gate, gates, a.p_bf16, GATE);
    t.out("dx", dx, n, a.g_bf16, ROWS);
    if (a.branch) t.out("d_delta", d_delta, n, a.g_bf16, ROWS);
    t.out("d_post_scale", d_post_scale, a.D, false, POST);
    t.out("d_branch_scale", d_branch_scale, a.D, false, SCALE);
    t.out("d_gate", d_gate, gates, false, GATE);
    t.out("d_norm_scale", d_norm_scale, a.D, false, NORM);
    t.check(RESNORM);
    const DeviceGuard guard(r->stream_ref->device);
    a.N = (int)rows;
    a.delta = delta;
    a.post = post_scale;
    a.scale = branch_scale;
    a.gatep = gate;
    a.w = norm_scale;
    a.h = const_cast<void*>(h_in);
    a.dh = dh;
    a.dy = dy;
    a.dx = dx;
    a.d_delta = d_delta;
    a.d_post = d_post_scale;
    a.d_scale = d_branch_scale;
    a.d_gate = d_gate;
    a.d_w = d_norm_scale;
    if (!mxm_launch_resnorm_bw(a, r->stream()))
      fail_rt(RESNORM " internal error: backward workspace too small");
    HIPCK(hipGetLastError());
    return MXM_OK;
  });
}

int64_t mxm_grads_create(const int64_t* sizes, const int32_t* dtypes, const float* decay, int n,
                         int64_t stream_of) {
  int64_t handle = 0;
  const int rc = fenced([&] {
    if (!sizes || !dtypes || n < 1) fail(GRADSET " requires sizes and dtypes of at least one tensor");
    int64_t total = 0;
    for (int i = 0; i < n; ++i) {
      if (sizes[i] < 0 || sizes[i] > ((int64_t)1 << 40) || (total += sizes[i]) > ((int64_t)1 << 40))
        fail(GRADSET " tensor %d: size %lld out of range (at most 2^40 elements in all)", i,
             (long long)sizes[i]);
      if (!float_dtype(dtypes[i]))
        fail(GRADSET " tensor %d: dtype %d unsupported (want fp32 or bf16)", i, dtypes[i]);
      if (decay && !std::isfinite(decay[i])) fail(GRADSET " tensor %d: decay is not finite", i);
    }
    auto shared = shared_stream(GRADSET, stream_of);

    auto g = std::make_shared<GradSet>();
    const DeviceGuard guard(shared ? shared->device : [] {
      int dev = 0;
      HIPCK(hipGetDevice(&dev));
      return dev;
    }());
    g->stream_ref = choose_stream(shared);
    g->n_cu = cu_count(g->stream_ref->device);
    const int64_t per = mxm_grad_chunk_elems(total, g->n_cu);
    int64_t pieces = 0;
    for (int i = 0; i < n; ++i) {
      g->tensors.push_back({sizes[i], dtypes[i] == MXM_DTYPE_BF16, decay ? decay[i] : 1.0f});
      pieces += (sizes[i] + per - 1) / per;
    }
    // (slices, at most 16 a piece, are counted in 31 bits)
    if (pieces > (INT32_MAX >> 4)) fail(GRADSET " too many pieces (%lld)", (long long)pieces);
    g->chunks.alloc((size_t)pieces * sizeof(GradChunk));
    g->partial.alloc((size_t)mxm_grad_norm_blocks((int)pieces) * sizeof(double));
    g->small.alloc(256);
    HIPCK(hipMemsetAsync(g->small.p, 0, 256, g->stream()));
    HIPCK(hipStreamSynchronize(g->stream()));
    GradArgs& a = g->base;
    a.chunks = g->chunks.as<GradChunk>();
    a.n_chunks = (int)pieces;
    a.chunk_elems = (int)per;
    a.all_bf16 = true;
    for (const auto& t : g->tensors) a.all_bf16 = a.all_bf16 && t.bf16;
    a.partial = g->partial.as<double>();
    a.ticket = g->small.as<int32_t>();
    a.scalars = reinterpret_cast<GradScalars*>(g->small.as<char>() + 64);
    handle = keep(std::move(g));
    return MXM_OK;
  });
  return rc == MXM_OK ? handle : 0;
}

int mxm_grads_destroy(int64_t h) { return destroy<GradSet>(h, GRADSET); }

int mxm_grads_bind(int64_t h, const void* const* grads, void* const* clipped, void* const* params,
                   void* const* m, void* const* v, void* const* params_bf16) {
  HANDLE_OR_RETURN(GradSet, g, h, GRADSET);
  return fenced([&] {
    if (!grads) fail(GRADSET " grads must be non-NULL");
    if ((params != nullptr) != (m != nullptr) || (params != nullptr) != (v != nullptr))
      fail(GRADSET " params, m and v are bound together");
    if (params_bf16 && !params) fail(GRADSET " params_bf16 needs params");
    const int64_t per = g->base.chunk_elems;
    struct Extent {
      uintptr_t from, to;
      size_t tensor;
      const char* name;
    };
    std::vector<Extent> extents;
    std::vector<GradChunk> chunks;
    chunks.reserve((size_t)g->base.n_chunks);
    for (size_t i = 0; i < g->tensors.size(); ++i) {
      const GradSet::Tensor& t = g->tensors[i];
      if (t.n == 0) continue;
      // tensor i's pointer in a list (null: the list is not bound)
      auto take = [&](const char* name, const void* const* list, bool bf16) {
        if (!list) return (char*)nullptr;
        const void* p = list[i];
        if (!p) fail(GRADSET " tensor %zu: %s is NULL", i, name);
        if (reinterpret_cast<uintptr_t>(p) % (bf16 ? 2 : 4) != 0)
          fail(GRADSET " tensor %zu: %s is not aligned to its elements", i, name);
        const uintptr_t from = reinterpret_cast<uintptr_t>(p);
        extents.push_back({from, from + (uintptr_t)t.n * (bf16 ? 2 : 4), i, name});
        return static_cast<char*>(const_cast<void*>(p));
      };
      char* const gp = take("grads", grads, t.bf16);
      char* const cp = clipped && clipped[i] != gp ? take("clipped", clipped, t.bf16) : gp;
      char* const pp = take("params", params, false);
      char* const mp = take("m", m, false);
      char* const vp = take("v", v, false);
      char* const hp = take("params_bf16", params_bf16, true);
      for (int64_t at = 0; at < t.n; at += per) {
        const int64_t wide = at * 4, own = at * (t.bf16 ? 2 : 4);
        GradChunk c{};
        c.g = gp + own;
        c.clipped = cp + own;
        if (pp) {
          c.p = reinterpret_cast<float*>(pp + wide);
          c.m = reinterpret_cast<float*>(mp + wide);
          c.v = reinterpret_cast<float*>(vp + wide);
        }
        if (hp) c.p16 = reinterpret_cast<uint16_t*>(hp + at * 2);
        c.count = (int32_t)std::min(t.n - at, per);
        c.decay = t.decay;
        c.bf16 = t.bf16;
        chunks.push_back(c);
      }
    }
    std::sort(extents.begin(), extents.end(),
              [](const Extent& a, const Extent& b) { return a.from < b.from; });
    for (size_t k = 1; k < extents.size(); ++k)
      if (extents[k].from < extents[k - 1].to)
        fail(GRADSET " tensor %zu: %s overlaps tensor %zu's %s", extents[k].tensor, extents[k].name,
             extents[k - 1].tensor, extents[k - 1].name);
    const DeviceGuard guard(g->stream_ref->device);
    // (waits for the calls that read the table, then for the copy)
    if (!chunks.empty())
      HIPCK(hipMemcpyAsync(g->chunks.p, chunks.data(), chunks.size() * sizeof(GradChunk),
                           hipMemcpyHostToDevice, g->stream()));
    HIPCK(hipStreamSynchronize(g->stream()));
    g->bound = true;
    g->has_params = params != nullptr;
    return MXM_OK;
  });
}

int mxm_grads_norm(int64_t h, float* norm) {
  HANDLE_OR_RETURN(GradSet, g, h, GRADSET);
  return fenced([&] {
    check_pointer(GRADSET, "norm", norm, false, true);
    if (!g->bound) fail_rt(GRADSET " norm before mxm_grads_bind");
    const DeviceGuard guard(g->stream_ref->device);
    GradArgs a = g->base;
    a.norm = norm;
    mxm_launch_grad_norm(a, false, g->stream());
    HIPCK(hipGetLastError());
    return MXM_OK;
  });
}

int mxm_grads_clip(int64_t h, double max_norm, float* norm) {
  HANDLE_OR_RETURN(GradSet, g, h, GRADSET);
  return fenced([&] {
    check_pointer(GRADSET, "norm", norm, false, false);
    if (!(max_norm > 0.0) || !std::isfinite(max_norm))
      fail(GRADSET " max_norm must be finite and > 0");
    if (!g->bound) fail_rt(GRADSET " clip before mxm_grads_bind");
    const DeviceGuard guard(g->stream_ref->device);
    GradArgs a = g->base;
    a.norm = norm;
    a.max_norm = max_norm;
    mxm_launch_grad_norm(a, true, g->stream());
    HIPCK(hipGetLastError());
    mxm_launch_grad_clip(a, g->stream());
    HIPCK(hipGetLastError());
    return MXM_OK;
  });
}

int mxm_grads_adamw(int64_t h, double lr, double beta1, double beta2, double eps,
                    double weight_decay, double max_norm, int64_t* step, float* norm,
                    int32_t* skipped) {
  HANDLE_OR_RETURN(GradSet, g, h, GRADSET);
  return fenced([&] {
    if (!(lr >= 0.0) || !std::isfinite(lr)) fail(GRADSET " lr must be finite and >= 0");
    if (!(beta1 >= 0.0 && beta1 < 1.0) || !(beta2 >= 0.0 && beta2 < 1.0))
      fail(GRADSET " beta1 and beta2 must be in [0,1)");
    if (!((float)eps > 0.0f) || !std::isfinite(eps)) fail(GRADSET " eps must be finite and > 0");
    if (!(weight_decay >= 0.0) || !std::isfinite(weight_decay))
      fail(GRADSET " weight_decay must be finite and >= 0");
    if (!std::isfinite((float)lr) || !std::isfinite((float)(lr * weight_decay)))
      fail(GRADSET " lr and lr * weight_decay must be finite in fp32");
    if (!(max_norm >= 0.0) || !std::isfinite(max_norm))
      fail(GRADSET " max_norm must be finite and >= 0 (0: no clipping)");
    if (!step || reinterpret_cast<uintptr_t>(step) % 8 != 0)
      fail(GRADSET " step must be non-NULL and aligned");
    check_pointer(GRADSET, "norm", norm, false, false);
    check_pointer(GRADSET, "skipped", skipped, false, false);
    if (!g->bound || !g->has_params) fail_rt(GRADSET " adamw before params, m and v are bound");
    const DeviceGuard guard(g->stream_ref->device);
    GradArgs a = g->base;
    a.norm = norm;
    a.max_norm = max_norm;
    a.adamw = true;
    a.step = step;
    a.skipped = skipped;
    a.lr = lr;
    a.beta1 = beta1;
    a.beta2 = beta2;
    a.eps = eps;
    a.weight_decay = weight_decay;
    mxm_launch_grad_norm(a, true, g->stream());
    HIPCK(hipGetLastError());
    mxm_launch_grad_adamw(a, g->stream());
    HIPCK(hipGetLastError());
    return MXM_OK;
  });
}

int mxm_stream(int64_t h, void** stream) {
  const auto s = stream_of_handle(h);
  if (!s) {
    g_last_error = "mxm_stream: invalid handle";
    return MXM_ERR_OP;
  }
  return fenced([&] {
    if (!stream) fail("mxm_stream: stream must be non-NULL");
    *stream = s->stream;
    return MXM_OK;
  });
}

int mxm_synchronize(int64_t h) {
  const auto s = stream_of_handle(h);
  if (!s) {
    g_last_error = "mxm_synchronize: invalid handle";
    return MXM_ERR_OP;
  }
  return fenced([&] {
    HIPCK(hipStreamSynchronize(s->stream));
    return MXM_OK;
  });
}

}  // extern "C"
