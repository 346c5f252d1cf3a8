// C ABI of the handles at the vocabulary's two ends of a training step (declared
// in include/mixmoe.h): token embeddings and token losses.  Same conventions as
// the handles of mxm_train.hip; every argument is checked before the device is
// touched.
#include <algorithm>
#include <cmath>
#include <cstdlib>

#include "../../include/mixmoe.h"
#include "mxm_handles.h"
#include "mxm_vocab.h"

namespace {

struct Embed : TrainHandle {
  EmbedArgs base{};  // what every call shares
  bool backward = false;
  DevBuf sorted, starts, part;
  // (the destructor's wait keeps the workspace until the calls that use it end)
  ~Embed() override {
    if (stream_ref) (void)hipStreamSynchronize(stream());
  }
};

struct Xent : TrainHandle {
  XentArgs base{};
  int64_t max_rows = 0;
  bool backward = false;
  DevBuf counts, weights, map, target, scalars, nll, at_target, row, x_pack, w_pack, exps, parts, stat, stat_exp, summands, dz, partial, dw32, zeros;
  ~Xent() override {
    if (stream_ref) (void)hipStreamSynchronize(stream());
  }
};

// Where a call's tensors lie: no output may overlap another tensor.
struct Places {
  struct One {
    const char* name;
    uintptr_t from, to;
    bool out;
  };
  One all[10];
  int n = 0;
  void add(const char* name, const void* p, int64_t elements, int item, bool out) {
    if (!p || elements <= 0) return;
    const uintptr_t from = reinterpret_cast<uintptr_t>(p);
    all[n++] = {name, from, from + (uintptr_t)elements * item, out};
  }
  void check(const char* what) const {
    for (int i = 0; i < n; ++i)
      for (int j = 0; j < n; ++j)
        if (i != j && all[i].out && all[i].from < all[j].to && all[j].from < all[i].to)
          fail("%s %s overlaps %s", what, all[i].name, all[j].name);
  }
};

void check_sizes(const char* what, int64_t V, int64_t D, int64_t rows) {
  if (V < 1 || V > MXM_VOCAB_MAX || D < 1 || D > MXM_RESNORM_MAX_D || rows < 0 ||
      rows > ((int64_t)1 << 30))
    fail("%s invalid dimensions (V in [1,%d], D in [1,%d], maxRows in [0,2^30])", what, MXM_VOCAB_MAX,
         MXM_RESNORM_MAX_D);
}
void check_dtype(const char* what, int64_t t) {
  if (!float_dtype(t)) fail("%s dtype %lld unsupported (want fp32 or bf16)", what, (long long)t);
}
void check_rows(const char* what, int64_t rows, int64_t max_rows) {
  if (rows < 0 || rows > max_rows)
    fail("%s rows %lld out of range [0,%lld]", what, (long long)rows, (long long)max_rows);
}
int item(bool bf16) { return bf16 ? 2 : 4; }

// A create allocates and clears memory on the stream, which a capture would only record.
void refuse_capture(const char* what, const std::shared_ptr<StreamRef>& shared) {
  if (!shared) return;
  hipStreamCaptureStatus now = hipStreamCaptureStatusNone;
  HIPCK(hipStreamIsCapturing(shared->stream, &now));
  if (now != hipStreamCaptureStatusNone) fail("%s cannot be created on a stream that is being captured", what);
}

// Softcaps: a capped logit is off by a few 2^-24 of the cap, 1.2e-4 at the largest.
constexpr float XENT_MIN_CAP = 1.0f / 64, XENT_MAX_CAP = 1024;

// Bytes that a loss's workspace holds of a piece of the rows at most (but for tables
// of which a tile's rows take more).
constexpr int64_t XENT_PIECE_BYTES = (int64_t)2 << 30;

// What a create returns; memory that there is not enough of leaves an error that the
// next call's launch would take for its own.
int64_t created(int rc, int64_t handle) {
  if (rc == MXM_OK) return handle;
  if (rc == MXM_ERR) (void)hipGetLastError();
  return 0;
}

#define EMBED "TOKEN_EMBEDDING"
#define XENT "TOKEN_LOSS"

int xent_run(Xent& x, bool backward, int64_t rows, const void* xp, const void* weight,
             const int32_t* targets, const float* row_weights, float d_total, float* loss, float* lse,
             float* total, void* dx, void* dw) {
  XentArgs a = x.base;
  check_rows(XENT, rows, x.max_rows);
  const bool any = rows > 0;
  check_pointer(XENT, "x", xp, a.bf16, any);
  check_pointer(XENT, "weight", weight, a.bf16, any);
  check_pointer(XENT, "targets", targets, false, any);
  check_pointer(XENT, "row_weights", row_weights, false, false);
  check_pointer(XENT, "loss", loss, false, false);
  check_pointer(XENT, "lse", lse, false, false);
  check_pointer(XENT, "total", total, false, false);
  check_pointer(XENT, "dx", dx, a.dx_bf16, false);
  check_pointer(XENT, "dw", dw, a.dw_bf16, false);
  if (!backward && !loss && !lse && !total) fail(XENT " forward needs loss, lse or total");
  if (backward && !dx && !dw) fail(XENT " backward needs dx or dw");
  if (!std::isfinite(d_total)) fail(XENT " d_total must be finite");
  Places t;
  t.add("x", xp, rows * a.D, item(a.bf16), false);
  t.add("weight", weight, (int64_t)a.V * a.D, item(a.bf16), false);
  t.add("targets", targets, rows, 4, false);
  t.add("row_weights", row_weights, rows, 4, false);
  t.add("loss", loss, rows, 4, true);
  t.add("lse", lse, rows, 4, true);
  t.add("total", total, 1, 4, true);
  t.add("dx", dx, rows * a.D, item(a.dx_bf16), true);
  t.add("dw", dw, (int64_t)a.V * a.D, item(a.dw_bf16), true);
  t.check(XENT);
  const DeviceGuard guard(x.stream_ref->device);
  a.rows = rows;
  a.x = xp;
  a.weight = weight;
  a.targets = targets;
  a.row_weights = row_weights;
  a.d_total = d_total;
  a.loss = loss;
  a.lse = lse;
  a.total = total;
  a.dx = dx;
  a.dw = dw;
  a.backward = backward;
  mxm_launch_xent(a, x.stream());
  HIPCK(hipGetLastError());
  return MXM_OK;
}

}  // namespace

extern "C" {

int64_t mxm_embed_create(const int64_t* params, int n_params, float scale, int64_t stream_of) {
  int64_t handle = 0;
  const int rc = fenced([&] {
    if (!params || n_params < 8)
      fail(EMBED " requires V,D,maxRows,tableDtype,outDtype,gradDtype,tableGradDtype,flags");
    const int64_t V = params[0], D = params[1], rows = params[2], flags = params[7];
    check_sizes(EMBED, V, D, rows);
    for (int i = 3; i < 7; ++i) check_dtype(EMBED, params[i]);
    if (flags & ~(int64_t)MXM_EMBED_BACKWARD) fail(EMBED " unknown flags 0x%llx", (unsigned long long)flags);
    if (!std::isfinite(scale)) fail(EMBED " scale must be finite");
    auto shared = shared_stream(EMBED, stream_of);
    refuse_capture(EMBED, shared);

    auto e = std::make_shared<Embed>();
    const DeviceGuard guard(device_of(shared));
    e->stream_ref = choose_stream(shared);
    e->n_cu = cu_count(e->stream_ref->device);
    e->backward = (flags & MXM_EMBED_BACKWARD) != 0;
    EmbedArgs& a = e->base;
    a.V = (int)V;
    a.D = (int)D;
    a.max_rows = rows;
    a.scale = scale;
    a.n_cu = e->n_cu;
    a.table_bf16 = params[3] == MXM_DTYPE_BF16;
    a.out_bf16 = params[4] == MXM_DTYPE_BF16;
    a.grad_bf16 = params[5] == MXM_DTYPE_BF16;
    a.dtable_bf16 = params[6] == MXM_DTYPE_BF16;
    if (e->backward) {
      e->sorted.alloc((size_t)rows * sizeof(int2));
      e->starts.alloc(((size_t)V + 1) * 4);
      e->part.alloc((size_t)mxm_embed_part_floats(rows, (int)D) * 4);
      a.sorted = e->sorted.as<int2>();
      a.starts = e->starts.as<int32_t>();
      a.part = e->part.as<float>();
    }
    handle = keep(std::move(e));
    return MXM_OK;
  });
  return created(rc, handle);
}

int mxm_embed_destroy(int64_t h) { return destroy<Embed>(h, EMBED); }

int mxm_embed_forward(int64_t h, int64_t rows, const int32_t* tokens, const void* table, void* out) {
  HANDLE_OR_RETURN(Embed, e, h, EMBED);
  return fenced([&] {
    EmbedArgs a = e->base;
    check_rows(EMBED, rows, a.max_rows);
    const bool any = rows > 0;
    check_pointer(EMBED, "tokens", tokens, false, any);
    check_pointer(EMBED, "table", table, a.table_bf16, any);
    check_pointer(EMBED, "out", out, a.out_bf16, any);
    Places t;
    t.add("tokens", tokens, rows, 4, false);
    t.add("table", table, (int64_t)a.V * a.D, item(a.table_bf16), false);
    t.add("out", out, rows * a.D, item(a.out_bf16), true);
    t.check(EMBED);
    const DeviceGuard guard(e->stream_ref->device);
    a.rows = rows;
    a.tokens = tokens;
    a.table = table;
    a.out = out;
    mxm_launch_embed(a, e->stream());
    HIPCK(hipGetLastError());
    return MXM_OK;
  });
}

int mxm_embed_backward(int64_t h, int64_t rows, const int32_t* tokens, const void* d_out,
                       void* d_table, int accumulate) {
  HANDLE_OR_RETURN(Embed, e, h, EMBED);
  return fenced([&] {
    EmbedArgs a = e->base;
    if (!e->backward) fail(EMBED " backward needs a handle created with MXM_EMBED_BACKWARD");
    check_rows(EMBED, rows, a.max_rows);
    const bool any = rows > 0;
    check_pointer(EMBED, "tokens", tokens, false, any);
    check_pointer(EMBED, "d_out", d_out, a.grad_bf16, any);
    check_pointer(EMBED, "d_table", d_table, a.dtable_bf16, true);
    Places t;
    t.add("tokens", tokens, rows, 4, false);
    t.add("d_out", d_out, rows * a.D, item(a.grad_bf16), false);
    t.add("d_table", d_table, (int64_t)a.V * a.D, item(a.dtable_bf16), true);
    t.check(EMBED);
    const DeviceGuard guard(e->stream_ref->device);
    a.rows = rows;
    a.tokens = tokens;
    a.d_out = d_out;
    a.d_table = d_table;
    a.accumulate = accumulate != 0;
    mxm_launch_embed_bw(a, e->stream());
    HIPCK(hipGetLastError());
    return MXM_OK;
  });
}

int64_t mxm_xent_create(const int64_t* params, int n_params, float softcap, int64_t stream_of) {
  int64_t handle = 0;
  const int rc = fenced([&] {
    if (!params || n_params < 7) fail(XENT " requires V,D,maxRows,dtype,dxDtype,dwDtype,flags");
    const int64_t V = params[0], D = params[1], rows = params[2], flags = params[6];
    check_sizes(XENT, V, D, rows);
    for (int i = 3; i < 6; ++i) check_dtype(XENT, params[i]);
    if (flags & ~(int64_t)(MXM_XENT_MEAN | MXM_XENT_BACKWARD))
      fail(XENT " unknown flags 0x%llx", (unsigned long long)flags);
    if (softcap != 0.0f && !(softcap >= XENT_MIN_CAP && softcap <= XENT_MAX_CAP))
      fail(XENT " softcap must be 0 or in [%g,%g]", XENT_MIN_CAP, XENT_MAX_CAP);
    auto shared = shared_stream(XENT, stream_of);
    refuse_capture(XENT, shared);

    auto x = std::make_shared<Xent>();
    const DeviceGuard guard(device_of(shared));
    x->stream_ref = choose_stream(shared);
    x->n_cu = cu_count(x->stream_ref->device);
    x->max_rows = rows;
    x->backward = (flags & MXM_XENT_BACKWARD) != 0;
    XentArgs& a = x->base;
    a.V = (int)V;
    a.D = (int)D;
    a.softcap = softcap;
    a.n_cu = x->n_cu;
    a.mean = (flags & MXM_XENT_MEAN) != 0;
    a.bf16 = params[3] == MXM_DTYPE_BF16;
    a.dx_bf16 = params[4] == MXM_DTYPE_BF16;
    a.dw_bf16 = params[5] == MXM_DTYPE_BF16;
    const auto up = [](int64_t n) { return (n + 63) / 64 * 64; };
    a.Dp = (int)up(D);
    // (rows of the summands an odd number of 128-byte lines apart: a power of two would
    // put a tile's rows into few memory channels)
    a.Vp = (int)(up(V) | 64);
    a.planes = a.bf16 ? 1 : 2;
    a.x_rows = std::max<int64_t>(rows, 1);
    // a row's share of the workspace: its blocks' sums, and backwards its summands
    // (and under fp32 their gradient's planes)
    int64_t bytes = XENT_PIECE_BYTES;
    if (const char* env = std::getenv("MXM_XENT_PIECE_BYTES")) bytes = std::max(0ll, std::atoll(env));
    const int64_t row_bytes = (V + 127) / 128 * (x->backward && !a.bf16 ? 12 : 8) + (x->backward ? a.Vp * (int64_t)(a.bf16 ? 2 : 8) : 0);
    a.piece_rows = std::max<int64_t>(256, std::min(up(rows), bytes / row_bytes / 256 * 256));
    if (rows < a.piece_rows) a.piece_rows = std::max<int64_t>(64, up(rows));
    x->counts.alloc(XENT_CHUNKS * 4);
    x->weights.alloc(XENT_CHUNKS * 8);
    x->map.alloc((size_t)rows * 4);
    x->target.alloc((size_t)rows * 4);
    x->scalars.alloc(sizeof(XentScalars));
    x->nll.alloc((size_t)rows * 4);
    x->at_target.alloc((size_t)rows * 4);
    x->x_pack.alloc((size_t)a.x_rows * a.Dp * 2 * a.planes);
    x->w_pack.alloc((size_t)V * a.Dp * 2 * a.planes);
    x->stat.alloc((size_t)mxm_xent_stats(a.piece_rows, a.V, a.n_cu) * sizeof(float2));
    if (!a.bf16) {
      const size_t v_tiles = ((size_t)V + 255) / 256 * 256, n = (size_t)rows;
      x->exps.alloc((v_tiles + 2 * n) * 4);
      a.w_exp = x->exps.as<int32_t>();  // (first: read by vectors)
      a.x_exp = a.w_exp + v_tiles;
      a.e_row = a.x_exp + n;
      if (x->backward) {
        x->parts.alloc((n / 4 + 1) * sizeof(int4));  // (4 rows a workgroup at least)
        x->stat_exp.alloc((size_t)mxm_xent_stats(a.piece_rows, a.V, a.n_cu) * 4);
        a.c_part = x->parts.as<int4>();
        a.stat_exp = x->stat_exp.as<int32_t>();
      }
    }
    x->zeros.alloc(4096);
    HIPCK(hipMemsetAsync(x->zeros.p, 0, 4096, x->stream()));
    a.counts = x->counts.as<int32_t>();
    a.weights = x->weights.as<double>();
    a.map = x->map.as<int32_t>();
    a.target = x->target.as<int32_t>();
    a.scalars = x->scalars.as<XentScalars>();
    a.nll = x->nll.as<float>();
    a.at_target = x->at_target.as<float>();
    a.x_pack = x->x_pack.as<uint16_t>();
    a.w_pack = x->w_pack.as<uint16_t>();
    a.stat = x->stat.as<float2>();
    a.zeros = x->zeros.as<uint16_t>();
    if (x->backward) {
      const size_t cells = (size_t)a.piece_rows * (size_t)a.Vp;
      x->row.alloc((size_t)rows * sizeof(XentRow));
      x->summands.alloc(cells * (a.bf16 ? 2 : 4));
      if (!a.bf16) x->dz.alloc(cells * 4);
      x->partial.alloc((size_t)mxm_xent_partial_bytes(a.n_cu));
      if (a.dw_bf16 && rows > a.piece_rows) x->dw32.alloc((size_t)V * (size_t)D * 4);
      a.row = x->row.as<XentRow>();
      a.summands = x->summands.p;
      a.dz = a.bf16 ? x->summands.as<uint16_t>() : x->dz.as<uint16_t>();
      a.partial = x->partial.as<float>();
      a.dw32 = x->dw32.as<float>();
    }
    handle = keep(std::move(x));
    return MXM_OK;
  });
  return created(rc, handle);
}

int mxm_xent_destroy(int64_t h) { return destroy<Xent>(h, XENT); }

int mxm_xent_forward(int64_t h, int64_t rows, const void* x, const void* weight,
                     const int32_t* targets, const float* row_weights, float* loss, float* lse,
                     float* total) {
  HANDLE_OR_RETURN(Xent, e, h, XENT);
  return fenced([&] {
    return xent_run(*e, false, rows, x, weight, targets, row_weights, 0.0f, loss, lse, total, nullptr,
                    nullptr);
  });
}

int mxm_xent_backward(int64_t h, int64_t rows, const void* x, const void* weight,
                      const int32_t* targets, const float* row_weights, float d_total, float* loss,
                      float* lse, float* total, void* dx, void* dw) {
  HANDLE_OR_RETURN(Xent, e, h, XENT);
  return fenced([&] {
    if (!e->backward) fail(XENT " backward needs a handle created with MXM_XENT_BACKWARD");
    return xent_run(*e, true, rows, x, weight, targets, row_weights, d_total, loss, lse, total, dx, dw);
  });
}

}  // extern "C"
