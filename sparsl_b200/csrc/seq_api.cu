// C entries of the sequence operators (sparsl_cuda.h): the checks of their
// arguments, and the launches.  Nothing here allocates, waits or keeps
// anything between calls.
#include <initializer_list>
#include <string>

#include "../../include/sparsl_cuda.h"
#include "seq.cuh"

namespace sparsl {
// capi.cu
int record_error(int code, const char* message);
int record_error_detail(int code, const char* reason, const std::string& detail);
bool admission_enter();
void admission_leave();
int check_device_array(const void* p, uint64_t bytes, int ordinal, const char* what);
int device_ordinal(const sparsl_dev* d);
}  // namespace sparsl

using namespace sparsl;

namespace {

struct Admitted {
  bool ok = admission_enter();
  ~Admitted() { admission_leave(); }
};

// The device current for the call, and the caller's again behind it.
struct OnDevice {
  int prev = -1;
  bool ok;
  explicit OnDevice(int ordinal) {
    cudaGetDevice(&prev);
    ok = prev == ordinal || cudaSetDevice(ordinal) == cudaSuccess;
    if (prev == ordinal) prev = -1;
  }
  ~OnDevice() {
    if (prev >= 0) cudaSetDevice(prev);
  }
};

// Whether [p, p + bytes) lies in one allocation of the GPU's own memory, by one
// driver call; anything else is left to check_device_array, which says why.
bool inside_allocation(const void* p, uint64_t bytes, int ordinal) {
  typedef int (*GetAttributes)(unsigned int, int*, void**, unsigned long long);
  static const GetAttributes get = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuPointerGetAttributes", &f, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      f = nullptr;
    return reinterpret_cast<GetAttributes>(f);
  }();
  if (!get) return false;
  // CU_POINTER_ATTRIBUTE_{MEMORY_TYPE, DEVICE_ORDINAL, RANGE_START_ADDR, RANGE_SIZE, IS_MANAGED}
  int which[5] = {2, 9, 11, 12, 8};
  unsigned int type = 0;
  int device = -1;
  unsigned long long start = 0;
  size_t size = 0;
  unsigned char managed = 1;
  void* out[5] = {&type, &device, &start, &size, &managed};
  const unsigned long long at = reinterpret_cast<unsigned long long>(p);
  if (get(5, which, out, at) != 0) return false;
  return type == 2 /* CU_MEMORYTYPE_DEVICE */ && device == ordinal && !managed && at >= start && at - start <= size &&
         bytes <= size - (at - start);
}

constexpr uint64_t kMostRows = 0x7fffffffull;  // seq_ptr's type
constexpr uint64_t kMostBytes = 1ull << 62;
constexpr uint64_t kMostGroup = 1ull << 36;  // elements from group to group: 2^24 of them fit 64 bits

// A device array of a call: `rows` rows of `width` elements of `size` bytes,
// `stride` elements apart.
struct Array {
  const char* name;
  const void* p;
  uint64_t rows, width, stride, size;
  bool out;
  bool state = false;  // a call's state or final state
  // A row of `width` elements may be runs of `run` ones, `group` apart (0: one run).
  uint64_t group = 0, run = 0;
  uint64_t bytes() const {
    if (!rows || !width) return 0;
    const unsigned __int128 b = ((unsigned __int128)(rows - 1) * stride + width) * size;
    return b > kMostBytes ? kMostBytes : (uint64_t)b;
  }
};

// Whether the rows of two arrays in runs, b's `off` bytes behind a's, may share an
// element: by where in a group their runs lie.
bool runs_meet(const Array& a, const Array& b, uint64_t off) {
  const uint64_t group = a.group * a.size;
  if (!group || group != b.group * b.size) return true;
  const uint64_t at = off % group;
  return at < a.run * a.size || group - at < b.run * b.size;
}

// Whether two arrays share an element.  Rows of one stride (column ranges of
// one wide array) may interleave, and so may the runs of their rows.
bool overlap(const Array& a, const Array& b) {
  const uint64_t na = a.bytes(), nb = b.bytes();
  if (!na || !nb) return false;
  const uint64_t pa = reinterpret_cast<uint64_t>(a.p), pb = reinterpret_cast<uint64_t>(b.p);
  if (pa + na <= pb || pb + nb <= pa) return false;
  if (a.rows < 2 && b.rows < 2) return pb >= pa ? runs_meet(a, b, pb - pa) : runs_meet(b, a, pa - pb);
  const uint64_t sa = a.stride * a.size, sb = b.stride * b.size;
  if (sa != sb || a.rows < 2 || b.rows < 2 || !sa) return true;
  const uint64_t wa = a.width * a.size, wb = b.width * b.size;
  const uint64_t off = pb >= pa ? (pb - pa) % sa : (sa - (pa - pb) % sa) % sa;  // b's columns behind a's
  if (off >= wa && sa - off >= wb) return false;
  if (off + wb <= sa) return runs_meet(a, b, off);  // b's row ends before a's next one begins
  if (wa <= off) return runs_meet(b, a, sa - off);  // a's row ends before b's next one begins
  return true;
}

struct Call {
  const char* op;
  int ordinal = 0;
  Array arrays[32];
  int count = 0;
  int rc = SPARSL_OK;

  int fail(int code, const char* reason, const std::string& detail) {
    if (rc == SPARSL_OK) rc = record_error_detail(code, reason, std::string(op) + ": " + detail);
    return rc;
  }
  void want(bool ok, int code, const char* reason, const char* detail) {
    if (!ok && rc == SPARSL_OK) fail(code, reason, detail);
  }
  void add(const char* name, const void* p, uint64_t rows, uint64_t width, uint64_t stride, uint64_t size, bool out,
           bool optional = false) {
    if (rc != SPARSL_OK || (optional && !p)) return;
    if (!rows || !width) return;
    if (rows > 1 && stride < width) {
      fail(SPARSL_ERR_LENGTH, "row stride", std::string(name) + ": rows overlap (the stride is below the row's length)");
      return;
    }
    const Array a{name, p, rows, width, stride, size, out};
    if (a.bytes() >= kMostBytes) {
      fail(SPARSL_ERR_LENGTH, "array size", std::string(name) + ": the array is too large");
      return;
    }
    if (reinterpret_cast<uint64_t>(p) % size) {
      fail(SPARSL_ERR_INVALID, "alignment", std::string(name) + ": not aligned to its elements");
      return;
    }
    if (!inside_allocation(p, a.bytes(), ordinal)) {
      const int c = check_device_array(p, a.bytes(), ordinal, name);
      if (c != SPARSL_OK) {
        rc = c;
        return;
      }
    }
    arrays[count++] = a;
  }
  void rows(const char* name, const sparsl_rows& r, uint64_t n, uint64_t width, uint64_t size, bool out, bool optional = false) {
    add(name, r.p, n, width, r.stride, size, out, optional);
  }
  // The same for the scan, whose kernels count a row's bytes in 31 bits.
  void scan_rows(const char* name, const sparsl_rows& r, uint64_t n, uint64_t width, uint64_t size, bool out, bool optional = false) {
    if ((r.p || !optional) && n > 1) want(r.stride <= kMostStride, SPARSL_ERR_LENGTH, "row stride", "a row stride is above 2^29 - 1 elements");
    rows(name, r, n, width, size, out, optional);
  }
  // Rows of `groups` runs of `run` elements, `group` apart.
  void runs(const char* name, const sparsl_rows& r, uint64_t n, uint64_t groups, uint64_t group, uint64_t run, uint64_t size, bool out) {
    const int before = count;
    rows(name, r, n, (groups == 1 ? 0 : (groups - 1) * group) + run, size, out);
    if (count > before && groups > 1) {
      arrays[before].group = group;
      arrays[before].run = run;
    }
  }
  // The state a call starts from, or the one it leaves.
  void states(const char* name, const void* p, uint64_t n, uint64_t row, uint64_t size, bool out, bool optional) {
    const int before = count;
    add(name, p, n, row, row, size, out, optional);
    if (count > before) arrays[before].state = true;
  }
  void flat(const char* name, const void* p, uint64_t n, uint64_t size, bool out, bool optional = false) {
    add(name, p, n ? 1 : 0, n, n, size, out, optional);
  }
  // A caller's scratch: 16-byte aligned, at least `need` bytes.
  void scratch(const char* name, const void* p, uint64_t have, uint64_t need, bool out = true) {
    if (rc != SPARSL_OK || !need) return;
    if (!p || have < need) {
      fail(SPARSL_ERR_LENGTH, "workspace", std::string(name) + " must have " + std::to_string(need) + " bytes, got " +
                                               std::to_string(p ? have : 0));
      return;
    }
    if (reinterpret_cast<uint64_t>(p) % 16) {
      fail(SPARSL_ERR_INVALID, "alignment", std::string(name) + ": must start on a 16-byte boundary");
      return;
    }
    add(name, p, 1, need, need, 1, out);
  }
  // Outputs apart from everything else.  A state and its final state (`state` and
  // `final_state`, arrays of one size) may be the same array.
  void apart() {
    for (int i = 0; i < count && rc == SPARSL_OK; ++i)
      for (int j = i + 1; j < count; ++j) {
        if (!arrays[i].out && !arrays[j].out) continue;
        if (arrays[i].state && arrays[j].state && arrays[i].p == arrays[j].p) continue;
        if (overlap(arrays[i], arrays[j])) {
          fail(SPARSL_ERR_INVALID, "overlap", std::string(arrays[i].name) + " and " + arrays[j].name + " overlap");
          return;
        }
      }
  }
  int done(cudaError_t e) {
    if (e == cudaSuccess) return SPARSL_OK;
    cudaGetLastError();
    return fail(SPARSL_ERR_EXECUTION, op, cudaGetErrorString(e));
  }
};

uint64_t size_of(int dtype) { return dtype == SEQ_F32 ? 4 : 2; }

// The split into sequences; `step`: one token of each.
SeqView view_of(Call& k, const sparsl_seqs& s, bool step, bool any_state) {
  SeqView v{};
  v.tokens = s.tokens;
  v.n_seq = s.n_seq;
  v.seq_ptr = step ? nullptr : s.seq_ptr;
  v.slots = s.slots;
  v.resume = step ? nullptr : s.resume;
  v.n_slots = any_state ? s.n_slots : 0;
  k.want(s.tokens <= kMostRows, SPARSL_ERR_LENGTH, "tokens", "more than 2147483647 tokens");
  k.want(s.n_seq < kMostRows, SPARSL_ERR_LENGTH, "n_seq", "too many sequences");
  k.want(s.n_slots <= kMostRows, SPARSL_ERR_LENGTH, "n_slots", "too many state rows");
  if (step) {
    v.run = 1;
    k.want(s.tokens == s.n_seq, SPARSL_ERR_LENGTH, "tokens", "a step takes one token of each sequence");
  } else if (!s.seq_ptr) {
    k.want(s.n_seq ? s.tokens % s.n_seq == 0 : s.tokens == 0, SPARSL_ERR_LENGTH, "tokens",
           "without seq_ptr, tokens must be a multiple of n_seq");
    v.run = s.n_seq ? s.tokens / s.n_seq : 0;
  }
  if (any_state && !s.slots)
    k.want(s.n_slots >= s.n_seq, SPARSL_ERR_LENGTH, "n_slots", "without slots, the state needs a row for each sequence");
  if (!step) k.flat("seq_ptr", s.seq_ptr, s.n_seq + 1, 4, false, true);
  k.flat("slots", s.slots, s.n_seq, 4, false, true);
  if (!step) k.flat("resume", s.resume, s.n_seq, 1, false, true);
  return v;
}

// Runs a call's body: admission, the device, and no exception across the C entry.
template <class F>
int entry(sparsl_dev* d, const void* args, const char* op, F body) {
  try {
    Admitted adm;
    if (!adm.ok)
      return record_error_detail(SPARSL_ERR_BACKEND, "CUDA backend is quarantined after a failed or timed-out dispatch",
                                 std::string(op) + ": CUDA backend is quarantined; call sparsl_device_reset once no work is in flight");
    if (!d || !args) return record_error_detail(SPARSL_ERR_INVALID, "null argument", std::string(op) + ": null argument");
    Call k{op};
    k.ordinal = device_ordinal(d);
    OnDevice on(k.ordinal);
    if (!on.ok) {
      cudaGetLastError();
      return k.fail(SPARSL_ERR_BACKEND, "cudaSetDevice failed", "cudaSetDevice failed");
    }
    return body(k);
  } catch (...) {
    return SPARSL_ERR_BACKEND;  // out of host memory: there is none left for a message either
  }
}

cudaStream_t stream_of(sparsl_dev* d, void* stream) {
  return static_cast<cudaStream_t>(stream ? stream : sparsl_dev_stream(d));
}

enum Form { FORWARD, BACKWARD, STEP };

// ---- causal convolution ----
int conv(sparsl_dev* d, const sparsl_conv_args* p, void* stream, const char* op, Form form) {
  return entry(d, p, op, [&](Call& k) -> int {
    const bool back = form == BACKWARD, step = form == STEP;
    k.want(p->dtype >= 0 && p->dtype <= 2, SPARSL_ERR_INVALID, "dtype", "unknown dtype");
    k.want(p->channels >= 1 && p->channels <= (1u << 30), SPARSL_ERR_LENGTH, "channels", "channels must be 1..2^30");
    k.want(p->width >= 2 && p->width <= 4, SPARSL_ERR_LENGTH, "width", "width must be 2..4");
    if (k.rc != SPARSL_OK) return k.rc;
    const bool states = p->state || p->final_state || (back && (p->dstate || p->dfinal_state));
    if (step) k.want(p->final_state != nullptr || !p->seqs.n_seq, SPARSL_ERR_INVALID, "null argument", "a step needs a state");
    if (back) k.want(!p->seqs.slots && !p->seqs.resume, SPARSL_ERR_INVALID, "slots", "the backward pass takes no slots or resume");
    ConvArgs a{};
    a.seq = view_of(k, p->seqs, step, states);
    const uint64_t e = size_of(p->dtype), t = p->seqs.tokens, ch = p->channels, w = p->width;
    const uint64_t pe = p->params_f32 ? 4 : e, row = (w - 1) * ch;
    k.rows("x", p->x, t, ch, e, false);
    k.flat("weight", p->weight, ch * w, pe, false);
    k.flat("bias", p->bias, ch, pe, false, true);
    if (!step) k.states("state", p->state, p->seqs.n_slots, row, e, false, true);
    a.type = p->dtype;
    a.channels = p->channels;
    a.width = p->width;
    a.silu = p->silu != 0;
    a.params_f32 = p->params_f32 != 0;
    a.x = p->x.p;
    a.x_stride = p->x.stride;
    a.w = p->weight;
    a.bias = p->bias;
    a.state = step ? nullptr : p->state;
    if (back) {
      k.rows("dy", p->dy, t, ch, e, false);
      k.rows("dx", p->dx, t, ch, e, true);
      k.flat("dweight", p->dweight, ch * w, 4, true);
      k.flat("dbias", p->dbias, ch, 4, true, true);
      k.add("dstate", p->dstate, p->seqs.n_slots, row, row, e, true, true);
      k.add("dfinal_state", p->dfinal_state, p->seqs.n_slots, row, row, e, false, true);
      k.scratch("workspace", p->workspace, p->workspace_bytes, conv_backward_bytes(t, ch, p->width));
      k.apart();
      a.dy = p->dy.p;
      a.dy_stride = p->dy.stride;
      a.dx = p->dx.p;
      a.dx_stride = p->dx.stride;
      a.dw = p->dweight;
      a.dbias = p->dbias;
      a.dstate = p->dstate;
      a.dfinal = p->dfinal_state;
      a.part = static_cast<float*>(p->workspace);
      return k.rc != SPARSL_OK ? k.rc : k.done(launch_conv_backward(a, stream_of(d, stream)));
    }
    k.rows("y", p->y, t, ch, e, true);
    k.states("final_state", p->final_state, p->seqs.n_slots, row, e, true, !step);
    k.apart();
    a.y = p->y.p;
    a.y_stride = p->y.stride;
    a.final_state = p->final_state;
    if (k.rc != SPARSL_OK || !p->seqs.n_seq) return k.rc;
    return k.done(step ? launch_conv_step(a, stream_of(d, stream)) : launch_conv(a, stream_of(d, stream)));
  });
}

// ---- selective scan ----
int scan(sparsl_dev* d, const sparsl_scan_args* p, void* stream, const char* op, Form form) {
  return entry(d, p, op, [&](Call& k) -> int {
    const bool back = form == BACKWARD, step = form == STEP;
    k.want(p->dtype >= 0 && p->dtype <= 2, SPARSL_ERR_INVALID, "dtype", "unknown dtype");
    k.want(p->channels >= 1 && p->channels <= (1u << 24), SPARSL_ERR_LENGTH, "channels", "channels must be 1..2^24");
    k.want(p->states >= 1 && p->states <= kMaxStates, SPARSL_ERR_LENGTH, "states", "states must be 1..64");
    k.want(p->groups >= 1 && p->groups <= p->channels && p->channels % p->groups == 0, SPARSL_ERR_LENGTH, "groups",
           "channels must be a multiple of groups");
    if (k.rc != SPARSL_OK) return k.rc;
    const bool states = p->state || p->final_state || (back && (p->dstate || p->dfinal_state));
    if (step) k.want(p->final_state != nullptr || !p->seqs.n_seq, SPARSL_ERR_INVALID, "null argument", "a step needs a state");
    if (back) k.want(!p->seqs.slots && !p->seqs.resume, SPARSL_ERR_INVALID, "slots", "the backward pass takes no slots or resume");
    SscanArgs a{};
    a.seq = view_of(k, p->seqs, step, states);
    const uint64_t e = size_of(p->dtype), t = p->seqs.tokens, ch = p->channels, n = p->states, g = p->groups;
    const uint64_t row = ch * n;
    const auto bc = [&](const char* name, const sparsl_rows& r, uint64_t group, bool out) {
      k.want(g == 1 || group >= n, SPARSL_ERR_LENGTH, "group stride", "the runs of b or c overlap");
      k.want(group <= kMostGroup, SPARSL_ERR_LENGTH, "group stride", "the group stride is too large");
      k.runs(name, r, t, g, group, n, e, out);
    };
    k.scan_rows("x", p->x, t, ch, e, false);
    k.scan_rows("dt", p->dt, t, ch, e, false);
    k.scan_rows("z", p->z, t, ch, e, false, true);
    bc("b", p->b, p->b_group, false);
    bc("c", p->c, p->c_group, false);
    k.flat("a", p->a, row, 4, false);
    k.flat("d", p->d, ch, 4, false, true);
    k.flat("dt_bias", p->dt_bias, ch, 4, false, true);
    if (!step) k.states("state", p->state, p->seqs.n_slots, row, 4, false, true);
    a.type = p->dtype;
    a.channels = p->channels;
    a.states = p->states;
    a.groups = p->groups;
    a.softplus = p->softplus != 0;
    a.x = p->x.p;
    a.dt = p->dt.p;
    a.z = p->z.p;
    a.b = p->b.p;
    a.c = p->c.p;
    a.x_stride = p->x.stride;
    a.dt_stride = p->dt.stride;
    a.z_stride = p->z.stride;
    a.b_stride = p->b.stride;
    a.c_stride = p->c.stride;
    a.b_group = p->b_group;
    a.c_group = p->c_group;
    a.a = p->a;
    a.d = p->d;
    a.dt_bias = p->dt_bias;
    const auto bytes = [&](const sparsl_rows& r) { return (uint32_t)(r.stride * e); };
    a.x_row = bytes(p->x);
    a.dt_row = bytes(p->dt);
    a.z_row = bytes(p->z);
    a.state = step ? nullptr : p->state;
    a.work = p->workspace;
    a.marks = step ? nullptr : static_cast<float*>(p->checkpoints);
    if (!step && (back || p->checkpoints))
      k.scratch("checkpoints", p->checkpoints, p->checkpoint_bytes, sscan_mark_bytes(t, ch, p->states), !back);
    if (back) {
      k.scan_rows("dy", p->dy, t, ch, e, false);
      k.scan_rows("dx", p->dx, t, ch, e, true);
      k.scan_rows("ddt", p->ddt, t, ch, e, true);
      if (p->z.p) k.scan_rows("dz", p->dz, t, ch, e, true);
      bc("db", p->db, p->db_group, true);
      bc("dc", p->dc, p->dc_group, true);
      k.flat("da", p->da, row, 4, true);
      k.flat("dd", p->dd, ch, 4, true, true);
      k.flat("ddt_bias", p->ddt_bias, ch, 4, true, true);
      k.add("dstate", p->dstate, p->seqs.n_slots, row, row, 4, true, true);
      k.add("dfinal_state", p->dfinal_state, p->seqs.n_slots, row, row, 4, false, true);
      k.scratch("workspace", p->workspace, p->workspace_bytes, sscan_backward_bytes(t, ch, p->states, p->seqs.n_seq, p->groups));
      k.apart();
      a.dy_row = bytes(p->dy);
      a.dx_row = bytes(p->dx);
      a.ddt_row = bytes(p->ddt);
      a.dz_row = bytes(p->dz);
      a.dy = p->dy.p;
      a.dx = p->dx.p;
      a.ddt = p->ddt.p;
      a.dz = p->dz.p;
      a.db = p->db.p;
      a.dc = p->dc.p;
      a.dy_stride = p->dy.stride;
      a.dx_stride = p->dx.stride;
      a.ddt_stride = p->ddt.stride;
      a.dz_stride = p->dz.stride;
      a.db_stride = p->db.stride;
      a.dc_stride = p->dc.stride;
      a.db_group = p->db_group;
      a.dc_group = p->dc_group;
      a.da = p->da;
      a.dd = p->dd;
      a.ddt_bias = p->ddt_bias;
      a.dstate = p->dstate;
      a.dfinal = p->dfinal_state;
      return k.rc != SPARSL_OK ? k.rc : k.done(launch_sscan_backward(a, stream_of(d, stream)));
    }
    k.scan_rows("y", p->y, t, ch, e, true);
    k.states("final_state", p->final_state, p->seqs.n_slots, row, 4, true, !step);
    if (!step) k.scratch("workspace", p->workspace, p->workspace_bytes, sscan_bytes(t, ch, p->states, p->seqs.n_seq, p->groups));
    k.apart();
    a.y = p->y.p;
    a.y_stride = p->y.stride;
    a.y_row = bytes(p->y);
    a.final_state = p->final_state;
    if (k.rc != SPARSL_OK || !p->seqs.n_seq) return k.rc;
    return k.done(step ? launch_sscan_step(a, stream_of(d, stream)) : launch_sscan(a, stream_of(d, stream)));
  });
}

// ---- layer norm ----
int norm(sparsl_dev* d, const sparsl_norm_args* p, void* stream, const char* op, Form form) {
  return entry(d, p, op, [&](Call& k) -> int {
    const bool back = form == BACKWARD;
    k.want(p->dtype >= 0 && p->dtype <= 2, SPARSL_ERR_INVALID, "dtype", "unknown dtype");
    k.want(p->channels >= 1 && p->channels <= (1u << 30), SPARSL_ERR_LENGTH, "channels", "channels must be 1..2^30");
    k.want(p->rows <= kMostRows, SPARSL_ERR_LENGTH, "rows", "more than 2147483647 rows");
    if (k.rc != SPARSL_OK) return k.rc;
    const uint64_t e = size_of(p->dtype), pe = p->params_f32 ? 4 : e, t = p->rows, ch = p->channels;
    k.rows("x", p->x, t, ch, e, false);
    k.flat("weight", p->weight, ch, pe, false, true);
    k.flat("bias", p->bias, ch, pe, false, true);
    k.flat("mean", p->mean, t, 4, !back, !back);
    k.flat("rstd", p->rstd, t, 4, !back, !back);
    NormArgs a{};
    a.type = p->dtype;
    a.params_f32 = p->params_f32 != 0;
    a.rows = t;
    a.channels = ch;
    a.x = p->x.p;
    a.x_stride = p->x.stride;
    a.w = p->weight;
    a.bias = p->bias;
    a.eps = p->eps;
    a.mean = p->mean;
    a.rstd = p->rstd;
    if (back) {
      k.rows("dy", p->dy, t, ch, e, false);
      k.rows("dx", p->dx, t, ch, e, true);
      k.flat("dweight", p->dweight, ch, 4, true, true);
      k.flat("dbias", p->dbias, ch, 4, true, true);
      k.scratch("workspace", p->workspace, p->workspace_bytes, norm_backward_bytes(t, ch));
      k.apart();
      a.dy = p->dy.p;
      a.dy_stride = p->dy.stride;
      a.dx = p->dx.p;
      a.dx_stride = p->dx.stride;
      a.dw = p->dweight;
      a.dbias = p->dbias;
      a.part = static_cast<float*>(p->workspace);
      return k.rc != SPARSL_OK ? k.rc : k.done(launch_norm_backward(a, stream_of(d, stream)));
    }
    k.want(p->eps >= 0.f, SPARSL_ERR_INVALID, "eps", "eps must not be negative");
    k.rows("y", p->y, t, ch, e, true);
    k.apart();
    a.y = p->y.p;
    a.y_stride = p->y.stride;
    return k.rc != SPARSL_OK ? k.rc : k.done(launch_norm(a, stream_of(d, stream)));
  });
}

}  // namespace

extern "C" {

int sparsl_dev_causal_conv_device(sparsl_dev* dev, const sparsl_conv_args* args, void* stream) {
  return conv(dev, args, stream, "causal_conv", FORWARD);
}
int sparsl_dev_causal_conv_backward_device(sparsl_dev* dev, const sparsl_conv_args* args, void* stream) {
  return conv(dev, args, stream, "causal_conv_backward", BACKWARD);
}
int sparsl_dev_causal_conv_step_device(sparsl_dev* dev, const sparsl_conv_args* args, void* stream) {
  return conv(dev, args, stream, "causal_conv_step", STEP);
}
uint64_t sparsl_causal_conv_backward_workspace(uint64_t tokens, uint64_t channels, uint32_t width) {
  return conv_backward_bytes(tokens, channels, width);
}

int sparsl_dev_selective_scan_device(sparsl_dev* dev, const sparsl_scan_args* args, void* stream) {
  return scan(dev, args, stream, "selective_scan", FORWARD);
}
int sparsl_dev_selective_scan_backward_device(sparsl_dev* dev, const sparsl_scan_args* args, void* stream) {
  return scan(dev, args, stream, "selective_scan_backward", BACKWARD);
}
int sparsl_dev_selective_scan_step_device(sparsl_dev* dev, const sparsl_scan_args* args, void* stream) {
  return scan(dev, args, stream, "selective_scan_step", STEP);
}
uint64_t sparsl_selective_scan_workspace(uint64_t tokens, uint64_t channels, uint32_t states, uint64_t n_seq, uint32_t groups) {
  if (!channels || !states || !groups || channels % groups) return 0;
  return sscan_bytes(tokens, channels, states, n_seq, groups);
}
uint64_t sparsl_selective_scan_checkpoints(uint64_t tokens, uint64_t channels, uint32_t states) {
  return sscan_mark_bytes(tokens, channels, states);
}
uint64_t sparsl_selective_scan_backward_workspace(uint64_t tokens, uint64_t channels, uint32_t states, uint64_t n_seq,
                                                  uint32_t groups) {
  if (!channels || !states || !groups || channels % groups) return 0;
  return sscan_backward_bytes(tokens, channels, states, n_seq, groups);
}

int sparsl_selective_scan_test_layout(uint64_t tokens, uint64_t channels, uint32_t states, uint64_t n_seq, uint32_t groups, int ragged,
                                      int backward, uint64_t* out) {
  if (!out || !channels || channels > (1u << 24) || !states || states > kMaxStates || !groups || channels % groups)
    return SPARSL_ERR_INVALID;
  const ScanLayout l = (backward ? sscan_backward_layout : sscan_layout)(tokens, (uint32_t)channels, states, n_seq, groups, ragged != 0);
  const uint64_t v[5] = {l.lanes, l.chunks, l.len, l.carry, l.chunk_lanes};
  for (int i = 0; i < 5; ++i) out[i] = v[i];
  return SPARSL_OK;
}

int sparsl_dev_layer_norm_device(sparsl_dev* dev, const sparsl_norm_args* args, void* stream) {
  return norm(dev, args, stream, "layer_norm", FORWARD);
}
int sparsl_dev_layer_norm_backward_device(sparsl_dev* dev, const sparsl_norm_args* args, void* stream) {
  return norm(dev, args, stream, "layer_norm_backward", BACKWARD);
}
uint64_t sparsl_layer_norm_backward_workspace(uint64_t rows, uint64_t channels) { return norm_backward_bytes(rows, channels); }

}  // extern "C"
