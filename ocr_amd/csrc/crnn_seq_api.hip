// C entry points of the sequence operators (include/crnn_hip.h): argument checks, then the launch.
#include "crnn_seq.h"

#include <exception>

using namespace crnn;

namespace {

constexpr int64_t I31 = 0x7FFFFFFF, FAR = (int64_t)1 << 40;

// Whether `count` steps of a stride leave what addresses can reach: offsets in bytes, sums of a few of them too, stay below 2^63.
bool far(int64_t stride, int64_t count) { return stride < 0 || stride > FAR || (count > 1 && stride > ((int64_t)1 << 56) / count); }

// [rows, cols] elements of `size` bytes, rows `ld` apart
struct Block {
  const char* p;
  int64_t rows, cols, ld, size;
};

// Whether two blocks share a byte.  Exact for rows the same distance apart (column slices of one buffer); otherwise blocks
// whose address ranges meet count as overlapping.
bool overlap(const Block& a, const Block& b) {
  if (!a.p || !b.p || a.rows <= 0 || b.rows <= 0) return false;
  const int64_t a0 = (int64_t)a.p, a1 = a0 + ((a.rows - 1) * a.ld + a.cols) * a.size;
  const int64_t b0 = (int64_t)b.p, b1 = b0 + ((b.rows - 1) * b.ld + b.cols) * b.size;
  if (a1 <= b0 || b1 <= a0) return false;
  const int64_t pitch = a.ld * a.size;
  if (pitch > 0 && pitch == b.ld * b.size && a.cols * a.size <= pitch && b.cols * b.size <= pitch) {
    const int64_t d = ((b0 - a0) % pitch + pitch) % pitch;   // b's row start within a row of a
    return d < a.cols * a.size || d + b.cols * b.size > pitch;
  }
  return true;
}

bool aligned(const void* p, int64_t size) { return ((uintptr_t)p & (uintptr_t)(size - 1)) == 0; }
int64_t type_size(int t) { return t == CRNN_FP32 ? 4 : t == CRNN_BF16 ? 2 : 1; }

const char* check_linear(const crnn_linear_args& a) {
  if (a.in_type != CRNN_FP32 && a.in_type != CRNN_BF16 && a.in_type != CRNN_E4M3) return "crnn_linear: in_type is none of CRNN_FP32, CRNN_BF16, CRNN_E4M3";
  if (a.out_type != CRNN_FP32 && a.out_type != CRNN_BF16) return "crnn_linear: out_type is neither CRNN_FP32 nor CRNN_BF16";
  if (a.act < CRNN_ACT_NONE || a.act > CRNN_ACT_SILU) return "crnn_linear: unknown activation";
  if (a.reserved != 0) return "crnn_linear: reserved is not 0";
  if (a.m < 0 || a.m > I31 || a.n < 1 || a.n > I31 || a.k < 1 || a.k > I31) return "crnn_linear: m, n or k out of range";
  if (a.m == 0) return nullptr;
  if (!a.x || !a.w || !a.y) return "crnn_linear: x, w or y is null";
  if (a.in_type != CRNN_E4M3 && (a.x_scale || a.w_scale)) return "crnn_linear: scales belong to CRNN_E4M3 operands";
  if (far(a.ldx, a.m) || far(a.ldw, a.n) || far(a.ldr, a.m) || far(a.ldy, a.m)) return "crnn_linear: a row stride is out of range";
  if (a.ldy < a.n && a.m > 1) return "crnn_linear: ldy is smaller than n";
  const int64_t ei = type_size(a.in_type), eo = type_size(a.out_type);
  if (!aligned(a.x, ei) || !aligned(a.w, ei) || !aligned(a.y, eo) || !aligned(a.residual, eo) || !aligned(a.bias, 4) || !aligned(a.x_scale, 4) || !aligned(a.w_scale, 4))
    return "crnn_linear: a pointer is not aligned to its type";
  const Block y{(const char*)a.y, a.m, a.n, a.ldy, eo};
  if (overlap(y, {(const char*)a.x, a.m, a.k, a.ldx, ei}) || overlap(y, {(const char*)a.w, a.n, a.k, a.ldw, ei}) ||
      overlap(y, {(const char*)a.bias, 1, a.n, a.n, 4}) || overlap(y, {(const char*)a.x_scale, 1, a.m, a.m, 4}) || overlap(y, {(const char*)a.w_scale, 1, a.n, a.n, 4}))
    return "crnn_linear: y overlaps an input";
  if (a.residual && !(a.residual == a.y && (a.ldr == a.ldy || a.m == 1)) && overlap(y, {(const char*)a.residual, a.m, a.n, a.ldr, eo}))
    return "crnn_linear: y overlaps the residual without being it";
  return nullptr;
}

const char* check_norm(const crnn_rms_norm_args& a) {
  if (a.in_type != CRNN_FP32 && a.in_type != CRNN_BF16) return "crnn_rms_norm: in_type is neither CRNN_FP32 nor CRNN_BF16";
  if (a.out_type != a.in_type && a.out_type != CRNN_E4M3) return "crnn_rms_norm: out_type is neither in_type nor CRNN_E4M3";
  if (a.reserved != 0) return "crnn_rms_norm: reserved is not 0";
  if (!(a.eps >= 0.f)) return "crnn_rms_norm: eps is negative or NaN";
  if (a.m < 0 || a.m > I31 || a.n < 1 || a.n > I31) return "crnn_rms_norm: m or n out of range";
  if (a.m == 0) return nullptr;
  const bool e8 = a.out_type == CRNN_E4M3;
  if (!a.x || !a.gain || !a.y) return "crnn_rms_norm: x, gain or y is null";
  if (e8 != (a.y_scale != nullptr)) return "crnn_rms_norm: y_scale belongs to CRNN_E4M3 outputs, and they need it";
  if (far(a.ldx, a.m) || far(a.ldr, a.m) || far(a.lds, a.m) || far(a.ldy, a.m)) return "crnn_rms_norm: a row stride is out of range";
  if (a.m > 1 && (a.ldy < a.n || (a.sum && a.lds < a.n))) return "crnn_rms_norm: the rows of an output overlap";
  const int64_t ei = type_size(a.in_type), eo = type_size(a.out_type);
  if (!aligned(a.x, ei) || !aligned(a.residual, ei) || !aligned(a.sum, ei) || !aligned(a.y, eo) || !aligned(a.gain, 4) || !aligned(a.y_scale, 4))
    return "crnn_rms_norm: a pointer is not aligned to its type";
  const Block in[3] = {{(const char*)a.x, a.m, a.n, a.ldx, ei}, {(const char*)a.residual, a.m, a.n, a.ldr, ei}, {(const char*)a.gain, 1, a.n, a.n, 4}};
  const Block out[3] = {{(const char*)a.y, a.m, a.n, a.ldy, eo}, {(const char*)a.sum, a.m, a.n, a.lds, ei}, {(const char*)a.y_scale, 1, a.m, a.m, 4}};
  for (int i = 0; i < 3; i++) {
    for (int j = 0; j < 3; j++) {
      const bool same = i < 2 && j < 2 && out[i].p == in[j].p && out[i].size == in[j].size && (out[i].ld == in[j].ld || a.m == 1);
      if (!same && overlap(out[i], in[j])) return "crnn_rms_norm: an output overlaps an input without being it";
    }
    for (int j = 0; j < i; j++)
      if (overlap(out[i], out[j])) return "crnn_rms_norm: two outputs overlap";
  }
  return nullptr;
}

const char* check_attention(const crnn_cross_attention_args& a, bool sizes_only) {
  if (a.type != CRNN_FP32 && a.type != CRNN_BF16) return "crnn_cross_attention: type is neither CRNN_FP32 nor CRNN_BF16";
  if (a.reserved != 0) return "crnn_cross_attention: reserved is not 0";
  if (a.heads < 1 || a.kv_heads < 1 || a.heads % a.kv_heads != 0) return "crnn_cross_attention: heads is not a multiple of kv_heads";
  if (a.head_dim < 1 || a.head_dim > 128) return "crnn_cross_attention: head_dim is outside 1 .. 128";
  if (a.batch < 0 || a.q_len < 0 || a.kv_len < 0 || a.batch > I31 || a.q_len > I31 || a.kv_len > I31) return "crnn_cross_attention: batch, q_len or kv_len out of range";
  // one workgroup takes at least one row of one batch entry's key head
  if ((double)a.batch * a.heads * (double)a.q_len > 2147483647.0) return "crnn_cross_attention: batch * heads * q_len passes 2^31 - 1";
  const int64_t qn[3] = {a.batch, a.q_len, a.heads}, kn[3] = {a.batch, a.kv_len, a.kv_heads};
  for (int i = 0; i < 3; i++)
    if (far(a.q_stride[i], qn[i]) || far(a.out_stride[i], qn[i]) || far(a.k_stride[i], kn[i]) || far(a.v_stride[i], kn[i]))
      return "crnn_cross_attention: a stride is out of range";
  if (sizes_only || a.batch == 0 || a.q_len == 0) return nullptr;
  if (!a.q || !a.out || (a.kv_len > 0 && (!a.k || !a.v))) return "crnn_cross_attention: q, k, v or out is null";
  if (a.mask && far(a.mask_stride, a.batch)) return "crnn_cross_attention: mask_stride is out of range";
  if (!(a.scale == a.scale) || a.scale - a.scale != 0.f) return "crnn_cross_attention: scale is not finite";
  const int64_t e = type_size(a.type);
  if (!aligned(a.q, e) || !aligned(a.k, e) || !aligned(a.v, e) || !aligned(a.out, e) || !aligned(a.lengths, 4))
    return "crnn_cross_attention: a pointer is not aligned to its type";
  // rows of the output: no two of them may meet.  Sorted by stride, each has to pass over the extent of the smaller ones.
  int64_t st[3] = {a.out_stride[0], a.out_stride[1], a.out_stride[2]}, len[3] = {a.batch, a.q_len, a.heads};
  for (int i = 0; i < 3; i++)
    for (int j = 0; j + 1 < 3; j++)
      if (st[j] > st[j + 1]) {
        const int64_t s = st[j], l = len[j];
        st[j] = st[j + 1]; len[j] = len[j + 1];
        st[j + 1] = s; len[j + 1] = l;
      }
  int64_t extent = a.head_dim;
  for (int i = 0; i < 3; i++) {
    if (len[i] == 1) continue;
    if (st[i] < extent) return "crnn_cross_attention: rows of out overlap";
    extent += st[i] * (len[i] - 1);
  }
  // (inputs may be views that interleave with one another, so of them only a common address range is looked at)
  auto span = [&](const int64_t* s, int64_t t, int64_t hh) { return s[0] * (a.batch - 1) + s[1] * (t - 1) + s[2] * (hh - 1) + a.head_dim; };
  const Block out{(const char*)a.out, 1, extent, extent, e};
  const int64_t qs = span(a.q_stride, a.q_len, a.heads);
  if (overlap(out, {(const char*)a.q, 1, qs, qs, e})) return "crnn_cross_attention: out overlaps q";
  if (a.kv_len > 0) {
    const int64_t ks = span(a.k_stride, a.kv_len, a.kv_heads), vs = span(a.v_stride, a.kv_len, a.kv_heads);
    if (overlap(out, {(const char*)a.k, 1, ks, ks, e}) || overlap(out, {(const char*)a.v, 1, vs, vs, e})) return "crnn_cross_attention: out overlaps k or v";
    if (a.mask) {
      const int64_t ms = a.mask_stride * (a.batch - 1) + a.kv_len;
      if (overlap(out, {(const char*)a.mask, 1, ms, ms, 1})) return "crnn_cross_attention: out overlaps the mask";
    }
  }
  if (overlap(out, {(const char*)a.lengths, 1, a.batch, a.batch, 4})) return "crnn_cross_attention: out overlaps the lengths";
  return nullptr;
}

int launched(crnn_handle* h) {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? 0 : seq_fail(h, CRNN_ERR_HIP, hipGetErrorString(e));
}

}  // namespace

extern "C" {

int crnn_linear(crnn_handle* h, const crnn_linear_args* a, void* stream) {
  if (!h) return CRNN_ERR_ARG;
  try {
    if (!a) return seq_fail(h, CRNN_ERR_ARG, "crnn_linear: no arguments");
    if (const char* bad = check_linear(*a)) return seq_fail(h, CRNN_ERR_ARG, bad);
    if (a->m == 0) return 0;
    SeqDevice dev;
    if (int rc = seq_enter(h, stream, &dev)) return rc;
    launch_linear(*a, (hipStream_t)stream);
    return launched(h);
  } catch (const std::exception&) {
    return CRNN_ERR_NOMEM;
  }
}

int crnn_rms_norm(crnn_handle* h, const crnn_rms_norm_args* a, void* stream) {
  if (!h) return CRNN_ERR_ARG;
  try {
    if (!a) return seq_fail(h, CRNN_ERR_ARG, "crnn_rms_norm: no arguments");
    if (const char* bad = check_norm(*a)) return seq_fail(h, CRNN_ERR_ARG, bad);
    if (a->m == 0) return 0;
    SeqDevice dev;
    if (int rc = seq_enter(h, stream, &dev)) return rc;
    launch_rms_norm(*a, (hipStream_t)stream);
    return launched(h);
  } catch (const std::exception&) {
    return CRNN_ERR_NOMEM;
  }
}

int64_t crnn_cross_attention_workspace(crnn_handle* h, const crnn_cross_attention_args* a) {
  if (!h) return CRNN_ERR_ARG;
  try {
    if (!a) return seq_fail(h, CRNN_ERR_ARG, "crnn_cross_attention_workspace: no arguments");
    if (const char* bad = check_attention(*a, true)) return seq_fail(h, CRNN_ERR_ARG, bad);
    return a->batch == 0 || a->q_len == 0 ? 0 : cross_attention_workspace(*a);
  } catch (const std::exception&) {
    return CRNN_ERR_NOMEM;
  }
}

int crnn_cross_attention(crnn_handle* h, const crnn_cross_attention_args* a, void* stream) {
  if (!h) return CRNN_ERR_ARG;
  try {
    if (!a) return seq_fail(h, CRNN_ERR_ARG, "crnn_cross_attention: no arguments");
    if (const char* bad = check_attention(*a, false)) return seq_fail(h, CRNN_ERR_ARG, bad);
    if (a->batch == 0 || a->q_len == 0) return 0;
    const int64_t need = cross_attention_workspace(*a);
    if (need > 0 && (!a->workspace || a->workspace_bytes < need || !aligned(a->workspace, 256)))
      return seq_fail(h, CRNN_ERR_ARG, "crnn_cross_attention: the workspace is missing, too small or not 256-byte aligned (crnn_cross_attention_workspace tells the size)");
    SeqDevice dev;
    if (int rc = seq_enter(h, stream, &dev)) return rc;
    launch_cross_attention(*a, (hipStream_t)stream);
    return launched(h);
  } catch (const std::exception&) {
    return CRNN_ERR_NOMEM;
  }
}

}  // extern "C"
