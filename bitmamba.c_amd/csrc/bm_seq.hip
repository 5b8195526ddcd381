// Host checks of the batched recurrence calls (bm_seq.h).
#include "bm_seq.h"

namespace bm {

hipStream_t stream_of(void* stream) {
  return stream ? (hipStream_t)stream : (hipStream_t)bm_hip_stream();
}

bool check_rows(const char* op, const char* name, const void* p, int64_t stride, int64_t width,
                int64_t rows, size_t elem) {
  // without rows nothing is read or written: an empty tensor's address may be null
  if ((!p && rows > 0) || (uintptr_t)p % elem || stride < width || stride >= (1 << 24)) {
    bm_set_error("%s: %s needs an address on %zu bytes and a row stride of %lld to 2^24 - 1 (%lld)", op,
                 name, elem, (long long)width, (long long)stride);
    return false;
  }
  return true;
}

bool check_apart(const char* op, const char* name, const void* p, int64_t stride, int64_t width,
                 const void* y, int64_t y_stride, int64_t y_width, int64_t rows, size_t elem,
                 bool same_ok) {
  if (rows <= 0 || !p) return true;
  const uintptr_t p0 = (uintptr_t)p, y0 = (uintptr_t)y;
  const uintptr_t p1 = p0 + ((rows - 1) * stride + width) * elem;
  const uintptr_t y1 = y0 + ((rows - 1) * y_stride + y_width) * elem;
  if (p1 <= y0 || y1 <= p0) return true;
  if (same_ok && p == y && stride == y_stride) return true;
  if (stride == y_stride) {
    // columns of one buffer: y's first column, seen from p's, within a row
    const int64_t bytes = stride * (int64_t)elem;
    const int64_t d = y0 >= p0 ? (int64_t)(y0 - p0) % bytes
                               : (bytes - (int64_t)(p0 - y0) % bytes) % bytes;
    if (d >= width * (int64_t)elem && d + y_width * (int64_t)elem <= bytes) return true;
  }
  bm_set_error("%s: y overlaps %s", op, name);
  return false;
}

bool check_seqs(const char* op, int n_seqs, int n_tokens, const int32_t* seq_start,
                const int32_t* slots, const float* state, int64_t state_stride, int n_slots,
                int64_t slot_floats, bool step) {
  if (n_seqs < 0 || n_seqs > (1 << 20) || (!step && (n_tokens < 0 || n_tokens >= (1 << 30)))) {
    bm_set_error("%s: n_seqs=%d n_tokens=%d (up to 2^20 and below 2^30)", op, n_seqs, n_tokens);
    return false;
  }
  if (!step && !seq_start && n_seqs > 1) {
    bm_set_error("%s: %d sequences need seq_start", op, n_seqs);
    return false;
  }
  if (state && slots && n_seqs > (1 << 16)) {  // each looks for its slot among those before it
    bm_set_error("%s: a list of %d slots (up to 2^16)", op, n_seqs);
    return false;
  }
  if (((uintptr_t)seq_start | (uintptr_t)slots | (uintptr_t)state) % 4) {
    bm_set_error("%s: seq_start, slots and state need addresses on 4 bytes", op);
    return false;
  }
  if (state && (n_slots < 1 || state_stride < slot_floats || (!slots && n_slots < n_seqs))) {
    bm_set_error("%s: %d slots of stride %lld for %d sequences of %lld floats", op, n_slots,
                 (long long)state_stride, n_seqs, (long long)slot_floats);
    return false;
  }
  return true;
}

}  // namespace bm
