// KV append with the position rotation on the way: a step's q, k and v rows
// are read once, as the projection left them; q comes back rotated, rotated k
// and plain v go to their slots of the pool.
//
// Of each head's D elements the first R (the rotary dims) form R / 2 pairs,
// (i, i + R / 2) or, interleaved, (2 i, 2 i + 1); pair i of a token at position
// p turns by p f_i. The table holds c = cos(p f_i) and s = sin(p f_i) in 32
// bits (computed in 64 on the host side), [position][cos, sin][R / 2]:
//   a' = a c - b s,   b' = b c + a s
// in 32 bits, rounded once to the pool dtype. Elements from R on are copied.
//
// Pure data movement otherwise: bound by the rows' bytes for prompts (5437
// tokens of 32 + 2 x 8 heads of 128, bf16: 23.2 us, 5.8 TB/s of the rows read and
// written), by its chain of two round trips (position, then table) for a few
// tokens (1 of head_dim 64: 2.3 us, 256 of head_dim 128: 3.7, 777 of 64: 4.4).
#include <algorithm>

#include "pkv_common.h"

namespace pkv {

struct RotatedArgs {
  const void* q; const void* k; const void* v;
  void* q_out; void* k_pool; void* v_pool;
  int64_t q_stride, k_stride, v_stride;      // elements from token to token
  const int32_t* slots; const int64_t* positions; const float* table;
  int64_t num_slots, max_positions, n_tokens;
  int32_t n_heads, n_kv_heads, head_dim, rotary_dim, interleaved;
  int32_t units, tokens;                     // per token; per workgroup
  int32_t* status;
};

// One unit is U elements of a head: U / 2 pairs of its rotary part (U / 2
// elements of either half, or U consecutive ones interleaved), or U
// consecutive elements of the rest. U = 16 with 16-byte accesses; U = 2 with
// element accesses for row strides, addresses or rotary dims that the former
// does not fit (an odd head_dim's last unit holds one element).
template <typename T, int U>
__global__ __launch_bounds__(1024) void append_rotated_kernel(RotatedArgs a) {
  constexpr int H = U / 2;
  typedef T vec __attribute__((ext_vector_type(H)));
  typedef float fvec __attribute__((ext_vector_type(H)));
  const int tl = threadIdx.x / a.units;
  const int64_t t = (int64_t)blockIdx.x * a.tokens + tl;
  if (tl >= a.tokens || t >= a.n_tokens) return;
  const int64_t pos = a.positions[t];
  const int64_t slot = a.slots[t];
  const bool at = pos >= 0 && pos < a.max_positions;
  const bool ok = slot >= 0 && slot < a.num_slots;
  const int D = a.head_dim, R = a.rotary_dim, per_head = (D + U - 1) / U;
  const int first = threadIdx.x - tl * a.units, step = a.tokens > 1 ? a.units : blockDim.x;
  if (first == 0) {
    if (!at) flag(a.status, PKV_STATUS_BAD_POSITION);
    if (!ok) flag(a.status, PKV_STATUS_BAD_SLOT);
  }
  const float* row = a.table + (at ? pos : 0) * R;
  for (int u = first; u < a.units; u += step) {
    int head = u / per_head;
    const int c = u - head * per_head;
    const bool is_v = head >= a.n_heads + a.n_kv_heads, is_q = head < a.n_heads;
    const T* src;
    T* dst;
    if (is_q) {
      src = (const T*)a.q + t * a.q_stride + (int64_t)head * D;
      dst = (T*)a.q_out + (t * a.n_heads + head) * D;
    } else {
      head -= is_v ? a.n_heads + a.n_kv_heads : a.n_heads;
      src = (is_v ? (const T*)a.v + t * a.v_stride : (const T*)a.k + t * a.k_stride) +
            (int64_t)head * D;
      dst = (T*)(is_v ? a.v_pool : a.k_pool) +
            ((ok ? slot : 0) * a.n_kv_heads + head) * (int64_t)D;
    }
    const bool turn = !is_v && c * U < R;
    // the unit's two groups of H elements
    const int e0 = turn && !a.interleaved ? c * H : c * U;
    const int e1 = turn && !a.interleaved ? e0 + R / 2 : e0 + H;
    const bool two = e1 < D;
    vec x = *reinterpret_cast<const vec*>(src + e0), y{};
    if (two) y = *reinterpret_cast<const vec*>(src + e1);
    if (turn) {
      const fvec cs = *reinterpret_cast<const fvec*>(row + c * H);
      const fvec sn = *reinterpret_cast<const fvec*>(row + R / 2 + c * H);
      if (!a.interleaved) {
#pragma unroll
        for (int i = 0; i < H; ++i) {
          const float p = Elem<T>::to_f(x[i]), r = Elem<T>::to_f(y[i]);
          x[i] = Elem<T>::from_f(p * cs[i] - r * sn[i]);
          y[i] = Elem<T>::from_f(r * cs[i] + p * sn[i]);
        }
      } else {
        T e[U];
#pragma unroll
        for (int i = 0; i < H; ++i) { e[i] = x[i]; e[H + i] = y[i]; }
#pragma unroll
        for (int i = 0; i < H; ++i) {
          const float p = Elem<T>::to_f(e[2 * i]), r = Elem<T>::to_f(e[2 * i + 1]);
          e[2 * i] = Elem<T>::from_f(p * cs[i] - r * sn[i]);
          e[2 * i + 1] = Elem<T>::from_f(r * cs[i] + p * sn[i]);
        }
#pragma unroll
        for (int i = 0; i < H; ++i) { x[i] = e[i]; y[i] = e[H + i]; }
      }
    }
    // a token without a table row gets zero queries and no row in the cache
    if (!at) { x = vec{}; y = vec{}; }
    if (is_q || (ok && at)) {
      *reinterpret_cast<vec*>(dst + e0) = x;
      if (two) *reinterpret_cast<vec*>(dst + e1) = y;
    }
  }
}

template <typename T>
static int launch_rotated(RotatedArgs& a, bool wide, hipStream_t s) {
  const int U = wide ? 16 : 2;
  const int64_t units =
      (int64_t)(a.n_heads + 2 * (int64_t)a.n_kv_heads) * ((a.head_dim + U - 1) / U);
  if (units > 0x7fffffffLL) return fail(PKV_ERR_INVALID, "too many heads");
  a.units = (int32_t)units;
  // tokens share a workgroup of 256 where a token needs less; a token takes up
  // to 1024 threads, each several units beyond
  a.tokens = units < 256 ? (int32_t)(256 / units) : 1;
  const int threads = (int)std::min<int64_t>(1024, (units * a.tokens + 63) / 64 * 64);
  const int64_t blocks = (a.n_tokens + a.tokens - 1) / a.tokens;
  if (blocks > 0x7fffffffLL) return fail(PKV_ERR_INVALID, "too many rows in one append");
  if (wide)
    hipLaunchKernelGGL((append_rotated_kernel<T, 16>), dim3((unsigned)blocks), dim3(threads), 0, s, a);
  else
    hipLaunchKernelGGL((append_rotated_kernel<T, 2>), dim3((unsigned)blocks), dim3(threads), 0, s, a);
  PKV_LAUNCH_CHECK();
  return PKV_OK;
}

}  // namespace pkv

using namespace pkv;

extern "C" int pkv_append_rotated(void* k_pool, void* v_pool, int64_t num_slots, const void* q,
                                  int64_t q_stride, void* q_out, const void* k, int64_t k_stride,
                                  const void* v, int64_t v_stride, const int32_t* slot_mapping,
                                  const int64_t* positions, int64_t n_tokens, const float* table,
                                  int64_t max_positions, int32_t rotary_dim, int32_t interleaved,
                                  int32_t n_heads, int32_t n_kv_heads, int32_t head_dim,
                                  int32_t dtype, int32_t* status_word, void* stream) {
  const int eb = elem_bytes(dtype);
  if (!eb) return fail(PKV_ERR_INVALID, "unsupported dtype code %d", dtype);
  if (n_heads <= 0 || n_kv_heads <= 0 || head_dim <= 0 || num_slots < 0 || n_tokens < 0 ||
      max_positions <= 0)
    return fail(PKV_ERR_INVALID, "non-positive geometry");
  if (rotary_dim <= 0 || rotary_dim % 2 || rotary_dim > head_dim)
    return fail(PKV_ERR_INVALID, "rotary_dim %d is not an even number in [2, head_dim %d]",
                rotary_dim, head_dim);
  if (n_tokens == 0) return PKV_OK;
  if (!k_pool || !v_pool || !q || !q_out || !k || !v || !slot_mapping || !positions || !table)
    return fail(PKV_ERR_INVALID, "null pointer argument");
  RotatedArgs a{q, k, v, q_out, k_pool, v_pool, q_stride, k_stride, v_stride, slot_mapping,
                positions, table, num_slots, max_positions, n_tokens, n_heads, n_kv_heads,
                head_dim, rotary_dim, interleaved, 0, 0, status_word};
  const uintptr_t at = (uintptr_t)q | (uintptr_t)q_out | (uintptr_t)k | (uintptr_t)v |
                       (uintptr_t)k_pool | (uintptr_t)v_pool | (uintptr_t)table |
                       (uintptr_t)(q_stride * eb) | (uintptr_t)(k_stride * eb) |
                       (uintptr_t)(v_stride * eb);
  const bool wide = at % 16 == 0 && rotary_dim % 16 == 0 && head_dim % 16 == 0;
  hipStream_t s = (hipStream_t)stream;
  if (dtype == PKV_DTYPE_F16) return launch_rotated<_Float16>(a, wide, s);
  if (dtype == PKV_DTYPE_BF16) return launch_rotated<__bf16>(a, wide, s);
  return launch_rotated<float>(a, wide, s);
}

static_assert(sizeof(pkv_rotated) == 104, "the layout the Python binding fills");

extern "C" int pkv_append_rotated_batch(const void* batch, void* k_pool, void* v_pool,
                                        const void* q, int64_t q_stride, void* q_out,
                                        const void* k, int64_t k_stride, const void* v,
                                        int64_t v_stride, void* lo, void* hi, void* stream) {
  if (!batch) return fail(PKV_ERR_INVALID, "null batch");
  const pkv_rotated& b = *static_cast<const pkv_rotated*>(batch);
  const int rc = pkv_append_rotated(k_pool, v_pool, b.num_blocks * b.page_size, q, q_stride, q_out,
                                    k, k_stride, v, v_stride, b.slot_mapping, b.positions,
                                    b.n_tokens, b.table, b.max_positions, b.rotary_dim,
                                    b.interleaved, b.n_heads, b.n_kv_heads, b.head_dim, b.dtype,
                                    b.status_word, stream);
  if (rc || b.n_complete <= 0) return rc;
  return pkv_page_bounds(k_pool, 0, lo, hi, 0, 1, b.num_blocks, b.complete, b.n_complete,
                         b.n_kv_heads, b.head_dim, b.page_size, b.dtype, b.status_word, stream);
}
