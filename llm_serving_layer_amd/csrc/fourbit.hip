// The 4-bit cache's rows: append (quantise), read (the values held), and
// attention over it for any geometry. The format is fourbit.h's.
#include <algorithm>

#include "fourbit.h"

namespace pkv {

// ----------------------------------------------------------------- append ---

// A tiled row group (64 elements) by 8 lanes of 8 elements: 16-byte loads, a
// minimum and maximum over the 8 lanes, and each lane's codes: K one word, V four
// bytes. HBM-bound by its inputs (4 of 5 bytes); small launches by their chain:
// slot and row read together, then two reductions of three steps.
template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&x)[8]) {
  typedef T TV __attribute__((ext_vector_type(8)));
  const TV v = *reinterpret_cast<const TV*>(p);
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = Elem<T>::to_f(v[i]);
}

__device__ __forceinline__ uint32_t dpp_u(uint32_t v, int) {   // quad_perm [2,3,0,1]
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xf, 0xf, false);
}

template <typename T>
__global__ __launch_bounds__(256) void append_4bit_kernel(
    unsigned char* __restrict__ kpool, unsigned char* __restrict__ vpool, int64_t num_slots,
    FourBit f, const T* __restrict__ k, int64_t k_stride, const T* __restrict__ v,
    int64_t v_stride, const int32_t* __restrict__ slots, int64_t n_tokens, int32_t* status) {
  const int per_token = f.n_kv * f.groups;               // groups of a token's K or V
  const int64_t unit = (int64_t)blockIdx.x * 32 + (threadIdx.x >> 3);
  const int64_t total = n_tokens * 2 * per_token;
  const bool live = unit < total;
  const int64_t u = live ? unit : total - 1;
  const int64_t row = u / per_token;                      // (token, K or V)
  const int hq = (int)(u - row * per_token);
  const int64_t t = row >> 1;
  const bool is_v = row & 1;
  const int h = hq / f.groups, q = hq - h * f.groups;
  const int l = threadIdx.x & 7;
  const int64_t slot = slots[t];
  float x[8];
  load8((is_v ? v + t * v_stride : k + t * k_stride) + (int64_t)h * f.d + q * 64 + l * 8, x);
  float lo = INFINITY, hi = -INFINITY;
  bool odd = false;                                       // a NaN or an infinity
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    odd |= !(__builtin_fabsf(x[i]) < INFINITY);
    x[i] = fminf(fmaxf(x[i], -kF16Max), kF16Max);
    lo = fminf(lo, x[i]);
    hi = fmaxf(hi, x[i]);
  }
  lo = fminf(lo, dpp<0xB1>(lo));     // quad_perm [1,0,3,2]
  hi = fmaxf(hi, dpp<0xB1>(hi));
  lo = fminf(lo, dpp<0x4E>(lo));     // quad_perm [2,3,0,1]
  hi = fmaxf(hi, dpp<0x4E>(hi));
  lo = fminf(lo, dpp<0x141>(lo));    // row_half_mirror: the 8 lanes
  hi = fmaxf(hi, dpp<0x141>(hi));
  const uint64_t odds = __builtin_amdgcn_ballot_w64(odd);
  const bool none = (odds >> (threadIdx.x & 56)) & 0xffu;
  const uint32_t pair = none ? kNanPair : group_pair(lo, hi);
  const float step = none ? 0.f : pair_step(pair), zero = pair_zero(pair), inv = 1.f / step;
  uint32_t c[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) c[i] = code_of(x[i], step, inv, zero);
  // (V: dims 32 b + n and 32 b + 16 + n share a byte: lanes two apart)
  uint32_t mine[2] = {c[0] | c[1] << 8 | c[2] << 16 | c[3] << 24,
                      c[4] | c[5] << 8 | c[6] << 16 | c[7] << 24};
  const uint32_t other0 = dpp_u(mine[0], 0), other1 = dpp_u(mine[1], 0);
  if (!live) return;
  if (slot < 0 || slot >= num_slots) {
    if (hq == 0 && l == 0) flag(status, PKV_STATUS_BAD_SLOT);
    return;
  }
  const int64_t block = slot / f.ps;
  const int r = (int)(slot - block * f.ps);
  unsigned char* base = (is_v ? vpool : kpool) + block * f.block;
  unsigned char* codes = base + h * f.head_bytes;
  if (l == 0)
    reinterpret_cast<uint32_t*>(base + f.pairs)[(h * f.groups + q) * f.ps + r] = pair;
  if (!is_v) {
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) w |= c[i] << (4 * i);
    *reinterpret_cast<uint32_t*>(codes + k_byte(f, r, q * 64 + l * 8)) = w;
    return;
  }
  // lanes (l & 2) == 0 hold dims n, the others n + 16; each writes four of the
  // pair's eight bytes
  const bool upper = l & 2;
  const uint32_t low = upper ? other1 : mine[0], high = upper ? mine[1] : other0;
  const uint32_t bytes = low | high << 4;
  const int e = q * 64 + (l >> 2) * 32 + (l & 1) * 8 + (upper ? 4 : 0);
#pragma unroll
  for (int i = 0; i < 4; ++i) codes[v_byte(f, r, e + i)] = (unsigned char)(bytes >> (8 * i));
}

// Any geometry: a wave per (token, K or V, head), one group.
template <typename T>
__global__ __launch_bounds__(64) void append_4bit_any_kernel(
    unsigned char* __restrict__ kpool, unsigned char* __restrict__ vpool, int64_t num_slots,
    FourBit f, const T* __restrict__ k, int64_t k_stride, const T* __restrict__ v,
    int64_t v_stride, const int32_t* __restrict__ slots, int32_t* status) {
  const int64_t row = blockIdx.x / f.n_kv;
  const int h = (int)(blockIdx.x - row * f.n_kv);
  const int64_t t = row >> 1;
  const bool is_v = row & 1;
  const int lane = threadIdx.x;
  const int64_t slot = slots[t];
  if (slot < 0 || slot >= num_slots) {
    if (h == 0 && lane == 0) flag(status, PKV_STATUS_BAD_SLOT);
    return;
  }
  const T* src = (is_v ? v + t * v_stride : k + t * k_stride) + (int64_t)h * f.d;
  const int64_t block = slot / f.ps;
  const int r = (int)(slot - block * f.ps);
  unsigned char* base = (is_v ? vpool : kpool) + block * f.block;
  const int size = f.d / f.groups;
  for (int q = 0; q < f.groups; ++q) {
    float lo = INFINITY, hi = -INFINITY;
    bool odd = false;
    for (int i = lane; i < size; i += 64) {
      float x = Elem<T>::to_f(src[q * size + i]);
      odd |= !(__builtin_fabsf(x) < INFINITY);
      x = fminf(fmaxf(x, -kF16Max), kF16Max);
      lo = fminf(lo, x);
      hi = fmaxf(hi, x);
    }
    const bool none = __builtin_amdgcn_ballot_w64(odd) != 0;
    lo = -wave_max(-lo);
    hi = wave_max(hi);
    const uint32_t pair = none ? kNanPair : group_pair(lo, hi);
    const float step = none ? 0.f : pair_step(pair), zero = pair_zero(pair), inv = 1.f / step;
    if (lane == 0)
      reinterpret_cast<uint32_t*>(base + f.pairs)[(h * f.groups + q) * f.ps + r] = pair;
    for (int i = lane; i < size / 2; i += 64) {   // a byte: elements a and b
      const int a = f.tiled && is_v ? (i / 16) * 32 + i % 16 : 2 * i;
      const int b = f.tiled && is_v ? a + 16 : a + 1;
      uint32_t c[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float x = Elem<T>::to_f(src[q * size + (j ? b : a)]);
        x = fminf(fmaxf(x, -kF16Max), kF16Max);
        c[j] = code_of(x, step, inv, zero);
      }
      const int e = q * size + a;
      base[h * f.head_bytes + (is_v ? v_byte(f, r, e) : k_byte(f, r, e))] =
          (unsigned char)(c[0] | c[1] << 4);
    }
  }
}

// ------------------------------------------------------------------- read ---

// The values that slots hold, 8 elements a thread (2 where the layout is not
// tiled), rounded once to the pool's type.
template <typename T, int N>
__global__ __launch_bounds__(256) void read_4bit_kernel(
    const unsigned char* __restrict__ kpool, const unsigned char* __restrict__ vpool,
    int64_t num_slots, FourBit f, const int32_t* __restrict__ slots, int64_t n_rows,
    T* __restrict__ k, T* __restrict__ v, int32_t* status) {
  typedef T TV __attribute__((ext_vector_type(N)));
  const int per_row = f.n_kv * f.d / N;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= n_rows * 2 * per_row) return;
  const int64_t row = i / per_row;
  const int at = (int)(i - row * per_row) * N;
  const int64_t t = row >> 1;
  const bool is_v = row & 1;
  const int h = at / f.d, e = at - h * f.d;
  const int64_t slot = slots[t];
  TV out{};
  if (slot < 0 || slot >= num_slots) {
    if (at == 0) flag(status, PKV_STATUS_BAD_SLOT);
  } else {
    const int64_t block = slot / f.ps;
    const int r = (int)(slot - block * f.ps);
    const unsigned char* base = (is_v ? vpool : kpool) + block * f.block;
    const unsigned char* codes = base + h * f.head_bytes;
    const uint32_t pair =
        reinterpret_cast<const uint32_t*>(base + f.pairs)[(h * f.groups + group_of(f, e)) * f.ps + r];
    const float step = pair_step(pair), zero = pair_zero(pair);
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int b = codes[is_v ? v_byte(f, r, e + j) : k_byte(f, r, e + j)];
      const int half = is_v ? v_half(f, e + j) : k_half(f, e + j);
      out[j] = Elem<T>::from_f(__builtin_fmaf((float)(b >> (4 * half) & 15), step, zero));
    }
  }
  *reinterpret_cast<TV*>((is_v ? v : k) + t * f.n_kv * f.d + at) = out;
}

// ------------------------------------------------ attention, any geometry ---

// One wave per (query token, query head), 64 keys at a time: a lane a key for
// the scores, a lane up to four dims for the values, the running maximum and sum
// between. Everything in 32 bits. Slow by design: for geometries without a
// matrix-core kernel.
template <typename T>
__global__ __launch_bounds__(64) void attend_4bit_any_kernel(
    const T* __restrict__ q, T* __restrict__ out, const unsigned char* __restrict__ kpool,
    const unsigned char* __restrict__ vpool, int64_t num_blocks, FourBit f,
    const int32_t* __restrict__ cu_q, const int32_t* __restrict__ indptr,
    const int32_t* __restrict__ indices, const int32_t* __restrict__ kv_lens,
    const int32_t* __restrict__ batch_idx, int32_t n_seqs, int32_t n_heads, float scale_log2,
    int32_t* status) {
  __shared__ float qs[256];
  __shared__ float ps[64];
  __shared__ int32_t page_of[64];
  const int lane = threadIdx.x;
  const int tok = blockIdx.x / n_heads, hq = blockIdx.x - tok * n_heads;
  const int h = hq / (n_heads / f.n_kv);
  const int seq = batch_idx[tok];
  if (seq < 0 || seq >= n_seqs) return;
  const int q0 = cu_q[seq], q_len = cu_q[seq + 1] - q0;
  const int limit = kv_lens[seq] - q_len + (tok - q0) + 1;   // keys this token sees
  const int first_page = indptr[seq];
  const T* qr = q + ((int64_t)tok * n_heads + hq) * f.d;
  for (int i = lane; i < f.d; i += 64) qs[i] = Elem<T>::to_f(qr[i]);
  __syncthreads();
  float m = -INFINITY, l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
  for (int t0 = 0; t0 < limit; t0 += 64) {
    const int t = t0 + lane;
    const bool in = t < limit;
    float s = -INFINITY;
    int id = -1;
    if (in) {
      id = indices[first_page + t / f.ps];
      s = 0.f;
      if (id < 0 || id >= num_blocks) {
        flag(status, PKV_STATUS_BAD_PAGE);
        id = -1;                                     // read as zeros
      } else {
        const int r = t % f.ps;
        const unsigned char* base = kpool + (int64_t)id * f.block;
        const uint32_t* words =
            reinterpret_cast<const uint32_t*>(base + f.pairs) + h * f.groups * f.ps + r;
        for (int e = 0; e < f.d; e += 2) {           // (a byte of K: two elements)
          const uint32_t w = words[group_of(f, e) * f.ps];
          const int b = base[h * f.head_bytes + k_byte(f, r, e)];
          const float st = pair_step(w), z = pair_zero(w);
          s += qs[e] * __builtin_fmaf((float)(b & 15), st, z);
          s += qs[e + 1] * __builtin_fmaf((float)(b >> 4), st, z);
        }
      }
      s *= scale_log2;
    }
    const float m_new = fmaxf(m, wave_max(s));
    const float ref = m_new == -INFINITY ? 0.f : m_new;
    const float p = in ? __builtin_amdgcn_exp2f(s - ref) : 0.f;
    const float alpha = __builtin_amdgcn_exp2f(m - ref);     // (0 at first)
    m = m_new;
    l = l * alpha + wave_sum(p);
    __syncthreads();
    ps[lane] = p;
    page_of[lane] = id;
    __syncthreads();
    const int n = min(64, limit - t0);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int e = lane + 64 * j;
      if (e >= f.d) break;
      float acc = 0.f;
      for (int i = 0; i < n; ++i) {
        if (page_of[i] < 0) continue;
        const int r = (t0 + i) % f.ps;
        const unsigned char* base = vpool + (int64_t)page_of[i] * f.block;
        const uint32_t w = reinterpret_cast<const uint32_t*>(
            base + f.pairs)[(h * f.groups + group_of(f, e)) * f.ps + r];
        const int b = base[h * f.head_bytes + v_byte(f, r, e)];
        acc += ps[i] * __builtin_fmaf((float)(b >> (4 * v_half(f, e)) & 15), pair_step(w),
                                      pair_zero(w));
      }
      o[j] = o[j] * alpha + acc;
    }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int e = lane + 64 * j;
    if (e < f.d) out[((int64_t)tok * n_heads + hq) * f.d + e] = Elem<T>::from_f(o[j] / l);
  }
}

int check_4bit(int32_t n_kv, int32_t d, int32_t ps) {
  if (n_kv <= 0 || d <= 0 || ps <= 0) return fail(PKV_ERR_INVALID, "non-positive geometry");
  if (d > 256 || d % 2) return fail(PKV_ERR_INVALID, "head_dim=%d is odd or above 256", d);
  if ((int64_t)n_kv * ps * d > (1ll << 30))
    return fail(PKV_ERR_INVALID, "a block of %d x %d x %d elements is too large", ps, n_kv, d);
  return PKV_OK;
}

}  // namespace pkv

using namespace pkv;

extern "C" {

int64_t pkv_block_bytes_4bit(int32_t n_kv_heads, int32_t head_dim, int32_t page_size) {
  if (check_4bit(n_kv_heads, head_dim, page_size)) return 0;
  return four_bit(n_kv_heads, head_dim, page_size).block;
}

int pkv_append_4bit(void* k_pool, void* v_pool, int64_t num_blocks, const void* k,
                    int64_t k_stride, const void* v, int64_t v_stride,
                    const int32_t* slot_mapping, int64_t n_tokens, int32_t n_kv_heads,
                    int32_t head_dim, int32_t page_size, int32_t dtype, int32_t* status_word,
                    void* stream) {
  const int rc = check_4bit(n_kv_heads, head_dim, page_size);
  if (rc) return rc;
  const int eb = elem_bytes(dtype);
  if (!eb) return fail(PKV_ERR_INVALID, "unsupported dtype code %d", dtype);
  if (n_tokens < 0 || num_blocks < 0) return fail(PKV_ERR_INVALID, "negative count");
  if (n_tokens == 0) return PKV_OK;
  if (!k_pool || !v_pool || !k || !v || !slot_mapping)
    return fail(PKV_ERR_INVALID, "null pointer argument");
  const FourBit f = four_bit(n_kv_heads, head_dim, page_size);
  hipStream_t s = (hipStream_t)stream;
  const bool wide = f.tiled && ((uintptr_t)k | (uintptr_t)v | (uint64_t)(k_stride * eb) |
                                (uint64_t)(v_stride * eb)) % 16 == 0;
  const int64_t work = wide ? (n_tokens * 2 * f.n_kv * f.groups + 31) / 32 : n_tokens * 2 * f.n_kv;
  if (n_tokens > (1ll << 40) || work > 0x7fffffffLL)
    return fail(PKV_ERR_INVALID, "too many rows in one append");
  auto go = [&](auto type) {
    typedef decltype(type) T;
    if (wide)
      hipLaunchKernelGGL(append_4bit_kernel<T>, dim3((unsigned)work), dim3(256), 0, s,
                         (unsigned char*)k_pool, (unsigned char*)v_pool, num_blocks * page_size, f,
                         (const T*)k, k_stride, (const T*)v, v_stride, slot_mapping, n_tokens,
                         status_word);
    else
      hipLaunchKernelGGL(append_4bit_any_kernel<T>, dim3((unsigned)work), dim3(64), 0, s,
                         (unsigned char*)k_pool, (unsigned char*)v_pool, num_blocks * page_size, f,
                         (const T*)k, k_stride, (const T*)v, v_stride, slot_mapping, status_word);
  };
  if (dtype == PKV_DTYPE_F16) go(_Float16{});
  else if (dtype == PKV_DTYPE_BF16) go(__bf16{});
  else go(float{});
  PKV_LAUNCH_CHECK();
  return PKV_OK;
}

int pkv_read_4bit(const void* k_pool, const void* v_pool, int64_t num_blocks,
                  const int32_t* slots, int64_t n_rows, void* k, void* v, int32_t n_kv_heads,
                  int32_t head_dim, int32_t page_size, int32_t dtype, int32_t* status_word,
                  void* stream) {
  const int rc = check_4bit(n_kv_heads, head_dim, page_size);
  if (rc) return rc;
  const int eb = elem_bytes(dtype);
  if (!eb) return fail(PKV_ERR_INVALID, "unsupported dtype code %d", dtype);
  if (n_rows < 0 || num_blocks < 0) return fail(PKV_ERR_INVALID, "negative count");
  if (n_rows == 0) return PKV_OK;
  if (!k_pool || !v_pool || !k || !v || !slots)
    return fail(PKV_ERR_INVALID, "null pointer argument");
  const FourBit f = four_bit(n_kv_heads, head_dim, page_size);
  hipStream_t s = (hipStream_t)stream;
  const int n = f.tiled ? 8 : 2;
  if (((uintptr_t)k | (uintptr_t)v) % (n * eb))
    return fail(PKV_ERR_INVALID, "k and v have to be aligned to %d bytes", n * eb);
  const int64_t threads = n_rows > (1ll << 40) ? INT64_MAX - 255
                                               : n_rows * 2 * (n_kv_heads * head_dim / n);
  const int64_t blocks = (threads + 255) / 256;
  if (blocks > 0x7fffffffLL) return fail(PKV_ERR_INVALID, "too many rows in one read");
  auto go = [&](auto type, auto width) {
    typedef decltype(type) T;
    hipLaunchKernelGGL((read_4bit_kernel<T, decltype(width)::value>), dim3((unsigned)blocks),
                       dim3(256), 0, s, (const unsigned char*)k_pool, (const unsigned char*)v_pool,
                       num_blocks * page_size, f, slots, n_rows, (T*)k, (T*)v, status_word);
  };
  auto by_type = [&](auto width) {
    if (dtype == PKV_DTYPE_F16) go(_Float16{}, width);
    else if (dtype == PKV_DTYPE_BF16) go(__bf16{}, width);
    else go(float{}, width);
  };
  if (f.tiled) by_type(std::integral_constant<int, 8>{});
  else by_type(std::integral_constant<int, 2>{});
  PKV_LAUNCH_CHECK();
  return PKV_OK;
}

}  // extern "C"

namespace pkv {

// attend_4bit's geometries without a matrix-core kernel (arguments checked there)
int run_4bit_any(const pkv_4bit& b, const void* q, void* out, const void* k_pool,
                 const void* v_pool, float scale, hipStream_t s) {
  const FourBit f = four_bit(b.n_kv_heads, b.head_dim, b.page_size);
  const int64_t work = (int64_t)b.n_tokens * b.n_heads;
  if (work > 0x7fffffffLL) return fail(PKV_ERR_INVALID, "too many query rows");
  auto go = [&](auto type) {
    typedef decltype(type) T;
    hipLaunchKernelGGL(attend_4bit_any_kernel<T>, dim3((unsigned)work), dim3(64), 0, s,
                       (const T*)q, (T*)out, (const unsigned char*)k_pool,
                       (const unsigned char*)v_pool, b.num_blocks, f, b.cu_query_lens, b.kv_indptr,
                       b.kv_indices, b.kv_lens, b.batch_indices, b.n_seqs, b.n_heads,
                       scale * kLog2e, b.status_word);
  };
  if (b.dtype == PKV_DTYPE_F16) go(_Float16{});
  else if (b.dtype == PKV_DTYPE_BF16) go(__bf16{});
  else go(float{});
  PKV_LAUNCH_CHECK();
  return PKV_OK;
}

}  // namespace pkv
