// Attention over pages held in 4 bits (layout: kv4.cuh): a warp per (token row, query head).
#include "common.cuh"
#include "kv4.cuh"

template <int D>
__global__ void __launch_bounds__(128)
kv4_attention_kernel(const __nv_bfloat16* __restrict__ q, long long q_stride, const unsigned char* __restrict__ cache,
                     const int* __restrict__ rows, const int* __restrict__ seq_of_token,
                     const int* __restrict__ positions, const int* __restrict__ items,
                     const int* __restrict__ block_tables, int table_stride, int table_rows,
                     int table_width, int T, __nv_bfloat16* __restrict__ out, long long out_stride, int nh, int nkv, int page_size, int num_pages,
                     int window, int keep, float scale, int* __restrict__ err) {
  constexpr int N = D / 32, NG = D / KV4_GROUP, REC = kv4_record(D);
  const int lane = threadIdx.x & 31, head = blockIdx.y * 4 + (threadIdx.x >> 5);
  if (head >= nh) return;
  int t, b, p;
  if (items) {
    const int* it = items + 4 * blockIdx.z;
    if ((int)blockIdx.x >= it[2]) return;
    t = it[1] + blockIdx.x, b = it[0], p = it[3] + blockIdx.x;
  } else {
    t = rows ? rows[blockIdx.x] : blockIdx.x;
    const int ok = t >= 0 && t < T;
    b = ok ? seq_of_token[t] : -1, p = ok ? positions[t] : 0;
  }
  if (t < 0 || t >= T || b < 0 || b >= table_rows) {
    if (lane == 0) atomicOr(err, BF_ERR_PAGE);
    return;
  }
  const int h = head / (nh / nkv), i0 = lane * N, g = i0 / 64;
  float qf[N], o[N], m = -INFINITY, l = 0.f;
  for (int e = 0; e < N; ++e) qf[e] = __bfloat162float(q[t * q_stride + head * D + i0 + e]), o[e] = 0.f;
  for (int j = 0; j <= p; ++j) {
    if (window > 0 && j <= p - window && j >= keep) {
      j = p - window;
      continue;
    }
    const int at = j / page_size;
    const int page = at < table_width ? block_tables[(size_t)b * table_stride + at] : -1;
    if (page < 0 || page >= num_pages) {
      if (lane == 0) atomicOr(err, BF_ERR_PAGE);
      continue;
    }
    const int off = j % page_size, tok = off % 8;
    const unsigned char* rec = cache + (((size_t)page * nkv + h) * (page_size / 8) + off / 8) * REC;
    const unsigned kp = *reinterpret_cast<const unsigned*>(rec + kv4_key_params_at(D) + (tok * NG + g) * 4);
    const unsigned vp = *reinterpret_cast<const unsigned*>(rec + kv4_value_params_at(D) + (tok * NG + g) * 4);
    float s = 0.f;
    for (int e = 0; e < N; ++e) {
      const int c = rec[kv4_key_byte(D, tok, i0 + e)] >> ((i0 + e) % 2 * 4) & 15;
      s += qf[e] * fmaf(kv4_scale(kp), (float)c, kv4_low(kp));
    }
    s = warp_sum(s) * scale;
    const float mn = fmaxf(m, s), f = mn == m ? 1.f : __expf(m - mn), w = __expf(s - mn);
    l = l * f + w;
    for (int e = 0; e < N; ++e) {
      const int c = rec[kv4_value_byte(D, tok, i0 + e)] >> ((i0 + e) % 2 * 4) & 15;
      o[e] = o[e] * f + w * fmaf(kv4_scale(vp), (float)c, kv4_low(vp));
    }
    m = mn;
  }
  for (int e = 0; e < N; ++e) out[t * out_stride + head * D + i0 + e] = __float2bfloat16_rn(o[e] / l);
}

BF_EXPORT int bf_kv4_attention(const void* q, long long q_stride, const void* cache, const int* rows, const int* seq_of_token,
                               const int* positions, const int* items, int n, int max_rows, int T,
                               const int* block_tables, int table_stride, int table_rows, int table_width,
                               void* out, long long out_stride,
                               int nh, int nkv, int d, int page_size, int num_pages, int window, int keep,
                               float scale, int* err, cudaStream_t stream) {
  if (n <= 0 || max_rows <= 0) return 0;
  const dim3 grid(items ? max_rows : n, (nh + 3) / 4, items ? n : 1);
  auto run = [&](auto kern) {
    kern<<<grid, 128, 0, stream>>>((const __nv_bfloat16*)q, q_stride, (const unsigned char*)cache, rows, seq_of_token,
                                   positions, items, block_tables, table_stride, table_rows, table_width, T,
                                   (__nv_bfloat16*)out, out_stride, nh, nkv, page_size, num_pages, window, keep, scale, err);
    return bf_launch_status();
  };
  if (d == 64) return run(kv4_attention_kernel<64>);
  if (d == 128) return run(kv4_attention_kernel<128>);
  if (d == 256) return run(kv4_attention_kernel<256>);
  return (int)cudaErrorInvalidValue;
}
