// A chunk of one sequence through the 8-bit cache from C++ (include/ms_b200_shim.hpp): head norms, write, read back, attention.  Inputs from a
// file (queries, keys, values, gains, factors, as F32), outputs to one: the test compares them with the same calls through the mirror.
#include <cstdio>
#include <cstdlib>
#include <vector>
#include "ms_b200_shim.hpp"

static ms::Buffer device(const void* src, size_t bytes) {
  void* d = nullptr;
  ms::check(msb_device_alloc(bytes, &d), "alloc");
  if (src) ms::check(msb_copy_to_device(d, src, bytes, nullptr), "copy");
  return ms::Buffer{d, 0, bytes};
}

int main(int argc, char** argv) {
  if (argc < 3) return 1;
  const int n = 70, heads = 12, kvh = 3, dim = 64, block = 32, blocks = 5;
  const size_t nq = (size_t)n * heads * dim, nk = (size_t)n * kvh * dim;
  std::vector<float> in(nq + 2 * nk + 2 * dim + (size_t)n * dim);
  FILE* f = std::fopen(argv[1], "rb");
  if (!f || std::fread(in.data(), 4, in.size(), f) != in.size()) return 2;
  std::fclose(f);
  const float* p = in.data();
  ms::Enc e;
  ms::attn::HeadNormRope r;
  r.heads = heads; r.kv_heads = kvh; r.dim = dim; r.n_tokens = n; r.n_pos = n; r.rot = dim; r.first = 0; r.halves = true;
  r.q = r.q_out = device(p, 4 * nq); p += nq;
  r.k = r.k_out = device(p, 4 * nk); p += nk;
  ms::Buffer v = device(p, 4 * nk); p += nk;
  r.q_w = device(p, 4 * dim); p += dim;
  r.k_w = device(p, 4 * dim); p += dim;
  r.cs = device(p, 4 * (size_t)n * dim);
  std::vector<int> pos(n);
  for (int i = 0; i < n; i++) pos[i] = i;
  r.pos = device(pos.data(), 4 * (size_t)n);
  ms::attn::encode_head_norm_rope(e, r);
  ms::attn::Kv8Cache c;
  c.n_blocks = blocks; c.kv_heads = kvh; c.head_dim = dim; c.block = block;
  c.k = device(nullptr, c.code_bytes()); c.v = device(nullptr, c.code_bytes());
  c.k_scale = device(nullptr, c.scale_bytes()); c.v_scale = device(nullptr, c.scale_bytes());
  const int start[2] = {0, n}, len[1] = {n}, table[3] = {4, 0, 2};
  ms::attn::Kv8Batch b;
  b.n_seq = 1; b.n_tokens = n; b.max_new = n; b.max_len = n; b.table_stride = 3;
  b.seq_start = device(start, sizeof start); b.kv_len = device(len, sizeof len); b.table = device(table, sizeof table);
  ms::attn::encode_kv8_write(e, c, b, MSB_F32, r.k, v);
  ms::Buffer ko = device(nullptr, 4 * nk), vo = device(nullptr, 4 * nk), out = device(nullptr, 4 * nq);
  ms::attn::encode_kv8_read(e, c, b, MSB_F32, ko, vo);
  const size_t bytes = ms::attn::kv8_attn_scratch_bytes(c, b, heads);
  ms::attn::encode_kv8_attn(e, c, b, MSB_F32, r.q, heads, 0.125f, out, device(nullptr, bytes), 40);
  e.wait();
  std::vector<float> host(nq + 2 * nk);
  ms::check(msb_copy_to_host(host.data(), out.ptr(), 4 * nq, nullptr), "copy");
  ms::check(msb_copy_to_host(host.data() + nq, ko.ptr(), 4 * nk, nullptr), "copy");
  ms::check(msb_copy_to_host(host.data() + nq + nk, vo.ptr(), 4 * nk, nullptr), "copy");
  f = std::fopen(argv[2], "wb");
  if (!f || std::fwrite(host.data(), 4, host.size(), f) != host.size()) return 3;
  std::fclose(f);
  return 0;
}
