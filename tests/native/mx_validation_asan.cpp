// Host AddressSanitizer run over the argument validation of the 4-bit token cache's and the
// page operators' C entry points (mx_api.hip with host-side ASan, its kernels' objects as they are).
// Every call is rejected by validation before any launch, or is a pure host query of a workspace
// size, so it needs no GPU. Well-formed attention calls are checked for a plan that fits them.
//
// Prints "mx-asan: N calls, M rejected" and exits 0; an ASan report aborts.

#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <random>

#include "iak.h"

namespace {

std::mt19937_64 rng(20261206);

template <typename T> void random_bytes(T& s) {
  unsigned char* p = reinterpret_cast<unsigned char*>(&s);
  for (size_t i = 0; i < sizeof(T); ++i) p[i] = static_cast<unsigned char>(rng());
}

int32_t pick_int() {
  static const int32_t v[] = {-1, 0, 1, 2, 3, 4, 7, 8, 15, 16, 17, 31, 32, 64, 100, 128, 255, 256, 1024, 4097,
                              65535, 65536, 1 << 24, 0x7FFFFF0, 0x7FFFFFFF, (int32_t)0x80000000};
  return v[rng() % (sizeof(v) / sizeof(v[0]))];
}

int calls = 0, rejected = 0;
void count(iak_status st) {
  ++calls;
  if (st != IAK_OK) ++rejected;
  (void)iak_last_error();
}
void must_reject(iak_status st, const char* what) {
  count(st);
  if (st == IAK_OK) {
    std::printf("mx-asan: %s was not rejected\n", what);
    std::exit(1);
  }
}

void* const fake = reinterpret_cast<void*>(0x100000);

void attention(int n) {
  size_t bytes = 0;
  for (int i = 0; i < n; ++i) {
    iak_mx_attention_args a;
    random_bytes(a);
    if (rng() % 4) {
      a.batch = pick_int(); a.q_len = pick_int(); a.num_q_heads = pick_int(); a.num_kv_heads = pick_int();
      a.head_dim = rng() % 2 ? 64 : 128; a.page_size = 16; a.table_width = pick_int(); a.num_pages = pick_int();
      a.q_dtype = pick_int() & 3; a.out_dtype = pick_int() & 3; a.causal = pick_int() & 1; a.splits = pick_int();
      a.sm_scale = 0.1f;
      a.k_codes = a.v_codes = a.k_scales = a.v_scales = fake;
    }
    count(iak_mx_attention_workspace(&a, &bytes));
  }
  for (int i = 0; i < n; ++i) {
    iak_mx_attention_args a{};
    a.num_kv_heads = 1 + (int)(rng() % 16);
    a.num_q_heads = a.num_kv_heads * (1 + (int)(rng() % 16));
    a.batch = 1 + (int)(rng() % 64); a.q_len = 1 + (int)(rng() % (rng() % 2 ? 4 : 600));
    a.head_dim = rng() % 2 ? 64 : 128; a.page_size = 16; a.table_width = (int)(rng() % 5000); a.num_pages = 1000;
    a.q_dtype = (int)(rng() % 3); a.splits = rng() % 2 ? 0 : (int)(rng() % 70);
    a.q = a.out = fake;
    a.page_table = a.valid_tokens = static_cast<const int32_t*>(fake);
    a.k_codes = a.v_codes = a.k_scales = a.v_scales = fake;
    a.sm_scale = 0.1f;
    const iak_status st = iak_mx_attention_workspace(&a, &bytes);
    count(st);
    // per part of two table entries at least a maximum, a sum and head_dim values for each of the
    // rows, in tiles of 16 to 256; more parts than tiles
    const int rows = a.q_len * (a.num_q_heads / a.num_kv_heads);
    const double value = 4.0 * (2 + a.head_dim) * a.batch * a.num_kv_heads;
    const double least = value * 16 * ((rows + 15) / 16), most = value * 256 * ((rows + 255) / 256) * (a.table_width / 2 + 1);
    if (st != IAK_OK || (bytes != 0 && (bytes < least || bytes > most + 8192)) || (a.splits == 1 && bytes != 0)) {
      std::printf("mx-asan: workspace of %zu bytes for a well-formed call (B=%d L=%d Hq=%d Hkv=%d W=%d splits=%d)\n", bytes,
                  a.batch, a.q_len, a.num_q_heads, a.num_kv_heads, a.table_width, a.splits);
      std::exit(1);
    }
    if (bytes) {
      must_reject(iak_mx_attention(&a, nullptr, bytes, nullptr), "no workspace");
      must_reject(iak_mx_attention(&a, fake, bytes - 1, nullptr), "a short workspace");
      must_reject(iak_mx_attention(&a, reinterpret_cast<void*>(0x100008), bytes, nullptr), "an unaligned workspace");
    }
    a.out = nullptr;
    must_reject(iak_mx_attention(&a, fake, bytes, nullptr), "no output");
  }
  must_reject(iak_mx_attention_workspace(nullptr, &bytes), "NULL");
  must_reject(iak_mx_attention(nullptr, nullptr, 0, nullptr), "NULL");
}

void tokens(int n) {
  for (int i = 0; i < n; ++i) {
    iak_mx_tokens_args a;
    random_bytes(a);
    if (rng() % 2) {
      a.batch = pick_int(); a.count = pick_int(); a.num_kv_heads = pick_int(); a.head_dim = 64 * (pick_int() & 3);
      a.page_size = 16; a.table_width = pick_int(); a.num_pages = pick_int(); a.dtype = pick_int() & 3;
    }
    if (a.batch == 0) a.batch = 1;
    if (a.count == 0) a.count = 1;
    a.k = nullptr;                        // never launched
    must_reject(iak_mx_append_tokens(&a, nullptr), "tokens from nowhere");
    must_reject(iak_mx_read_tokens(&a, nullptr), "tokens to nowhere");
  }
  must_reject(iak_mx_append_tokens(nullptr, nullptr), "NULL");
  must_reject(iak_mx_read_tokens(nullptr, nullptr), "NULL");
}

void sequences(int n) {
  size_t bytes = 0;
  for (int i = 0; i < n; ++i) {
    iak_sequences_args a;
    random_bytes(a);
    a.num_seqs = pick_int(); a.rows_per_seq = pick_int(); a.table_width = pick_int(); a.page_size = pick_int();
    a.num_pages = pick_int(); a.count = pick_int(); a.num_arrays = pick_int();
    a.page_table = a.valid_tokens = a.refs = static_cast<int32_t*>(fake);
    a.seqs = a.parents = a.new_tokens = static_cast<const int32_t*>(fake);
    const iak_status st = iak_sequences_workspace(&a, &bytes);
    count(st);
    a.missing = nullptr;                  // never launched
    must_reject(iak_grow_sequences(&a, fake, ~(size_t)0, nullptr), "grow without a verdict");
    must_reject(iak_fork_sequences(&a, fake, ~(size_t)0, nullptr), "fork without a verdict");
    a.missing = static_cast<int32_t*>(fake);
    must_reject(iak_fork_sequences(&a, fake, st == IAK_OK ? bytes - 1 : 0, nullptr), "a short workspace");
    a.rows_per_seq = -1;
    must_reject(iak_free_sequences(&a, nullptr), "rows below zero");
  }
  must_reject(iak_sequences_workspace(nullptr, &bytes), "NULL");
  must_reject(iak_free_sequences(nullptr, nullptr), "NULL");
  must_reject(iak_grow_sequences(nullptr, fake, 1, nullptr), "NULL");
  must_reject(iak_fork_sequences(nullptr, fake, 1, nullptr), "NULL");
}

void pages(int n) {
  size_t bytes = 0;
  for (int i = 0; i < n; ++i) {
    iak_compact_pages_args c;
    random_bytes(c);
    c.num_rows = pick_int(); c.table_width = pick_int(); c.page_size = pick_int(); c.num_pages = pick_int();
    c.num_arrays = pick_int();
    count(iak_compact_pages_workspace(&c, &bytes));
    c.page_size = 0;
    must_reject(iak_compact_pages(&c, fake, ~(size_t)0, nullptr), "pages of no tokens");
    iak_copy_pages_args p;
    random_bytes(p);
    p.num_pages = 1 + (int64_t)(rng() % 100); p.count = 1; p.num_arrays = pick_int(); p.src = nullptr;
    if (p.num_arrays == 0) p.num_arrays = 1;
    must_reject(iak_copy_pages(&p, nullptr), "copies from nowhere");
  }
  must_reject(iak_compact_pages_workspace(nullptr, &bytes), "NULL");
  must_reject(iak_compact_pages(nullptr, fake, 1, nullptr), "NULL");
  must_reject(iak_copy_pages(nullptr, nullptr), "NULL");
}

}  // namespace

int main() {
  attention(20000);
  tokens(5000);
  sequences(5000);
  pages(5000);
  std::printf("mx-asan: %d calls, %d rejected\n", calls, rejected);
  return 0;
}
