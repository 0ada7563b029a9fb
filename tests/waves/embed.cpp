// embed.cpp -- the embedding's kernels on the CPU: every buffer lies between pages that cannot be touched, its first byte or its last
// against one, so an access out of range ends the program. Sums are of small whole numbers, exact in any order.
//
//   embed TOKENS VOCAB COLS IDS PADDING ADD IDS64 TABLE_F32 GRADIENT_F32 APART
//
// IDS: text (a few are most of the tokens, a third of the places padding's where there is any), same, padding (all of
// them), outside (half of them no row's), any. APART: elements between rows beyond COLS.
#include "tm_embed.hip"

#include <sys/mman.h>

#include <random>
#include <string>
#include <vector>

namespace {

constexpr size_t kPage = 4096;

char* between_pages(size_t bytes, bool at_end, size_t align) {
  const size_t room = (bytes + kPage - 1) / kPage * kPage;
  char* p = static_cast<char*>(mmap(nullptr, room + 2 * kPage, PROT_NONE, MAP_PRIVATE | MAP_ANONYMOUS, -1, 0));
  if (p == MAP_FAILED || mprotect(p + kPage, room, PROT_READ | PROT_WRITE)) std::abort();
  memset(p + kPage, 0xC3, room);
  return p + kPage + (at_end ? (room - bytes) / align * align : 0);
}

struct Values {
  char* p;
  bool f32;
  size_t bytes;
  Values(int64_t n, bool f, bool at_end) : f32(f), bytes(n * (f ? 4 : 2)) { p = between_pages(bytes, at_end, f ? 4 : 2); }
  void set(int64_t i, float v) {
    if (f32) reinterpret_cast<float*>(p)[i] = v;
    else reinterpret_cast<uint16_t*>(p)[i] = static_cast<uint16_t>(__float_as_uint(v) >> 16);  // (numbers that bf16 holds)
  }
  float get(int64_t i) const {
    return f32 ? reinterpret_cast<float*>(p)[i] : __uint_as_float(static_cast<uint32_t>(reinterpret_cast<uint16_t*>(p)[i]) << 16);
  }
};

float rounded(float v, bool f32) {
  if (f32) return v;
  const uint32_t u = __float_as_uint(v);
  return __uint_as_float((u + 0x7FFFu + (u >> 16 & 1u)) & 0xFFFF0000u);
}

int off(const char* what, int64_t i, double got, double want) {
  std::printf("%s %lld: %g, expected %g\n", what, static_cast<long long>(i), got, want);
  return 1;
}

int run(int64_t n, int64_t vocab, int64_t cols, const std::string& kind, int64_t padding, bool add, bool ids64, bool w32, bool y32,
        int64_t apart, bool at_end) {
  std::mt19937_64 random(static_cast<uint64_t>(n * 31 + vocab * 7 + cols));
  const float scale = 0.5f;
  const int64_t ld = cols + apart, ldw = add ? ld : cols;
  char* ids = between_pages(n * (ids64 ? 8 : 4), at_end, ids64 ? 8 : 4);
  std::vector<int64_t> id(n);
  for (int64_t i = 0; i < n; ++i) {
    const double u = (random() >> 11) * 0x1p-53;
    if (kind == "text") id[i] = padding >= 0 && i >= n - n / 3 ? padding : std::min(vocab - 1, static_cast<int64_t>(u * u * u * u * vocab));
    else if (kind == "same") id[i] = vocab / 2;
    else if (kind == "padding") id[i] = padding;
    else id[i] = std::min(vocab - 1, static_cast<int64_t>(u * vocab));
    if (kind == "outside" && random() % 2) {
      const int64_t wide[] = {-1, vocab, INT64_MIN, INT64_MAX, (int64_t(1) << 32) + 1}, narrow[] = {-1, vocab, INT32_MIN, INT32_MAX, -vocab};
      id[i] = (ids64 ? wide : narrow)[random() % 5];
    }
    if (ids64) reinterpret_cast<int64_t*>(ids)[i] = id[i];
    else reinterpret_cast<int32_t*>(ids)[i] = static_cast<int32_t>(id[i]);
  }
  auto there = [&](int64_t v) { return v >= 0 && v < vocab; };

  {
    Values table((vocab - 1) * ld + cols, w32, at_end), y(n * cols, y32, at_end);
    for (int64_t v = 0; v < vocab; ++v)
      for (int64_t c = 0; c < cols; ++c) table.set(v * ld + c, static_cast<float>(static_cast<int>((v * 5 + c * 3) % 127) - 63));
    if (tm_embed_lookup(y.p, y32, table.p, w32, ld, ids, ids64, n, vocab, cols, scale, nullptr)) return 1;
    for (int64_t i = 0; i < n; ++i)
      for (int64_t c = 0; c < cols; ++c) {
        const float got = y.get(i * cols + c), want = there(id[i]) ? scale * table.get(id[i] * ld + c) : 0.0f;
        if (there(id[i]) ? got != want : got == got) return off("y", i * cols + c, got, want);
      }
  }

  Values dy((n - 1) * ld + cols, y32, at_end), dw((vocab - 1) * ldw + cols, w32, at_end);
  std::vector<float> want(vocab * cols, 0.0f);
  std::vector<char> occurs(vocab, 0);
  int64_t listed = 0;
  for (int64_t i = 0; i < n; ++i) {
    const bool takes_part = there(id[i]) && id[i] != padding;
    listed += takes_part;
    for (int64_t c = 0; c < cols; ++c) {
      const float v = static_cast<float>(static_cast<int>(random() % 7) - 3);
      dy.set(i * ld + c, v);
      if (takes_part) want[id[i] * cols + c] += v;
    }
    if (takes_part) occurs[id[i]] = 1;
  }
  std::vector<char> before(dw.p, dw.p + dw.bytes);
  if (add) {
    for (int64_t v = 0; v < vocab; ++v)
      for (int64_t c = 0; c < cols; ++c) dw.set(v * ldw + c, static_cast<float>((v + c) % 9));
    before.assign(dw.p, dw.p + dw.bytes);
  }
  const size_t need = tm_embed_grad_workspace_bytes(n, vocab, cols);
  char* ws = between_pages(need, at_end, 16);
  if (tm_embed_grad(dw.p, w32, ldw, dy.p, y32, ld, ids, ids64, n, vocab, cols, scale, padding, add, ws, need, nullptr)) return 1;

  // the list: each token that takes part once, by id, in order
  const int32_t total = *reinterpret_cast<int32_t*>(ws), *order = reinterpret_cast<int32_t*>(ws + 16);
  const int32_t* of = order + (4 * n + 15) / 16 * 4;
  if (total != listed) return off("tokens on the list", 0, total, static_cast<double>(listed));
  std::vector<char> seen(n, 0), begun(vocab, 0);
  for (int64_t i = 0; i < total; ++i) {
    if (order[i] < 0 || order[i] >= n || seen[order[i]] || id[order[i]] != of[i] || of[i] == padding) return off("entry", i, order[i], -1);
    seen[order[i]] = 1;
    if (i && of[i] == of[i - 1]) {
      if (order[i] <= order[i - 1]) return off("order of entry", i, order[i], order[i - 1]);
    } else if (begun[of[i]]++) {
      return off("id in two places", i, of[i], -1);
    }
  }
  for (int64_t v = 0; v < vocab; ++v)
    for (int64_t c = 0; c < cols; ++c) {
      const float got = dw.get(v * ldw + c), sum = rounded(want[v * cols + c] * scale + (add ? static_cast<float>((v + c) % 9) : 0.0f), w32);
      if (got != sum) return off("dw", v * ldw + c, got, sum);
    }
  if (add) {  // what lies between rows, and rows that do not occur, as they were
    const size_t size = w32 ? 4 : 2;
    for (int64_t v = 0; v < vocab; ++v) {
      const int64_t first = v * ldw + (occurs[v] ? cols : 0), last = v + 1 < vocab ? (v + 1) * ldw : v * ldw + cols;
      if (last > first && memcmp(dw.p + first * size, before.data() + first * size, (last - first) * size)) return off("row", v, 0, 0);
    }
  }
  return 0;
}

}  // namespace

int main(int argc, char** argv) {
  if (argc != 11) return 2;
  auto number = [&](int i) { return std::atoll(argv[i]); };
  for (bool at_end : {false, true})
    if (int rc = run(number(1), number(2), number(3), argv[4], number(5), number(6), number(7), number(8), number(9), number(10), at_end))
      return rc;
  std::printf("ok\n");
  return 0;
}
