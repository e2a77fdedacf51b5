// The host's bound on one request's places on the attention kernels' line against the
// line itself, over the shapes a call may have.  Runs on the CPU.
#include <cstdio>
#include <random>

#include "kv_attention.cuh"

using namespace qg;

static long long bad = 0, tried = 0;

template <int RG, int TL>
static void check(const KvAttnArgs& a, int n, int n_all, int len) {
  KvRequest q;
  q.start = 0; q.n = n; q.n_all = n_all; q.len = len;
  const KvLine<RG, TL> line(a, q);
  // upto() in 64 bits
  const long long g = line.groups, places =
      (((g * line.h0 + (long long)line.slope * (g * (g + 1) / 2)) >> TL) + g * KvLine<RG, TL>::kStart) * a.heads;
  const long long most = kv_line_most(a, RG, TL);
  ++tried;
  if (places > most && most <= INT32_MAX && ++bad < 6)  // past 2^31 the call is refused
    std::printf("group %d heads %d n %d of %d, %d of %lld tokens, window %d causal %d, rows of %d: %lld places, bound %lld\n",
                a.group, a.heads, n, n_all, len, (long long)a.width << a.block_log2, a.window, a.causal, RG, places, most);
}

int main() {
  std::mt19937 rng(5);
  auto up_to = [&](long long most) {  // evenly over the logarithm
    const int bits = (int)(rng() % 31) + 1;
    const long long v = 1 + (long long)(rng() % (1u << bits));
    return (int)(v < most ? v : most);
  };
  for (int i = 0; i < 2000000; ++i) {
    KvAttnArgs a = {};
    a.block_log2 = 4 + (int)(rng() % 4);
    a.width = up_to(INT32_MAX >> a.block_log2);
    a.heads = up_to(64);
    a.group = up_to(i % 2 ? 64 : 8192);
    a.max_new = up_to((INT32_MAX - 256) / a.group);
    a.rows_max = i % 3 ? INT32_MAX : i % 2 ? 48 : 32;
    a.causal = (int)(rng() % 4) != 0;
    a.window = rng() % 3 ? 0 : up_to(INT32_MAX);
    const long long rows = (long long)a.max_new * a.group < a.rows_max ? (long long)a.max_new * a.group : a.rows_max;
    const int most_n = (int)(rows / a.group);
    if (most_n < 1) continue;
    const int n = rng() % 2 ? most_n : up_to(most_n);
    const int n_all = n < a.max_new ? n : n + (rng() % 2 ? up_to(1000) : 0);
    const long long room = (long long)a.width << a.block_log2;
    const int len = rng() % 2 ? (int)room : up_to(room);
    check<256, 7>(a, n, n_all, len);
    check<8, 4>(a, n, n_all, len);
    check<16, 4>(a, n, n_all, len);
  }
  std::printf("%lld lines, %lld past the bound\n", tried, bad);
  return bad != 0;
}
