// The shape of a product straight from memory (direct_product.h). Without kernels: a host test includes it.
#pragma once

#include <cstdint>

struct DpForm {
  int mt, wk;  // rows of a wave in sixteens; waves that share K (1: each has columns of its own)
};

// Rows of a wave: those there are, up to 64, where the weights are much to read; otherwise as many as leave the card waves to run (a
// wave's work is then latency and code that runs once: the four products of 135 rows of 64 x 128, float32, forward and VJP for x, 10.9,
// 8.7, 10.4 and 6.8 us with 64 rows a wave, 5.7, 5.5, 6.7 and 5.2 with 16). K shared by eight or sixteen waves where the tiles are too few
// to fill the card with waves of their own. `unit`: of K, what one matrix instruction takes.
inline DpForm dp_form(int64_t rows_n, int64_t rows_m, int64_t k, int parts, int unit) {
  const int64_t columns = (rows_n + 15) / 16, units = parts * ((k + unit - 1) / unit);
  const auto waves = [&](int mt) { return columns * ((rows_m + 16 * mt - 1) / (16 * mt)); };
  const bool much = rows_n * k * parts >= 1 << 20;
  int mt = 1;
  if (rows_m > 32 && (much || waves(4) >= 1024))
    mt = 4;
  else if (rows_m > 16 && (much || waves(2) >= 1024))
    mt = 2;
  if (mt == 1 && waves(1) <= 192 && units >= 64) return {1, 16};
  return {mt, waves(mt) < 1024 && units >= 8 ? 8 : 1};
}
