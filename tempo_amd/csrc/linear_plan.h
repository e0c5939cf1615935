// Which kernel of linear.hip runs a product  C[i, j] = sum_k A(i, k) B(j, k)  of I x J x K, and in
// which tiles: host code alone, so that it also builds without a GPU compiler (tests/emul).
#ifndef TEMPO_LINEAR_PLAN_H
#define TEMPO_LINEAR_PLAN_H

#include <stdint.h>

#include <algorithm>

#include "../../include/tempo_unproject.h"

namespace {

using std::min;

// an operand's neighbours in memory: its k, or its own rows
enum { K_ADJACENT = 0, ROW_ADJACENT = 1 };

constexpr int kUnits = 256;  // compute units to fill

// Which kernel runs a product, by sizes and alignment alone.  Measured with the rule and with
// the other side of it, in us:
//   FEW    up to kFewRows rows, both operands with k adjacent (forward), where the columns fill
//          the card and their sums are short: see few_cost.  8 x 4096 x 4096 in bf16 9 against 12
//          (tiles), 64 rows 21 against 16; 64 x 1000 x 1000 6 against 7; 16 x 512 x 4096 9 against
//          6; 32 x 16384 x 4096 48 against 25, in fp32 110 against 78
//   THIN   more than thin_rows rows, up to kThinColumns columns, A with k adjacent, B in LDS.
//          153600 x 16 x 64 in bf16 7 against 10, 614400 x 32 x 256 71 against 74, 65536 rows 10
//          against 8; 153600 x 32 x 256 in fp32 38 against 49, 32768 rows 15 against 14; with B
//          at 78 KB (31 x 500 in fp32) 88 against 96, at 64 KB in 16 bits (15 x 768) 49 against
//          38.  Twice the columns lost: 614400 x 64 x 256 in bf16 91 against 82, in fp32 299
//          against 205
//   STREAM_32x256  both operands aligned, A's rows adjacent, at most 32 of them (the weight's
//          gradient of a thin layer).  153600 x 32 x 256 in fp32 44 against 91, in bf16 75
//          against 71 of which memory takes 74
//   STREAM_256     both aligned, 16 bits, a 256 x 256 tile for every compute unit.  4096 x 4096 x
//          1024 (256 tiles) 40 against 50 with 128 x 128; 4096 x 2048 x 2048 (128) 64 against 46;
//          not where its estimate is more than the smaller tiles': 153600 x 128 x 256 49 against 28
//   STREAM  both aligned;   TILE  anything;  both in tiles of 64 or 128 rows and columns, whichever
//          leave the compute units the least to do: see tile_shape
enum Kernel { FEW, THIN, TILE, STREAM, STREAM_32x256, STREAM_256 };

struct Product {
  Kernel kernel;
  int xi, xj;  // tiles of 64 xi x 64 xj
  uint32_t ti, tj, split;
  long long k_part;
  long long bytes(long long I, long long J) const {
    return split > 1 ? (long long)split * I * J * 4 : 0;
  }
};

constexpr int kFewRows = 64;
constexpr int kThinColumns = 32;

// three workgroups to a compute unit in 16 bits; fp32 is paid back with two as well
uint32_t thin_room(int size) { return size == 4 ? 81920 : 49152; }

long long thin_rows(int size) { return size == 4 ? 32768 : 65536; }

uint32_t thin_lds(long long K, int size) {
  const long long steps = (K * size + 31) / 32;
  const long long bytes = steps * 1024 + 4 * 4096;
  return bytes > thin_room(size) ? 0 : (uint32_t)bytes;
}

// An operand that stream_kernel can take: every 16-byte chunk aligned and not across an end,
// a tile's offsets below 2^31.
bool streamable(const void* p, long long ld, int layout, long long rows, long long K, int size) {
  const int e = 16 / size;
  if (((uintptr_t)p & 15) || ld % e || ld * size > (1 << 22)) return false;
  return layout == K_ADJACENT ? K % e == 0 && K * size <= (1 << 22) && ld >= 0
                              : rows % e == 0 && ld >= rows;
}

// How many parts k is cut into where the tiles alone leave compute units idle: workgroups that
// keep the card busy are one a compute unit where it alone does (256 x 256 tiles, fp32, whose
// products take 16 times as long: 4096 x 1024 x 1024 trained 274 us, 294 with two), else two; a
// part has at least four steps (512 bytes of k).
long long parts_of(long long tiles, long long steps, bool one) {
  const long long split = min((one ? kUnits : 2 * kUnits) / tiles, steps / 4);
  return split < 1 ? 1 : split;
}

// Tiles of 128 x 128 read each operand least often; smaller ones compute less that lies beyond the
// matrix, spread better over the compute units and leave less of k to split.  An estimate in ns
// of each, from what was measured, decides:
//   - 64 x 64 products over 128 bytes of k take a compute unit 150 ns in 16 bits, as they come
//     from L2, which 128 x 64 tiles ask 1.5 times as much for and 64 x 64 twice; in fp32 500 ns,
//     the matrix units' time, and 15 or 30 % more
//   - no less than the operands at memory's rate: each XCD reads its run of tiles for itself
//   - split sums are written and read again and take one more launch
// us in tiles of 128 x 128, 128 x 64, 64 x 128, 64 x 64 (what it picks in brackets):
//   bf16  4096 x 1024 x 1024 33 [19] 19 20        128 x 4096 x 4096      27 21 21 [17]
//         2048 x 2048 x 2048 42 [34] 34 38        5000 x 2000 x 2000     [71] 85 84 103
//         256 x 256 x 153600 [63] 76 77 86        16384 x 192 x 768      26 [13] 15 14
//   fp32  6066 x 1282 x 3076 571 [419] 477 457    1282 x 3076 x 6066     849 693 689 [577]
//         161713 x 33 x 296  131 [70] 144 83      16384 x 192 x 768      58 53 55 [43]
double tile_shape(long long I, long long J, long long K, int size, Product* p) {
  const long long steps = (K * size + 127) / 128;
  const double unit = size == 4 ? 500 : 150;
  double best = 0;
  for (int xi = 2; xi > 0; --xi) {
    for (int xj = 2; xj > 0; --xj) {
      const long long ti = (I + 64 * xi - 1) / (64 * xi), tj = (J + 64 * xj - 1) / (64 * xj);
      const long long parts = parts_of(ti * tj, steps, size == 4);
      const double more = 4 - xi - xj, area = xi * xj;
      const double rounds = (double)((ti * tj * parts + kUnits - 1) / kUnits);
      const double work = rounds * ((steps + parts - 1) / parts) * area * unit *
                          (size == 4 ? 1 + .15 * more : 1 + .5 * more);
      const long long run = (ti * tj + 7) / 8, high = min(min(run, ti), 8ll);
      const long long across = min(tj, (run + high - 1) / high), down = (run + across - 1) / across;
      const double read =
          (double)min(ti * tj, 8ll) * 64 * (down * xi + across * xj) * K * size / 4800;
      const double join = parts > 1 ? 5000 + (double)parts * I * J * 8 / 4800 : 0;
      const double cost = (work > read ? work : read) + join;
      if (xi + xj == 4 || cost < best) best = cost, p->xi = xi, p->xj = xj;
    }
  }
  return best;
}

// few_kernel's time by the same measure: 16 columns a compute unit, a step's loads and products
// one behind the other
double few_cost(long long I, long long J, long long K, int size) {
  const int blocks = I <= 16 ? 1 : I <= 32 ? 2 : 4;
  const double rounds = (double)((J + 16 * kUnits - 1) / (16 * kUnits));
  return rounds * ((K * size + 127) / 128) * (60 + (size == 4 ? 83 : 62) * blocks);
}

bool plan_product(long long I, long long J, long long K, int al, int bl, int dtype, bool direct,
                  Product* p) {
  const int size = dtype == TEMPO_DTYPE_F32 ? 4 : 2;
  p->split = 1;
  p->k_part = K;
  const double cost = tile_shape(I, J, K, size, p);
  if (al == K_ADJACENT && bl == K_ADJACENT && I <= kFewRows && few_cost(I, J, K, size) <= cost) {
    p->kernel = FEW;
    return true;
  }
  if (al == K_ADJACENT && J <= kThinColumns && I > thin_rows(size) && thin_lds(K, size)) {
    p->kernel = THIN;
    return true;
  }
  const long long depth = 128 / size;
  const long long steps = (K + depth - 1) / depth;
  p->kernel = direct ? STREAM : TILE;
  long long high = 64 * p->xi, wide = 64 * p->xj;
  if (direct && al == ROW_ADJACENT && I <= 32) {
    p->kernel = STREAM_32x256;
    high = 32, wide = 256;
  } else if (direct && size == 2) {
    const long long tiles = (I + 255) / 256 * ((J + 255) / 256);
    if (tiles >= kUnits && (tiles + kUnits - 1) / kUnits * (double)steps * 16 * 120 <= cost) {
      p->kernel = STREAM_256;
      high = wide = 256;
    }
  }
  const long long ti = (I + high - 1) / high, tj = (J + wide - 1) / wide;
  if (ti > 0xffffff / tj) return false;  // a grid's threads are counted in 32 bits
  p->ti = (uint32_t)ti;
  p->tj = (uint32_t)tj;
  const long long split = parts_of(ti * tj, steps, p->kernel == STREAM_256 || size == 4);
  const long long part = (steps + split - 1) / split;
  p->k_part = part * depth;
  p->split = (uint32_t)((steps + part - 1) / part);
  return p->split <= 65535;
}

// Scratch memory is planned from sizes alone: either kernel may run in the end.
bool product_bytes(long long I, long long J, long long K, int al, int bl, int dtype,
                   long long* bytes) {
  Product a, b;
  if (!plan_product(I, J, K, al, bl, dtype, false, &a) ||
      !plan_product(I, J, K, al, bl, dtype, true, &b))
    return false;
  const long long x = a.bytes(I, J), y = b.bytes(I, J);
  *bytes = x > y ? x : y;
  return true;
}

}  // namespace

#endif
