// mx_product.hip -- which kernel an MXFP4 product takes.
//
// Four are there: the stream (16 rows a wave, weights through LDS from memory's lines), and
// tiles of 32 x 128, 128 x 128 and 256 x 256.  The rule is on the rows that an expert has on
// average and on how many tiles the call has for 256 CUs; the figures are us on both
// sides of each border, one expert unless said (rows x N x K, or rows of each of E experts on average, four drawn for
// each token with equal chances, at N = 5760, K = 2880 with SwiGLU and MXFP4 results).  How uneven the experts' rows are
// is known on the device only, and the average misleads where few of many have them: 512 rows in 8 of 128 experts
// take the stream 64 us, where 32 x 128 would take 30 and 128 x 128 27; in 32 of them 71, 73 and 78.  With exactly 32
// rows each of 128, 128 x 128 takes 306 and 32 x 128 277.
#include "mx_kernels.h"

namespace gxmoe {

hipError_t launch_mx_product(const MxProductArgs& a, hipStream_t s) {
  const int64_t each = a.rows / (a.offsets ? a.E : 1);  // rows of an expert on average
  const auto tiles = [&](int rows, int cols) { return most_m_tiles(a, rows) * ((static_cast<int64_t>(a.N) + cols - 1) / cols); };

  // The stream holds the whole of the weights' bandwidth with few rows, and with few tiles its short chain counts:
  //                  stream    32 x 128                          stream    32 x 128
  //   1 x 5120 x 2880   7.4      14.5        2 each of 128       164       207
  //   32 x 5120 x 2880  8.5      15.0        4 each of 128       210       238
  //   64 x 2880 x 4096 11.3      16.2        8 each of 128       244       251
  //   96 x 5120 x 2880 16.6      14.0        4 each of 32         56        62
  //   32 x 32768 x 4096  42      19.9        8 each of 32         66        62
  const int64_t waves = tiles(kStreamRows, 16);
  if (a.K >= 512 && (each <= 4 || waves <= 4 * kMxCus)) {
    // Waves of 32 columns read a's rows half as often, and are half as many: 2 each of 128 at N = 2880 take 87 (16 columns:
    // 96), 1 x 5120 x 2880 8.4 (7.5).  Four waves share a long K while there are CUs for it: 1 x 2048 x 8192 7.3
    // (one wave 11.9), 1 x 8192 x 8192 11.7 (14.2); 1 x 10240 x 4096 10.9 (9.5), 32 x 2880 x 4096 11.9 (9.1).  Below
    // K = 4096 it gains nothing: 1 x 5120 x 2880 7.6 (7.3).
    return launch_mx_stream(a, a.quantized() || waves > 64 * kMxCus,
                            a.K >= 4096 && a.rows <= kStreamRows && waves <= 2 * kMxCus, s);
  }
  //                        32 x 128  128 x 128                        32 x 128  128 x 128
  //   256 x 5120 x 2880      18.4      17.6        16 each of 128       266       296
  //   512 x 5120 x 2880      24.3      17.6        32 each of 128       349       310
  //   777 x 1001 x 2016      10.6      13.6        32 each of 32         89        72
  if (each <= 24 || tiles(32, 128) < 2 * kMxCus) return launch_mx_tile(a, MxTile::low, s);
  //                       128 x 128 256 x 256                       128 x 128 256 x 256
  //   1500 x 5120 x 2880     26.9      33.1        96 each of 32         94        92
  //   2048 x 5120 x 2880     40.6      32.0        128 each of 32       132       105
  if (each <= 96 || tiles(128, 128) <= 2 * kMxCus) return launch_mx_tile(a, MxTile::middle, s);
  return launch_mx_tile(a, MxTile::large, s);
}

}  // namespace gxmoe
