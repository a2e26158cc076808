// Tiles of ones times ones whose sums wait for k-blocks that nobody loads, when told so: the waits run out, which is their bound of two seconds
// and no fault. For tests/test_lm_sync_gpu.py.
#include "../../tbb_test_b200/csrc/lm_tile.cuh"
#include "../../tbb_test_b200/csrc/wait_reports.h"

namespace b2 {
namespace {

struct LateParams {
  int late;
  float* out;  // 256 x 256
};
template <bool SPLIT, bool ONE>
struct LateOp {
  typedef LateParams Params;
  typedef TileForm<SPLIT, ONE> Form;
  static constexpr bool STORES = false, LONG = SPLIT, INFINITE = false;
  static constexpr int SUM = 4, W = Form::CHUNK, COLS = 256 / Form::BN;
  const Params& p;
  __device__ explicit LateOp(const Params& q, const TileMaps&) : p(q) {}
  __device__ int tiles() const { return 256 / Form::M * COLS; }
  __device__ Tile tile(int t) const {
    Tile r{};
    r.m0 = r.a_mn = t / COLS * Form::M;
    r.n0 = r.b_mn = t % COLS * Form::BN;
    r.kblocks = p.late && threadIdx.x < 32 ? 1 : 2;  // the loading warp's list is one k-block short
    return r;
  }
  __device__ void begin(const Tile&, int, int, int) {}
  __device__ void chunk(const Tile&, int row0, int col0, float (&v)[W], uint8_t*, int lane) {
    for (int j = 0; j < W; ++j) p.out[(row0 + lane) * 256 + col0 + j] = v[j];
  }
  __device__ void end(const Tile&, int, int) {}
};

}  // namespace
}  // namespace b2

using namespace b2;

extern "C" {

// ones, zeros: 256 x 128 of fp16. form: 0 pairs, 1 single CTAs; + 2: operands in halves, ones + zeros.
int late_launch(int form, int late, const void* ones, const void* zeros, float* out, void* stream) {
  int sms, rc = lm_device(&sms);
  if (rc != B2_OK) return rc;
  const TileOperand x{ones, zeros, 256, 128, 128, false};
  Chain chain(static_cast<cudaStream_t>(stream));
  auto launch = form == 0   ? tile_launch<LateOp<false, false>>
                : form == 1 ? tile_launch<LateOp<false, true>>
                : form == 2 ? tile_launch<LateOp<true, false>>
                            : tile_launch<LateOp<true, true>>;
  return launch("late_launch", x, x, nullptr, LateParams{late, out}, false, 8, sms, chain);
}

// CTAs that have given up so far, and whether that is news to the stream.
int late_report(void* stream, unsigned int* count, int* news) {
  static WaitReports reports;
  TileReport r{};
  unsigned long long id = 0;
  cudaError_t e = tile_report_read(&r, static_cast<cudaStream_t>(stream));
  if (e == cudaSuccess) e = cudaStreamGetId(static_cast<cudaStream_t>(stream), &id);
  if (e != cudaSuccess) return launch_error(e, "late_report");
  *count = r.count;
  *news = reports.news(0, id, r.count);
  return B2_OK;
}
}
