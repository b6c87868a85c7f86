// Layers of block-scaled 8-bit products, one call each way: the casts and products of a linear layer and of a
// gated feed-forward block on two pieces of storage that the caller provides, one that the backward reads
// (`saved`) and one that lasts for the call (`tmp`). Their launches are programmatic dependent ones from the
// second on.
//
// A call from Python per launch (ten for a training step of the feed-forward block, each with its tensors to
// allocate) took 10-15 us apiece, more than the kernels below a few thousand tokens.
#include <cuda_bf16.h>

#include "../common/pdl.h"
#include "block_gemm.h"
#include "block_scale.cuh"

namespace lb {
namespace {

// Pieces of a caller's storage, each on its own 256 bytes; with no base only their sizes are added up.
struct Arena {
  uint8_t* base;
  size_t at = 0;
  explicit Arena(void* p) : base(static_cast<uint8_t*>(p)) {}
  void* take(size_t bytes) {
    uint8_t* p = base != nullptr ? base + at : nullptr;
    at += (bytes + 255) / 256 * 256;
    return p;
  }
  BlockMat mat(long long rows, long long cols) {
    const long long ld = (cols + 15) / 16 * 16;
    BlockMat m{static_cast<uint8_t*>(take(size_t(rows * ld))), ld, nullptr, rows, 0};
    m.scales = static_cast<uint32_t*>(take(size_t((cols + 511) / 512 * rows * 4)));
    return m;
  }
};

BlockMat rows_of(const BlockMat& m, long long first) {
  BlockMat r = m;
  r.data += first * m.ld;
  r.scales += first;
  return r;
}

// Where a result goes: 0 = bf16, 1 = fp32, 2 = added to fp32.
struct Out {
  void* p;
  int mode;
};

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

struct Call {
  int* status;
  cudaStream_t stream;
  void* ws;   // of the largest product of the call
  int rc = 0;
  bool first = true;
  template <typename F>
  void run(F&& f) {
    if (rc) return;
    PdlScope scope(!first);
    rc = f();
    first = false;
  }
  void product(const BlockMat& a, const BlockMat& b, const Out& out, int M, int N, int K, long long ldc,
               const void* bias = nullptr, int deepest = 0) {
    run([&] {
      const BlockPlan p = block_plan(M, N, K, aligned16(out.p) && !(N & 7) && !(ldc & 7), deepest);
      return block_gemm(p, a, b, out.p, M, N, K, ldc, out.mode > 0, out.mode == 2, bias, ws, status, stream);
    });
  }
};

// Storage of a product whatever the alignment of its output.
size_t product_bytes(int M, int N, int K, int deepest = 0) {
  return block_plan_bytes(block_plan(M, N, K, !(N & 7), deepest), M, N);
}
size_t max2(size_t a, size_t b) { return a > b ? a : b; }

struct LinearStorage {
  BlockMat x, w, x_t, w_t, dy, dy_t;
  float* colsum;
  void *ws_fwd, *ws_bwd;
  size_t saved, fwd, bwd;
};

LinearStorage linear_storage(int T, int K, int N, int need, void* saved, void* tmp) {
  LinearStorage s{};
  const bool need_x = need & 1, need_w = need & 2, need_b = need & 4;
  Arena keep(saved), fwd(tmp), bwd(tmp);
  if (need_w) s.x_t = keep.mat(K, T);
  if (need_x) s.w_t = keep.mat(K, N);
  s.x = fwd.mat(T, K);
  s.w = fwd.mat(N, K);
  s.ws_fwd = fwd.take(product_bytes(T, N, K));
  if (need_x) s.dy = bwd.mat(T, N);
  if (need_w) s.dy_t = bwd.mat(N, T);
  if (need_b) s.colsum = static_cast<float*>(bwd.take(size_t((T + 127) / 128) * N * 4));
  s.ws_bwd = bwd.take(max2(need_x ? product_bytes(T, K, N) : 0, need_w ? product_bytes(N, K, T) : 0));
  s.saved = keep.at;
  s.fwd = fwd.at;
  s.bwd = bwd.at;
  return s;
}

struct MlpStorage {
  __nv_bfloat16 *gu, *dh;
  BlockMat x, w, wd, h, x_t, w_t, wd_t, dy, dy_t, d, d_t, h_t;
  void *ws_fwd, *ws_bwd;
  size_t saved, fwd, bwd;
};

// need: 1 = x, 2 = gate or up weight, 4 = down weight
MlpStorage mlp_storage(int T, int H, int I, int need, void* saved, void* tmp) {
  MlpStorage s{};
  const bool need_x = need & 1, need_gu = need & 2, need_d = need & 4;
  Arena keep(saved), fwd(tmp), bwd(tmp);
  s.gu = static_cast<__nv_bfloat16*>(keep.take(size_t(T) * 2 * I * 2));
  if (need_gu) s.x_t = keep.mat(H, T);
  if (need_x) s.w_t = keep.mat(H, 2LL * I);
  if (need_x || need_gu) s.wd_t = keep.mat(I, H);
  s.x = fwd.mat(T, H);
  s.w = fwd.mat(2LL * I, H);
  s.wd = fwd.mat(H, I);
  s.h = fwd.mat(T, I);
  s.ws_fwd = fwd.take(max2(product_bytes(T, 2 * I, H, kDeepestSum), product_bytes(T, H, I)));
  if (need_x || need_gu) {
    s.dy = bwd.mat(T, H);
    s.dh = static_cast<__nv_bfloat16*>(bwd.take(size_t(T) * I * 2));
  }
  if (need_d) s.dy_t = bwd.mat(H, T);
  if (need_x) s.d = bwd.mat(T, 2LL * I);
  if (need_gu) s.d_t = bwd.mat(2LL * I, T);
  if (need_d) s.h_t = bwd.mat(I, T);
  size_t ws = 0;
  if (need_x || need_gu) ws = max2(ws, product_bytes(T, I, H, kDeepestSum));
  if (need_x) ws = max2(ws, product_bytes(T, H, 2 * I));
  if (need_gu) ws = max2(ws, max2(product_bytes(2 * I, H, T), product_bytes(I, H, T)));
  if (need_d) ws = max2(ws, product_bytes(H, I, T));
  s.ws_bwd = bwd.take(ws);
  s.saved = keep.at;
  s.fwd = fwd.at;
  s.bwd = bwd.at;
  return s;
}

// y = (act(x Wgᵀ) * (x Wuᵀ)) Wdᵀ from cast operands. The two products stay in s.gu for the backward, are dropped, or
// are there already. What the backward reads is summed in parts (kDeepestSum); an encoder's gate and up products
// go through h into one row of y alone, where a step of one value is lost among those of the row's others.
enum GateUp { kKeepProducts, kDropProducts, kHaveProducts };
void mlp_products(Call& c, int kind, const MlpStorage& s, int T, int H, int I, GateUp gu, void* y) {
  const bool keep = gu == kKeepProducts;
  const int deepest = keep ? kDeepestSum : 0;
  if (gu != kHaveProducts && block_glu_fused(T, I, H, deepest)) {
    c.run([&] {
      return block_gemm_glu(kind, deepest, s.x, s.w, rows_of(s.w, I), T, I, H, keep ? s.gu : nullptr,
                            keep ? s.gu + I : nullptr, 2LL * I, s.h, c.status, c.stream);
    });
  } else {
    if (gu != kHaveProducts) c.product(s.x, s.w, Out{s.gu, 0}, T, 2 * I, H, 2LL * I, nullptr, deepest);
    c.run([&] { return block_glu_fwd(kind, s.gu, s.gu + I, 2LL * I, T, I, s.h, c.stream); });
  }
  c.product(s.h, s.wd, Out{y, 0}, T, H, I, H);
}

}  // namespace
}  // namespace lb

using namespace lb;

// Bytes that the calls below want: out = {saved, tmp of the forward, tmp of the backward}. need: gradients of 1 = x,
// 2 = weight, 4 = bias. Modes of outputs throughout: 0 = bf16, 1 = fp32, 2 = added to fp32.
extern "C" int lb_linear_block_bytes(int T, int K, int N, int need, long long* out) {
  const LinearStorage s = linear_storage(T, K, N, need, nullptr, nullptr);
  out[0] = (long long)s.saved;
  out[1] = (long long)s.fwd;
  out[2] = (long long)s.bwd;
  return 0;
}

// y [T, N] = x [T, K] · wᵀ + bias from bf16 x and w (rows ldx / ldw elements apart), T, K, N > 0.
extern "C" int lb_linear_block_fwd(const void* x, long long ldx, const void* w, long long ldw, const void* bias,
                                   int T, int K, int N, int need, int y_mode, void* y, void* saved, void* tmp,
                                   int* status, void* stream_) {
  if (T <= 0 || K <= 0 || N <= 0) return -3;
  const LinearStorage s = linear_storage(T, K, N, need, saved, tmp);
  Call c{status, reinterpret_cast<cudaStream_t>(stream_), s.ws_fwd};
  const BlockCast casts[2] = {{x, T, K, ldx, 0, s.x, s.x_t, 0, true}, {w, N, K, ldw, 1, s.w, s.w_t, 0, true}};
  c.run([&] { return block_casts(casts, 2, c.stream); });
  c.product(s.x, s.w, Out{y, y_mode}, T, N, K, N, bias);
  return c.rc;
}

// The same with a weight in 8 bits (bytes, rows ldw apart; scale words, rows_w a group). tmp: lb_linear_kept_bytes.
extern "C" long long lb_linear_kept_bytes(int T, int K, int N) {
  if (block_casts_itself(block_plan(T, N, K, !(N & 7)), T, K)) return 0;
  Arena a(nullptr);
  a.mat(T, K);
  a.take(product_bytes(T, N, K));
  return (long long)a.at;
}
extern "C" int lb_linear_kept_fwd(const void* x, long long ldx, const void* w, long long ldw, const void* scales,
                                  long long rows_w, int w_e5m2, const void* bias, int T, int K, int N, int y_mode,
                                  void* y, void* tmp, int* status, void* stream_) {
  if (T <= 0 || K <= 0 || N <= 0) return -3;
  const BlockMat wq{(uint8_t*)w, ldw, (uint32_t*)scales, rows_w, w_e5m2};
  Call c{status, reinterpret_cast<cudaStream_t>(stream_), nullptr};
  const BlockPlan p = block_plan(T, N, K, !(N & 7));
  if (block_casts_itself(p, T, K)) {
    c.run([&] {
      return block_gemm_cast(p, x, ldx, wq, y, T, N, K, N, y_mode, bias, status, c.stream);
    });
    return c.rc;
  }
  Arena a(tmp);
  const BlockMat xq = a.mat(T, K);
  c.ws = a.take(0);
  c.run([&] { return block_cast(x, T, K, ldx, 0, 0, xq, BlockMat{}, 0, nullptr, c.stream); });
  c.product(xq, wq, Out{y, y_mode}, T, N, K, N, bias);
  return c.rc;
}

// dx [T, K] = dy · w, dw [N, K] = or += dyᵀ · x, db [N] = column sums of dy (rows lddy elements apart), of those
// that `need` names, from what the forward saved. dx_mode, db_mode: 0 or 1. dy32 (rows lddy32 elements apart; null:
// none): dy before it was rounded to bf16, which db then is the sum of.
extern "C" int lb_linear_block_bwd(const void* dy, long long lddy, const float* dy32, long long lddy32, int T, int K, int N, int need, void* saved,
                                   void* tmp, void* dx, int dx_mode, void* dw, int dw_mode, void* db, int db_mode,
                                   int* status, void* stream_) {
  if (T <= 0 || K <= 0 || N <= 0) return -3;
  const LinearStorage s = linear_storage(T, K, N, need, saved, tmp);
  Call c{status, reinterpret_cast<cudaStream_t>(stream_), s.ws_bwd};
  const bool apart = dy32 != nullptr && (need & 4);
  c.run([&] { return block_cast(dy, T, N, lddy, 0, 0, s.dy, s.dy_t, 0, apart ? nullptr : s.colsum, c.stream); });
  if (apart) c.run([&] { return block_colsum(dy32, T, N, lddy32, s.colsum, c.stream); });
  if (need & 1) c.product(s.dy, s.w_t, Out{dx, dx_mode}, T, K, N, K);
  if (need & 2) c.product(s.dy_t, s.x_t, Out{dw, dw_mode}, N, K, T, K);
  if (need & 4)
    c.run([&] { return block_sum(s.colsum, (T + 127) / 128, N, 1, N, db, N, db_mode, 0, nullptr, c.stream); });
  return c.rc;
}

// The gated block. need: gradients of 1 = x, 2 = the gate or up weight, 4 = the down weight; modes: of the gate (or
// fused), up and down weights' gradients.
extern "C" int lb_mlp_block_bytes(int T, int H, int I, int need, long long* out) {
  const MlpStorage s = mlp_storage(T, H, I, need, nullptr, nullptr);
  out[0] = (long long)s.saved;
  out[1] = (long long)s.fwd;
  out[2] = (long long)s.bwd;
  return 0;
}

// y [T, H] from bf16 x [T, H], gate and up weights [I, H] (wu null: wg is [2 I, H]) and down weight [H, I].
extern "C" int lb_mlp_block_fwd(int kind, const void* x, long long ldx, const void* wg, long long ldg, const void* wu,
                                long long ldu, const void* wd, long long ldd, int T, int H, int I, int need, void* y,
                                void* saved, void* tmp, int* status, void* stream_) {
  if (T <= 0 || H <= 0 || I <= 0 || (I % kScaleBlock)) return -3;
  const MlpStorage s = mlp_storage(T, H, I, need, saved, tmp);
  Call c{status, reinterpret_cast<cudaStream_t>(stream_), s.ws_fwd};
  BlockCast casts[4] = {{x, T, H, ldx, 0, s.x, s.x_t, 0, true}, {wd, H, I, ldd, 1, s.wd, s.wd_t, 0, true}};
  if (wu == nullptr) {
    casts[2] = BlockCast{wg, 2 * I, H, ldg, 1, s.w, s.w_t, 0, true};
  } else {
    BlockMat t = s.w_t;
    if (t.data != nullptr) t.data += I;   // columns I on: blocks I / 128 on
    casts[2] = BlockCast{wg, I, H, ldg, 1, s.w, s.w_t, 0, false};
    casts[3] = BlockCast{wu, I, H, ldu, 1, rows_of(s.w, I), t, I / kScaleBlock, true};
  }
  c.run([&] { return block_casts(casts, wu == nullptr ? 3 : 4, c.stream); });
  mlp_products(c, kind, s, T, H, I, kKeepProducts, y);
  return c.rc;
}

// The same with weights in 8 bits, gate and up fused. tmp: lb_mlp_kept_bytes.
namespace {
// Whether the gate and up product casts x itself.
bool mlp_casts_itself(int T, int H, int I, const BlockPlan& p) {
  return !block_glu_fused(T, I, H, 0) && block_casts_itself(p, T, H);
}
MlpStorage mlp_kept_storage(int T, int H, int I, bool cast_x, void* tmp) {
  MlpStorage s{};
  Arena a(tmp);
  if (!cast_x) s.x = a.mat(T, H);
  s.h = a.mat(T, I);
  if (!block_glu_fused(T, I, H, 0)) s.gu = static_cast<__nv_bfloat16*>(a.take(size_t(T) * 2 * I * 2));
  s.ws_fwd = a.take(max2(product_bytes(T, 2 * I, H), product_bytes(T, H, I)));
  s.fwd = a.at;
  return s;
}
}  // namespace
extern "C" long long lb_mlp_kept_bytes(int T, int H, int I) {
  const bool cast_x = mlp_casts_itself(T, H, I, block_plan(T, 2 * I, H, true));
  return (long long)mlp_kept_storage(T, H, I, cast_x, nullptr).fwd;
}
extern "C" int lb_mlp_kept_fwd(int kind, const void* x, long long ldx, const void* w, long long ldw, const void* ws,
                               long long rows_w, int w_e5m2, const void* wd, long long ldd, const void* wds,
                               long long rows_d, int wd_e5m2, int T, int H, int I, void* y, void* tmp, int* status,
                               void* stream_) {
  if (T <= 0 || H <= 0 || I <= 0 || (I % kScaleBlock)) return -3;
  const BlockPlan p = block_plan(T, 2 * I, H, true);
  const bool cast_x = mlp_casts_itself(T, H, I, p);
  MlpStorage s = mlp_kept_storage(T, H, I, cast_x, tmp);
  s.w = BlockMat{(uint8_t*)w, ldw, (uint32_t*)ws, rows_w, w_e5m2};
  s.wd = BlockMat{(uint8_t*)wd, ldd, (uint32_t*)wds, rows_d, wd_e5m2};
  Call c{status, reinterpret_cast<cudaStream_t>(stream_), s.ws_fwd};
  if (cast_x)
    c.run([&] { return block_gemm_cast(p, x, ldx, s.w, s.gu, T, 2 * I, H, 2LL * I, 0, nullptr, status, c.stream); });
  else
    c.run([&] { return block_cast(x, T, H, ldx, 0, 0, s.x, BlockMat{}, 0, nullptr, c.stream); });
  mlp_products(c, kind, s, T, H, I, cast_x ? kHaveProducts : kDropProducts, y);
  return c.rc;
}

// Gradients from dy [T, H]: dx [T, H] (bf16), dwg [I, H] and dwu (fused: dwg is [2 I, H] and dwu null), dwd [H, I]; those
// that `need` names, of a gate and up weight apart those that are not null.
extern "C" int lb_mlp_block_bwd(int kind, const void* dy, long long lddy, int T, int H, int I, int need, int fused,
                                void* saved, void* tmp, void* dx, void* dwg, void* dwu, void* dwd, const int* modes,
                                int* status, void* stream_) {
  if (T <= 0 || H <= 0 || I <= 0 || (I % kScaleBlock)) return -3;
  const MlpStorage s = mlp_storage(T, H, I, need, saved, tmp);
  Call c{status, reinterpret_cast<cudaStream_t>(stream_), s.ws_bwd};
  c.run([&] { return block_cast(dy, T, H, lddy, 0, 0, s.dy, s.dy_t, 0, nullptr, c.stream); });
  const bool inner = need & 3;
  if (inner) c.product(s.dy, s.wd_t, Out{s.dh, 0}, T, I, H, I, nullptr, kDeepestSum);
  c.run([&] {
    // (for h alone the gradient is not used; anything of its size will do)
    return block_glu_bwd(kind, inner ? s.dh : s.gu, inner ? I : 2LL * I, s.gu, s.gu + I, 2LL * I, T, I, s.d, s.d_t,
                         s.h_t, c.stream);
  });
  if (need & 1) c.product(s.d, s.w_t, Out{dx, 0}, T, H, 2 * I, H);
  if (need & 2) {
    if (fused) {
      c.product(s.d_t, s.x_t, Out{dwg, modes[0]}, 2 * I, H, T, H);
    } else {
      if (dwg != nullptr) c.product(s.d_t, s.x_t, Out{dwg, modes[0]}, I, H, T, H);
      if (dwu != nullptr) c.product(rows_of(s.d_t, I), s.x_t, Out{dwu, modes[1]}, I, H, T, H);
    }
  }
  if (need & 4) c.product(s.dy_t, s.h_t, Out{dwd, modes[2]}, H, I, T, I);
  return c.rc;
}
