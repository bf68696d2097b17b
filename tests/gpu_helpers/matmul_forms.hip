// Test helper (not part of libftmoe.so): one form of the matrix products, named by
// its number, at sizes where the library would take another.  Forms 0 to 2 are the
// streaming shapes, 3 to 7 the tiles (kTile128x64, kTile256x128, kTile256x256), the first two
// without and with the weights read past the caches.  The caller has checked what
// the library's entry points check.
#include "matmul_stream.hip"
#include "matmul_tile.hip"

struct FormArgs {
  const void* x;
  const float* xs;
  const void* w;
  const float* ws;
  const int32_t* offsets;
  const int32_t* order;
  const int32_t* ids;
  const float* row_weight;
  const void* extra_w;
  const float* extra_ws;
  void* y;
  int int8, E, N, K, rows, x_rows, top_k, act, extra, extra_x, quantise, out_f32;
  float limit, extra_limit;
};

extern "C" int ftmoe_test_matmul_form(const FormArgs* f, int form, hipStream_t stream) {
  ftmoe::MatmulArgs a{};
  a.int8 = f->int8;
  a.x = static_cast<const uint8_t*>(f->x);
  a.xs = f->xs;
  a.w = static_cast<const uint8_t*>(f->w);
  a.ws = f->ws;
  a.E = f->E;
  a.N = f->N;
  a.K = f->K;
  a.rows = f->rows;
  a.x_rows = f->x_rows;
  a.offsets = f->offsets;
  a.order = f->order;
  a.ids = f->ids;
  a.top_k = f->top_k;
  a.row_weight = f->row_weight;
  a.act = f->act;
  a.limit = f->limit;
  a.extra = f->extra;
  a.extra_x = f->extra_x;
  a.extra_w = static_cast<const uint8_t*>(f->extra_w);
  a.extra_ws = f->extra_ws;
  a.extra_limit = f->extra_limit;
  a.quantise = f->quantise;
  a.out_f32 = f->out_f32;
  a.y = f->y;
  if (form < 0 || form > 7) return -1;
  const hipError_t err = form < 3 ? ftmoe::launch_matmul_stream(a, static_cast<ftmoe::StreamShape>(form), stream)
                                  : ftmoe::launch_matmul_tile(a, static_cast<ftmoe::TileShape>((form - 3) / 2),
                                                              (form - 3) % 2 != 0, stream);
  return static_cast<int>(err);
}
