// Arguments of the layer-norm, dropout and gated feed-forward entry points, one struct per call: what autograd.cpp fills in
// and layer_norm.cu, dropout.cu and gated_ffn.cu take.  Types: 0 fp32, 1 bf16, 2 fp16.  stream / st: cudaStream_t.
// A return code other than 0 is a cudaError_t or, below 0, a refusal.  launches (out): kernels that the call has launched.
#pragma once

// y = layer_norm(x) w + b; stats: mean [n] and 1 / sqrt(var + eps) [n], or null (evaluation)
struct LnForwardCall {
  const void* x;
  long long ldx;
  const void *w, *b;
  void* y;
  float* stats;
  long long n, d, dt, w_dt;
  double eps;
  void* stream;
  long long launches;
};

// dx (may be null) and dw, db (may be null; partial: layer_norm_partial_floats(d) floats of scratch, or null without both)
struct LnBackwardCall {
  const void* x;
  long long ldx;
  const void* dy;
  long long lddy;
  const void* w;
  float* stats;
  void *dx, *dw, *db;
  float* partial;
  long long n, d, dt, w_dt;
  void* stream;
  long long launches;
};

// y[i] = res[i] + keep(i) x[i] 65536 / (65536 - drop), i < n; res may be null; key: 8 bytes on the device; drop = 0 .. 65536 (nothing is kept)
struct DropoutCall {
  const void *x, *res;
  void* y;
  long long n;
  const void* key;
  long long site, drop, dt;
  void* stream;
  long long launches;
};

// few: no operand images, no partial sums and no z; h: m x pad16(f) fp32.  Else every operand comes with an optional image:
// [S][rows][pad16(cols)] 16-bit elements, S = 3 for fp32, needed for fp32 and for rows that do not start on 16-byte boundaries;
// h: [S][m][pad16(f)] 16-bit; z: 2 x (m rounded up to 32) x pad16(f) fp32 or null; partial: gated_ffn_partial_floats.
struct FfnForwardCall {
  const void* x;
  long long ldx;
  void* x_img;
  const void* w_in;
  long long ld_in;
  void* in_img;
  const void* w_out;
  long long ld_out;
  void *out_img, *h;
  float *z, *partial;
  void* y;
  long long m, d, f, n, act, dt, few;
  void* st;
  long long launches;
};

// x, w_in, w_out: as in the forward pass; where an image is given it holds the forward pass' image already, or (bits 0, 1, 2 of
// `make`) is scratch for one that is still to be made.
// dz: [S][2][m][pad16(f)] 16-bit scratch.  dx, dw_in, dw_out may be null.
struct FfnBackwardCall {
  const void* x;
  long long ldx;
  void* x_img;
  const void* w_in;
  long long ld_in;
  void* in_img;
  const void* w_out;
  long long ld_out;
  void* out_img;
  const void* dy;
  long long ldy;
  void* dy_img;
  const void* h;
  float* z;
  void* dz;
  float* partial;
  void *dx, *dw_in, *dw_out;
  long long make, m, d, f, n, act, dt;
  void* st;
  long long launches;
};

extern "C" {
int layer_norm_forward(LnForwardCall* c);
int layer_norm_backward(LnBackwardCall* c);
long long layer_norm_partial_floats(int d);
int dropout_apply(DropoutCall* c);
int gated_ffn_forward(FfnForwardCall* c);
int gated_ffn_backward(FfnBackwardCall* c);
int gated_ffn_few(int m, int d, int f, int n, int dt);
long long gated_ffn_partial_floats(int m, int d, int f, int n, int dt, int backward);
const char* choco_cuda_error_string(int code);
}
