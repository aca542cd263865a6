// Parameter block and launchers of the selective scan in unquantised states (selective.cu).
#pragma once
#include <stdint.h>
#include <cuda_runtime.h>

namespace sq {

constexpr int kScanChunk = 128;       // tokens of a chunk
constexpr int kScanTile = 64;         // rows of a head's state that one CTA works on
constexpr int kScanMaxDim = 1024;
constexpr int kScanMaxUnits = 30000;                // heads * tiles of 64 rows: a grid holds two B/C tiles a group and eighths of the heads besides
enum { SQ_TYPE_F16 = 0, SQ_TYPE_BF16 = 1, SQ_TYPE_F32 = 2 };

struct SelectiveParams {
  int batch, length, heads, dim, groups, type;              // type: SQ_F16 / SQ_BF16 of x, dt, B, C, y and their gradients
  const void* x; long long x_sb, x_st;                      // (b,t,h,p) at x + b*x_sb + t*x_st + h*dim + p
  const void* dt; long long dt_sb, dt_st;
  const float* A;
  const void* B; long long b_sb, b_st;
  const void* C; long long c_sb, c_st;
  const void* D; int d_type;                                // may be null; SQ_F16 / SQ_BF16 / SQ_F32
  const void* dt_bias; int bias_type;                       // may be null
  const float* state_in;                                    // [B,H,P,128], may be null
  const int* lengths;                                       // [B], may be null
  void* y; long long y_sb, y_st;
  float* state_out;                                         // may be null
  // backward
  const void* dy; long long dy_sb, dy_st;
  const float* dstate_out;                                  // may be null
  void* dx; long long dx_sb, dx_st;                         // gradients in `type`, of x, dt (contiguous), B and C; tiled: of x, B and C in fp32
  void* ddt;
  void *dB, *dC; long long dg_sb, dg_st;
  float* dA; void* dD; void* dbias;                         // each may be null
  float* dstate_in;                                         // may be null
  void* workspace;
  int* err;
  int tiled;                                                // x, B and C are tiles in the workspace (conv_tiles), not read from above
};

// Where a convolution puts its output for a scan: tiles of 128 tokens by 64 (x) or 128 (B, C) channels, scaled fp16 as
// shared memory holds them, and what brings each back.
struct ConvTiles {
  int heads, dim, groups, chunks, units;
  uint16_t *x, *b, *c;
  float *xback, *bback, *cback;
};
ConvTiles selective_tiles(const SelectiveParams& p, bool backward);

struct SelectiveStepParams {
  int batch, heads, dim, groups, type;
  const void* x; long long x_sb;
  const void* dt; long long dt_sb;
  const float* A;
  const void* B; long long b_sb;
  const void* C; long long c_sb;
  const void* D; int d_type;
  const void* dt_bias; int bias_type;
  float* state;                                             // [B,H,P,128], updated in place
  void* y;                                                  // contiguous
  int x_f32;                                                // x, B and C are fp32
  int behind;                                               // launched behind the kernel that writes x, B and C
};

long long selective_workspace(int batch, int length, int heads, int dim, int groups, bool backward, bool tiled);
int launch_selective_forward(const SelectiveParams& p, cudaStream_t stream);
int launch_selective_backward(const SelectiveParams& p, cudaStream_t stream);
int launch_selective_step(const SelectiveStepParams& p, cudaStream_t stream);

}  // namespace sq
