// Parameter blocks and launchers of the short causal convolution and of activations in 8 bits (conv.cu).
#pragma once
#include <stdint.h>
#include <cuda_runtime.h>

namespace sq {

constexpr int kPackBlock = 128;       // values that share a scale

struct ConvParams {
  int batch, length, channels, taps, silu, type, weight_type;
  const void* x; long long x_sb, x_st;              // (b,t,c) at x + b*x_sb + t*x_st + c; null: the codes are read instead
  int8_t* codes; float* scales;                     // [B,L,C], [B,L,ceil(C/128)]: a forward with x writes them; may be null
  const void* weight; const void* bias;             // [C,taps], [C] or null
  const void* state_in;                             // [B,taps-1,C] in `type`, may be null
  const int* lengths;                               // [B], may be null
  void* y; long long y_sb, y_st;
  void* state_out;                                  // [B,taps-1,C], may be null
  // backward
  const void* dy; long long dy_sb, dy_st;           // in `type`, or fp32 where dy_f32 (a 16-bit type's)
  int dy_f32;
  const void* dstate_out;                           // [B,taps-1,C], may be null
  void* dx;                                         // contiguous
  void* dstate_in;                                  // may be null
  void *dweight, *dbias;                            // in the weights' type; may be null
  float* workspace;                                 // conv_workspace() bytes
};

struct ConvStepParams {
  int batch, channels, taps, silu, type, weight_type;
  const void* x; long long x_sb;
  const void *weight, *bias;
  void* state;                                      // [B,taps-1,C], updated in place
  void* y;                                          // contiguous, in `type`, or fp32 where y_f32
  int y_f32;
};

struct PackParams {
  long long rows; int width, type;
  const void* x; long long x_stride;
  int8_t* codes; float* scales;
  void* y;                                          // unpacked, contiguous
};

struct ConvTiles;
// The convolution (silu) of P's x or codes as a scan's tiles; P's channels are x, B and C side by side.
int launch_conv_tiles(const ConvParams& p, const ConvTiles& tiles, cudaStream_t stream);
// state_out alone, of x or codes.
int launch_conv_last(const ConvParams& p, cudaStream_t stream);
long long conv_workspace(int batch, int length, int channels);
int launch_conv_forward(const ConvParams& p, cudaStream_t stream);
int launch_conv_backward(const ConvParams& p, cudaStream_t stream);
int launch_conv_step(const ConvStepParams& p, cudaStream_t stream);
int launch_pack(const PackParams& p, cudaStream_t stream);
int launch_unpack(const PackParams& p, cudaStream_t stream);

}  // namespace sq
