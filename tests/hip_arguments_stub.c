/* A stand-in for the part of the HIP runtime that a kernel launch uses, loaded ahead of it: launches do
 * nothing and are counted, and the first bytes of the last one's first argument, its grid and its block are kept. Settings of
 * a kernel's attributes are counted, and the one whose number is llmopt_stub_refuse fails. For the products of 8-bit
 * floating point. */
#include <stddef.h>
#include <string.h>

typedef struct { unsigned x, y, z; } dim3_t;

int llmopt_stub_launches = 0;
int llmopt_stub_attributes = 0;
int llmopt_stub_refuse = 0;
unsigned char llmopt_stub_argument[96]; /* the products' argument blocks are larger */
unsigned llmopt_stub_grid[3], llmopt_stub_block[3];
static dim3_t grid_, block_;
static size_t shared_;
static void* stream_;

int __hipPushCallConfiguration(dim3_t grid, dim3_t block, size_t shared, void* stream) {
  grid_ = grid, block_ = block, shared_ = shared, stream_ = stream;
  return 0;
}

int __hipPopCallConfiguration(dim3_t* grid, dim3_t* block, size_t* shared, void** stream) {
  *grid = grid_, *block = block_, *shared = shared_, *stream = stream_;
  return 0;
}

int hipLaunchKernel(const void* f, dim3_t grid, dim3_t block, void** args, size_t shared, void* stream) {
  (void)f, (void)shared, (void)stream;
  memcpy(llmopt_stub_argument, args[0], sizeof(llmopt_stub_argument));
  llmopt_stub_grid[0] = grid.x, llmopt_stub_grid[1] = grid.y, llmopt_stub_grid[2] = grid.z;
  llmopt_stub_block[0] = block.x, llmopt_stub_block[1] = block.y, llmopt_stub_block[2] = block.z;
  ++llmopt_stub_launches;
  return 0;
}

int hipGetLastError(void) { return 0; }

int hipFuncSetAttribute(const void* f, int attribute, int value) {
  (void)f, (void)attribute, (void)value;
  return ++llmopt_stub_attributes == llmopt_stub_refuse ? 1 : 0; /* hipErrorInvalidValue */
}
