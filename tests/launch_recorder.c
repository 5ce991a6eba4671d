/* Stands in for the HIP runtime under libgq_hip.so in a process without a GPU: it launches nothing and writes down what would have
 * been launched, and every limit of LDS that is set.  Loaded globally before the library, whose references then end here. */
#include <stdint.h>
#include <stdio.h>
#include <stdlib.h>

typedef struct {
  uint32_t x, y, z;
} dim3;

typedef struct {
  int32_t launch;   /* 1: a launch; 0: a limit of LDS was set */
  int32_t device;
  uint32_t grid[3], block[3];
  uint64_t lds;     /* of the launch, or the limit */
  char kernel[160];
} record;

static record *records;
static int n_records, room, device;

static const void *functions[4096];
static const char *names[4096];
static int n_functions;

static dim3 grid_, block_;
static size_t lds_;
static void *stream_;

static record *add(const void *function) {
  if (n_records == room) records = realloc(records, (room = 2 * room + 64) * sizeof(record));
  record *r = records + n_records++;
  const char *name = "?";
  for (int i = 0; i < n_functions; ++i)
    if (functions[i] == function) name = names[i];
  snprintf(r->kernel, sizeof(r->kernel), "%s", name);
  r->device = device;
  return r;
}

/* for the test */
int recorder_count(void) { return n_records; }
const record *recorder_record(int i) { return records + i; }
void recorder_clear(void) { n_records = 0; }
void recorder_device(int d) { device = d; }

/* for the library */
void **__hipRegisterFatBinary(const void *data) {
  static void *handle;
  (void)data;
  return &handle;
}
void __hipUnregisterFatBinary(void **handle) { (void)handle; }
void __hipRegisterFunction(void **handle, const void *function, char *device_function, const char *name, unsigned threads, void *tid,
                           void *bid, void *block, void *grid, int *warp) {
  (void)handle, (void)device_function, (void)threads, (void)tid, (void)bid, (void)block, (void)grid, (void)warp;
  functions[n_functions] = function, names[n_functions++] = name;
}
void __hipRegisterVar(void **handle, void *var, char *host, char *name, int external, size_t size, int constant, int global) {
  (void)handle, (void)var, (void)host, (void)name, (void)external, (void)size, (void)constant, (void)global;
}
int __hipPushCallConfiguration(dim3 grid, dim3 block, size_t lds, void *stream) {
  grid_ = grid, block_ = block, lds_ = lds, stream_ = stream;
  return 0;
}
int __hipPopCallConfiguration(dim3 *grid, dim3 *block, size_t *lds, void **stream) {
  *grid = grid_, *block = block_, *lds = lds_, *stream = stream_;
  return 0;
}
int hipLaunchKernel(const void *function, dim3 grid, dim3 block, void **args, size_t lds, void *stream) {
  record *r = add(function);
  (void)args, (void)stream;
  r->launch = 1;
  r->grid[0] = grid.x, r->grid[1] = grid.y, r->grid[2] = grid.z;
  r->block[0] = block.x, r->block[1] = block.y, r->block[2] = block.z;
  r->lds = lds;
  return 0;
}
int hipFuncSetAttribute(const void *function, int attribute, int value) {
  record *r = add(function);
  (void)attribute;
  r->launch = 0;
  r->lds = (uint64_t)value;
  return 0;
}
int hipGetDevice(int *d) {
  *d = device;
  return 0;
}
int hipDeviceGetAttribute(int *value, int attribute, int d) {
  (void)attribute, (void)d;
  *value = 256;
  return 0;
}
int hipGetLastError(void) { return 0; }
const char *hipGetErrorString(int e) {
  (void)e;
  return "";
}
int hipGetSymbolAddress(void **p, const void *symbol) {
  (void)symbol;
  *p = (void *)256;
  return 0;
}
int hipStreamIsCapturing(void *stream, int *status) {
  (void)stream;
  *status = 0;
  return 0;
}
int hipStreamQuery(void *stream) {
  (void)stream;
  return 0;
}
