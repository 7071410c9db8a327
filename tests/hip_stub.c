/* A stand-in for the HIP runtime, for tests of what the library does around its GPU calls (test_start_up_cpu.py and others):
 * device memory is host memory, copies are done at once, kernels do nothing; it counts launches, allocations and frees, and
 * says that every stream is captured while stub_capturing is set. */
#define _GNU_SOURCE
#include <dirent.h>
#include <pthread.h>
#include <stdatomic.h>
#include <stdio.h>
#include <stdlib.h>
#include <string.h>
#include <sys/mman.h>
#include <unistd.h>

typedef struct { unsigned x, y, z; } dim3;
typedef int hipError_t;

atomic_int stub_launches, stub_mallocs, stub_frees, stub_capturing;

static int threads_of_this_process(void)
{
    int n = 0;
    DIR *d = opendir("/proc/self/task");
    for (struct dirent *e; d && (e = readdir(d));) n += e->d_name[0] != '.';
    if (d) closedir(d);
    return n;
}
/* the runtime comes up with the first call: it takes its time, and says how many threads the process has meanwhile */
static void start_up(void)
{
    static pthread_mutex_t mu = PTHREAD_MUTEX_INITIALIZER;
    static int up;
    pthread_mutex_lock(&mu);
    if (!up && getenv("STUB_START_UP")) {
        int most = threads_of_this_process();
        for (int i = 0; i < 20; i++) {
            usleep(5000);
            const int n = threads_of_this_process();
            most = n > most ? n : most;
        }
        fprintf(stderr, "stub: %d thread(s) while the runtime comes up\n", most);
    }
    up = 1;
    pthread_mutex_unlock(&mu);
}
static void enter(void) { start_up(); }
static hipError_t leave(void) { return 0; }
#define PLAIN { enter(); return leave(); }

hipError_t hipGetDeviceCount(int *n) { enter(); *n = 1; return leave(); }
hipError_t hipSetDevice(int d) { (void)d; PLAIN }
hipError_t hipGetDevice(int *d) { enter(); *d = 0; return leave(); }
hipError_t hipGetLastError(void) { return 0; }
const char *hipGetErrorString(hipError_t e) { (void)e; return "stub error"; }
static hipError_t get(void **p, size_t n)
{
    enter();
    *p = calloc(1, n ? n : 1);
    atomic_fetch_add(&stub_mallocs, 1);
    return leave();
}
static hipError_t put(void *p)
{
    enter();
    if (p) atomic_fetch_add(&stub_frees, 1);
    free(p);
    return leave();
}
hipError_t hipMalloc(void **p, size_t n) { return get(p, n); }
hipError_t hipFree(void *p) { return put(p); }
/* pinned: mappings of their own, a page that holds the length in front, pages that nobody may touch around them */
hipError_t hipHostMalloc(void **p, size_t n, unsigned f)
{
    (void)f;
    enter();
    const size_t len = (n + 4095) / 4096 * 4096;
    char *m = mmap(0, len + 12288, PROT_NONE, MAP_PRIVATE | MAP_ANONYMOUS, -1, 0);
    mprotect(m, 4096, PROT_READ | PROT_WRITE);
    *(size_t *)m = len + 12288;
    mprotect(m, 4096, PROT_READ);
    mprotect(m + 4096, 4096, PROT_NONE);
    mprotect(m + 8192, len, PROT_READ | PROT_WRITE);
    *p = m + 8192;
    return leave();
}
hipError_t hipHostFree(void *p)
{
    enter();
    if (p) munmap((char *)p - 8192, *(size_t *)((char *)p - 8192));
    return leave();
}
hipError_t hipHostGetDevicePointer(void **d, void *h, unsigned f) { (void)f; enter(); *d = h; return leave(); }
hipError_t hipMemcpy(void *d, const void *s, size_t n, int k) { (void)k; enter(); memcpy(d, s, n); return leave(); }
hipError_t hipMemcpyAsync(void *d, const void *s, size_t n, int k, void *q) { (void)k; (void)q; enter(); memcpy(d, s, n); return leave(); }
hipError_t hipMemsetAsync(void *d, int v, size_t n, void *q) { (void)q; enter(); memset(d, v, n); return leave(); }
hipError_t hipStreamCreateWithFlags(void **s, unsigned f) { (void)f; return get(s, 16); }
hipError_t hipStreamDestroy(void *s) { return put(s); }
hipError_t hipStreamSynchronize(void *s) { (void)s; PLAIN }
hipError_t hipStreamWaitEvent(void *s, void *e, unsigned f) { (void)s; (void)e; (void)f; PLAIN }
hipError_t hipStreamIsCapturing(void *s, int *status) { (void)s; enter(); *status = atomic_load(&stub_capturing) ? 1 : 0; return leave(); }
hipError_t hipEventCreate(void **e) { return get(e, 16); }
hipError_t hipEventCreateWithFlags(void **e, unsigned f) { (void)f; return get(e, 16); }
hipError_t hipEventDestroy(void *e) { return put(e); }
hipError_t hipEventRecord(void *e, void *s) { (void)e; (void)s; PLAIN }
hipError_t hipEventSynchronize(void *e) { (void)e; PLAIN }
hipError_t hipEventQuery(void *e) { (void)e; PLAIN }
hipError_t hipEventElapsedTime(float *ms, void *a, void *b) { (void)a; (void)b; enter(); *ms = 1.0f; return leave(); }
hipError_t hipFuncSetAttribute(const void *f, int a, int v) { (void)f; (void)a; (void)v; PLAIN }
hipError_t hipFuncGetAttributes(void *a, const void *f) { (void)a; (void)f; PLAIN }
hipError_t hipDeviceGetAttribute(int *v, int a, int d) { (void)a; (void)d; enter(); *v = 256; return leave(); }
hipError_t hipDeviceGetPCIBusId(char *b, int n, int d) { (void)d; enter(); snprintf(b, (size_t)n, "0000:00:00.0"); return leave(); }
hipError_t hipLaunchKernel(const void *f, dim3 g, dim3 b, void **a, size_t l, void *s)
{
    (void)f; (void)g; (void)b; (void)a; (void)l; (void)s;
    enter();
    atomic_fetch_add(&stub_launches, 1);
    return leave();
}
hipError_t __hipPushCallConfiguration(dim3 g, dim3 b, size_t l, void *s) { (void)g; (void)b; (void)l; (void)s; return 0; }
hipError_t __hipPopCallConfiguration(dim3 *g, dim3 *b, size_t *l, void **s)
{
    g->x = g->y = g->z = b->x = b->y = b->z = 1;
    *l = 0;
    *s = 0;
    return 0;
}
void **__hipRegisterFatBinary(const void *d) { static void *handle; (void)d; return &handle; }
void __hipUnregisterFatBinary(void **h) { (void)h; }
void __hipRegisterFunction(void **m, const void *f, char *d, const char *n, unsigned t, void *a, void *b, void *c, void *e, int *w)
{
    (void)m; (void)f; (void)d; (void)n; (void)t; (void)a; (void)b; (void)c; (void)e; (void)w;
}
