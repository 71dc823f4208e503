/*
 * A HIP runtime of no devices but two imagined ones, for tests of the library's host code on a machine without a GPU: memory
 * is addresses nobody touches, kernels and copies end at once.  Loaded with RTLD_GLOBAL before libndbhip.so, whose calls then
 * come here; the stub_ functions tell what was asked for.
 */
#include <hip/hip_runtime_api.h>
#include <atomic>
#include <chrono>
#include <cstdlib>
#include <cstring>
#include <map>
#include <mutex>
#include <thread>

static thread_local int t_device;
static thread_local hipError_t t_last;
static std::mutex m;
static std::map<char *, size_t> live;
static size_t in_use, most, room = ~(size_t) 0;
static char *next_address = (char *) 0x100000000000;
static std::atomic<long> mallocs, frees, launches;
static std::atomic<int> launch_device{-1}, sync_ms;

static hipError_t
done(hipError_t e)
{
	if (e != hipSuccess)
		t_last = e;
	return e;
}

extern "C"
{
	long		stub_mallocs(void) { return mallocs; }
	long		stub_frees(void) { return frees; }
	long		stub_launches(void) { return launches; }
	int			stub_launch_device(void) { return launch_device; }
	size_t		stub_in_use(void) { return in_use; }
	size_t		stub_most(void) { size_t v = most; most = in_use; return v; }
	void		stub_set_room(size_t bytes) { room = bytes; }
	void		stub_set_sync_ms(int ms) { sync_ms = ms; }		/* what waiting for a stream takes */

	hipError_t	hipGetDeviceCount(int *n) { *n = 2; return hipSuccess; }
	hipError_t	hipSetDevice(int d) { t_device = d; return hipSuccess; }
	hipError_t	hipGetDevice(int *d) { *d = t_device; return hipSuccess; }
	hipError_t	hipGetDeviceProperties(hipDeviceProp_t *p, int)		/* (a macro: the symbol carries a version) */
	{
		memset(p, 0, sizeof(*p));
		strcpy(p->gcnArchName, "gfx950");
		p->multiProcessorCount = 256;
		return hipSuccess;
	}
	hipError_t	hipStreamCreateWithFlags(hipStream_t *s, unsigned) { *s = (hipStream_t) malloc(16); return hipSuccess; }
	hipError_t	hipStreamDestroy(hipStream_t s) { free(s); return hipSuccess; }
	hipError_t	hipStreamSynchronize(hipStream_t)
	{
		if (sync_ms)
			std::this_thread::sleep_for(std::chrono::milliseconds(sync_ms));
		return hipSuccess;
	}
	hipError_t	hipFuncSetAttribute(const void *, hipFuncAttribute, int) { return hipSuccess; }
	hipError_t	hipGetLastError(void) { hipError_t e = t_last; t_last = hipSuccess; return e; }
	hipError_t	hipHostMalloc(void **p, size_t n, unsigned) { *p = malloc(n); return hipSuccess; }
	hipError_t	hipHostFree(void *p) { free(p); return hipSuccess; }
	hipError_t	hipMemset(void *, int, size_t) { return hipSuccess; }
	hipError_t	hipMemcpyAsync(void *, const void *, size_t, hipMemcpyKind, hipStream_t) { return hipSuccess; }

	hipError_t	hipMalloc(void **p, size_t n)
	{
		std::lock_guard<std::mutex> lk(m);

		if (n > room - in_use)
			return done(hipErrorOutOfMemory);
		mallocs++;
		*p = next_address;
		live[next_address] = n;
		next_address += (n + 4095) / 4096 * 4096;
		in_use += n;
		if (in_use > most)
			most = in_use;
		return hipSuccess;
	}
	hipError_t	hipFree(void *p)
	{
		std::lock_guard<std::mutex> lk(m);
		auto		it = live.find((char *) p);

		if (!p)
			return hipSuccess;
		if (it == live.end())
			abort();			/* (freed twice, or never given) */
		frees++;
		in_use -= it->second;
		live.erase(it);
		return hipSuccess;
	}

	static thread_local struct { dim3 g, b; size_t s; hipStream_t q; } t_cfg;
	hipError_t	__hipPushCallConfiguration(dim3 g, dim3 b, size_t s, hipStream_t q) { t_cfg = {g, b, s, q}; return hipSuccess; }
	hipError_t	__hipPopCallConfiguration(dim3 *g, dim3 *b, size_t *s, hipStream_t *q)
	{
		*g = t_cfg.g;
		*b = t_cfg.b;
		*s = t_cfg.s;
		*q = t_cfg.q;
		return hipSuccess;
	}
	hipError_t	hipLaunchKernel(const void *, dim3 g, dim3 b, void **, size_t, hipStream_t)
	{
		/* what HIP refuses: nothing to do, or more threads along an axis than 32 bits count */
		if (!g.x || !g.y || !g.z || (uint64_t) g.x * b.x >> 32 || (uint64_t) g.y * b.y >> 32 || g.y > 65535 || g.z > 65535 || b.x * b.y * b.z > 1024)
			return done(hipErrorInvalidConfiguration);
		launches++;
		launch_device = t_device;
		return hipSuccess;
	}
}
