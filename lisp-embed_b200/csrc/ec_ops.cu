// ec_ops.cu -- the device of an operator call and the checks of packed rows.
#include "ec_ops.h"

#include <mutex>

namespace ec {

int OpDevice::enter(std::initializer_list<const void*> ptrs, int dev) {
  for (const void* p : ptrs) {
    if (!p) continue;
    cudaPointerAttributes a;
    if (int rc = check_cuda(cudaPointerGetAttributes(&a, p), "cudaPointerGetAttributes")) return rc;
    if (a.type != cudaMemoryTypeDevice && a.type != cudaMemoryTypeManaged)
      return set_error(EC_EINVAL, "a buffer is not device memory");
    if (dev < 0) dev = a.device;
    if (a.device != dev)
      return set_error(EC_EINVAL, "buffers on devices %d and %d: one call takes buffers of one device", dev, a.device);
  }
  if (dev < 0) return set_error(EC_EINVAL, "no device buffer");
  int cur = -1;
  if (int rc = check_cuda(cudaGetDevice(&cur), "cudaGetDevice")) return rc;
  if (cur != dev) {
    if (int rc = check_cuda(cudaSetDevice(dev), "cudaSetDevice")) return rc;
    prev_ = cur;
  }
  dev_ = dev;
  // number of SMs per device, looked up once; the library is built for sm_100a
  static std::mutex mu;
  static int sms[64] = {};
  std::lock_guard<std::mutex> lk(mu);
  if (dev >= 64) return set_error(EC_EINVAL, "device ordinal %d out of range", dev);
  if (!sms[dev]) {
    int major = 0, minor = 0, n = 0;
    int rc = check_cuda(cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev), "attr");
    if (!rc) rc = check_cuda(cudaDeviceGetAttribute(&minor, cudaDevAttrComputeCapabilityMinor, dev), "attr");
    if (!rc) rc = check_cuda(cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev), "attr");
    if (rc) return rc;
    if (major != 10)
      return set_error(EC_EUNSUPPORTED, "device %d is sm_%d%d; this library is built for sm_100a", dev, major, minor);
    sms[dev] = n;
  }
  sms_ = sms[dev];
  return EC_OK;
}

int kv_enter(OpDevice& dev, const KvOpen& c, std::initializer_list<const void*> ptrs) {
  int on = c.device.load(std::memory_order_relaxed);
  if (on < 0) {
    if (int rc = dev.enter({c.k, c.v, c.tables, c.lens, c.refs, c.work})) {
      const std::string why = ec_last_error();
      return set_error(rc, "the cache's memory: %s", why.c_str());
    }
    c.device.store(on = dev.ordinal(), std::memory_order_relaxed);
  }
  return dev.enter(ptrs, on);
}

OpDevice::~OpDevice() {
  if (prev_ >= 0) cudaSetDevice(prev_);
}

bool op_rows_apart(int64_t token, int64_t head, int64_t tokens, int heads, int head_dim) {
  if (tokens <= 1 || heads <= 1) return true;
  // one of the two strides steps over everything of the other (in double: the
  // products pass 64 bits where they are far apart)
  return static_cast<double>(token) >= static_cast<double>(heads - 1) * head + head_dim ||
         static_cast<double>(head) >= static_cast<double>(tokens - 1) * token + head_dim;
}

int op_check_rows(const char* name, OpRows& r, int64_t tokens, int heads, int head_dim) {
  if (heads == 1) r.head = 0;
  if (tokens <= 1) r.token = 0;
  if (!r.p && tokens > 0) return set_error(EC_EINVAL, "%s is NULL", name);
  if (!op_aligned(r.p, 16)) return set_error(EC_EINVAL, "%s must be 16-byte aligned", name);
  if (r.token % 8 || r.head % 8)
    return set_error(EC_EINVAL, "%s: strides %lld / %lld are not multiples of 8 elements (16 bytes)", name,
                     static_cast<long long>(r.token), static_cast<long long>(r.head));
  if ((heads > 1 && r.head < head_dim) || (tokens > 1 && r.token < head_dim) || r.token < 0 || r.head < 0 ||
      r.token >= (int64_t(1) << 38) || r.head >= (int64_t(1) << 38))
    return set_error(EC_EINVAL, "%s: strides %lld / %lld overlap heads of %d", name, static_cast<long long>(r.token),
                     static_cast<long long>(r.head), head_dim);
  return EC_OK;
}

}  // namespace ec
