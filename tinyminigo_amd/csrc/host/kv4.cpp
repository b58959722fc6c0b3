// The kernel-level entry points of the 4-bit KV cache: argument checks and
// launches.  Whatever the caller's arguments say about sizes, strides and
// alignment is checked here; positions that live on the device are checked by
// the kernels (kv4_pos in kv4.cuh).
#include <cmath>
#include <cstring>

#include "../kernels/kernels.hpp"
#include "common.hpp"

using namespace tmg;

namespace {

// Makes the device of a stream current for a call.
class StreamDevice {
  public:
    // TMG_OK, or an error: the memory at `data` must be on that device
    int enter(hipStream_t s, const void *data) {
        int cur = 0, dev = 0;
        if (hipGetDevice(&cur) != hipSuccess) return device_error("no HIP device available");
        dev = cur;
        if (s && hipStreamGetDevice(s, &dev) != hipSuccess) return device_error("bad stream");
        hipPointerAttribute_t at;
        memset(&at, 0, sizeof(at));
        if (hipPointerGetAttributes(&at, data) != hipSuccess ||
            (at.type != hipMemoryTypeDevice && at.type != hipMemoryTypeManaged)) {
            (void)hipGetLastError();
            return set_error(TMG_E_INVALID, "the cache is not in device memory");
        }
        if (at.type == hipMemoryTypeDevice && at.device != dev)
            return set_error(TMG_E_INVALID, "the cache is on another device than the stream");
        if (dev != cur) {
            if (hipSetDevice(dev) != hipSuccess) return device_error("cannot use the stream's device");
            back_ = cur;
        }
        return TMG_OK;
    }
    ~StreamDevice() {
        if (back_ >= 0) (void)hipSetDevice(back_);
    }

  private:
    static int device_error(const char *what) {
        (void)hipGetLastError();
        return set_error(TMG_E_DEVICE, what);
    }
    int back_ = -1;
};

int launched(hipError_t e, const char *what) {
    return e == hipSuccess ? TMG_OK : set_error(TMG_E_DEVICE, std::string("HIP error ") + hipGetErrorString(e) + " in " + what);
}

bool shape_ok(uint32_t cap, uint32_t nkv, uint32_t hd) {
    const bool head = hd == 16 || hd == 32 || hd == 64 || hd == 128 || hd == 256;
    return head && nkv >= 1 && nkv <= 32767 && cap >= 1 && cap <= 1u << 30;
}

bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }

// The checks that write, read and attention share; `rows` rows at pos.
int check_cache(const tmg_kv4 *kv, uint32_t rows, const int32_t *pos_dev, uint32_t pos) {
    if (!kv || !kv->data) return set_error(TMG_E_INVALID, "null 4-bit cache");
    if (!shape_ok(kv->cap, kv->nkv, kv->hd))
        return set_error(TMG_E_INVALID, "a 4-bit cache has 1..2^30 positions, 1..32767 KV heads and a head_dim of 16, 32, 64, 128 or 256");
    if (!aligned16(kv->data) || kv->seq_stride % 16 != 0)
        return set_error(TMG_E_INVALID, "a 4-bit cache is 16-byte aligned, and so is its sequence stride");
    if (kv->n_seq > 65535) return set_error(TMG_E_INVALID, "at most 65535 sequences");
    if (kv->n_seq > 1 && kv->seq_stride < kv4_slab_bytes(kv->cap, (int)kv->nkv, (int)kv->hd))
        return set_error(TMG_E_INVALID, "sequence stride below a sequence's bytes");
    if ((uintptr_t)pos_dev & 3) return set_error(TMG_E_INVALID, "positions must be 4-byte aligned");
    // a launch has fewer than 2^32 threads along a dimension
    if ((uint64_t)rows * (kv->hd / 8) > 1u << 31) return set_error(TMG_E_INVALID, "too many rows for one call");
    if (rows > kv->cap || (!pos_dev && (uint64_t)pos + rows > kv->cap))
        return set_error(TMG_E_CAPACITY, "rows past the 4-bit cache's capacity (" + std::to_string(kv->cap) + " positions)");
    return TMG_OK;
}

// A row stride of 0 is `width` itself.
int check_rows(const char *what, const void *p, size_t *stride, size_t width) {
    if (*stride == 0) *stride = width;
    if (!aligned16(p)) return set_error(TMG_E_INVALID, std::string(what) + " must be 16-byte aligned");
    if (*stride < width || *stride % 4 != 0)
        return set_error(TMG_E_INVALID, std::string(what) + "'s row stride must be a multiple of 4 and hold a row");
    return TMG_OK;
}

Kv4Cache view(const tmg_kv4 *kv) {
    return Kv4Cache{(uint8_t *)kv->data, kv->seq_stride, (int)kv->n_seq, kv->cap, (int)kv->nkv, (int)kv->hd};
}

}  // namespace

extern "C" size_t tmg_kv4_bytes(uint32_t cap, uint32_t nkv, uint32_t hd) {
    return shape_ok(cap, nkv, hd) ? kv4_slab_bytes(cap, (int)nkv, (int)hd) : 0;
}

extern "C" int tmg_kv4_write(const tmg_kv4 *kv, const float *k, const float *v, size_t row_stride, uint32_t rows,
                             const int32_t *pos_dev, uint32_t pos, void *stream) {
    clear_error();
    int rc = check_cache(kv, rows, pos_dev, pos);
    if (rc) return rc;
    if (!k || !v) return set_error(TMG_E_INVALID, "null rows");
    if ((rc = check_rows("k", k, &row_stride, (size_t)kv->nkv * kv->hd)) ||
        (rc = check_rows("v", v, &row_stride, (size_t)kv->nkv * kv->hd)))
        return rc;
    if (rows == 0 || kv->n_seq == 0) return TMG_OK;
    StreamDevice dev;
    if ((rc = dev.enter((hipStream_t)stream, kv->data))) return rc;
    const Kv4WriteArgs a{view(kv), k, v, row_stride, (int)rows, pos_dev, (int)pos};
    return launched(launch_kv4_write(a, (hipStream_t)stream), "tmg_kv4_write");
}

extern "C" int tmg_kv4_read(const tmg_kv4 *kv, float *k, float *v, size_t row_stride, uint32_t rows,
                            const int32_t *pos_dev, uint32_t pos, void *stream) {
    clear_error();
    int rc = check_cache(kv, rows, pos_dev, pos);
    if (rc) return rc;
    if (!k && !v) return set_error(TMG_E_INVALID, "null rows");
    if ((rc = check_rows("k", k, &row_stride, (size_t)kv->nkv * kv->hd)) ||
        (rc = check_rows("v", v, &row_stride, (size_t)kv->nkv * kv->hd)))
        return rc;
    if (rows == 0 || kv->n_seq == 0) return TMG_OK;
    StreamDevice dev;
    if ((rc = dev.enter((hipStream_t)stream, kv->data))) return rc;
    const Kv4ReadArgs a{view(kv), k, v, row_stride, (int)rows, pos_dev, (int)pos};
    return launched(launch_kv4_read(a, (hipStream_t)stream), "tmg_kv4_read");
}

namespace {

int check_heads(const tmg_kv4 *kv, uint32_t rows, uint32_t nq) {
    if (nq == 0 || nq % kv->nkv != 0 || nq > 65536)
        return set_error(TMG_E_INVALID, "query heads must be a multiple of the KV heads");
    // columns stay within 31 bits, and the threads of 256 for 16 of them
    const uint64_t ncol = (uint64_t)rows * (nq / kv->nkv);
    if (ncol > 0x7ffffff0u || (ncol + 15) / 16 * kv->nkv * kv->n_seq > 1u << 23)
        return set_error(TMG_E_INVALID, "too many query rows for one call");
    return TMG_OK;
}

}  // namespace

extern "C" int tmg_kv4_attn_workspace(const tmg_kv4 *kv, uint32_t rows, uint32_t nq, size_t *bytes) {
    clear_error();
    if (!bytes) return set_error(TMG_E_INVALID, "null argument");
    int rc = check_cache(kv, rows, nullptr, 0);
    if (!rc) rc = check_heads(kv, rows, nq);
    if (rc) return rc;
    *bytes = rows && kv->n_seq ? kv4_attn_ws_bytes(view(kv), (int)rows, (int)nq) : 0;
    return TMG_OK;
}

extern "C" int tmg_kv4_attn(const tmg_kv4 *kv, const tmg_kv4_attn_args *p, void *stream) {
    clear_error();
    if (!p) return set_error(TMG_E_INVALID, "null argument");
    int rc = check_cache(kv, p->rows, p->pos_dev, p->pos);
    if (!rc) rc = check_heads(kv, p->rows, p->nq);
    if (rc) return rc;
    if (!p->q || !p->out) return set_error(TMG_E_INVALID, "null rows");
    if (!p->k_new != !p->v_new) return set_error(TMG_E_INVALID, "new keys and new values come together");
    size_t q_stride = p->q_stride, out_stride = p->out_stride, new_stride = p->new_stride;
    if ((rc = check_rows("q", p->q, &q_stride, (size_t)p->nq * kv->hd)) ||
        (rc = check_rows("out", p->out, &out_stride, (size_t)p->nq * kv->hd)) ||
        (rc = check_rows("k_new", p->k_new, &new_stride, (size_t)kv->nkv * kv->hd)) ||
        (rc = check_rows("v_new", p->v_new, &new_stride, (size_t)kv->nkv * kv->hd)))
        return rc;
    if (!std::isfinite(p->scale)) return set_error(TMG_E_INVALID, "the scale must be finite");
    if (p->rows == 0 || kv->n_seq == 0) return TMG_OK;
    const size_t need = kv4_attn_ws_bytes(view(kv), (int)p->rows, (int)p->nq);
    if (need && (!p->ws || p->ws_bytes < need || !aligned16(p->ws)))
        return set_error(TMG_E_INVALID, "the workspace must be 16-byte aligned and hold " + std::to_string(need) + " bytes");
    StreamDevice dev;
    if ((rc = dev.enter((hipStream_t)stream, kv->data))) return rc;
    Kv4AttnArgs a{};
    a.c = view(kv);
    a.q = p->q;
    a.q_stride = q_stride;
    a.out = p->out;
    a.out_stride = out_stride;
    a.nq = (int)p->nq;
    a.rows = (int)p->rows;
    a.pos_dev = p->pos_dev;
    a.pos = (int)p->pos;
    a.k_new = p->k_new;
    a.v_new = p->v_new;
    a.new_stride = new_stride;
    a.scale = p->scale != 0.0f ? p->scale : 1.0f / sqrtf((float)kv->hd);
    return launched(launch_kv4_attn(a, p->ws, (hipStream_t)stream), "tmg_kv4_attn");
}
