// The operators of normalised layers and activation checkpoints on torch tensors.  Included by torch_ops.cpp; the same
// rules: the straightforward case only, None for anything else (khan_b200/layer_mod.py then converts or refuses).
#pragma once

namespace {

using NormFn = int (*)(const void*, long long, const void* const*, const void* const*, int, double, const int*, void*, void*,
                       void*, void*);
using NormGradFn = int (*)(const void*, long long, const void*, long long, const void* const*, const void*, const void*, int,
                           const int*, void*, void* const*, void* const*, void*, void*);
using SumsBytesFn = size_t (*)(int, const int*, int, int);
using CheckpointFn = int (*)(const float*, long long, const void* const*, const void* const*, int, double, int, const int*,
                             float*, unsigned char*, float*, float*, float*, void*);
using CheckpointGradFn = int (*)(const unsigned char*, const float*, const float*, const float*, const float*, long long,
                                 const void* const*, const void* const*, int, int, const int*, float*, void* const*,
                                 void* const*, void* const*, void*, void*);
using CheckpointWgradFn = int (*)(const unsigned char*, const float*, const float*, const float*, const void* const*,
                                  const void* const*, int, int, const float*, long long, int, const int*, void* const*, void*,
                                  void*);
using WgradBytesFn = size_t (*)(int, int, const int*);
using WidthFn = int (*)(int);

constexpr int64_t kMaxWidth = 4096;

struct LayerFns {
    NormFn norm[2];            // f32, f64
    NormGradFn norm_grad[2];
    SumsBytesFn sums_bytes;
    CheckpointFn checkpoint;
    CheckpointGradFn checkpoint_grad;
    CheckpointWgradFn checkpoint_wgrad;
    WgradBytesFn wgrad_bytes;
    WidthFn row_bytes, blocks;
} g_layers = {};

void bind_layers(const std::vector<uintptr_t>& f)
{
    if (f.size() != 11) throw py::value_error("bind_layers takes eleven addresses");
    g_layers.norm[0] = reinterpret_cast<NormFn>(f[0]);
    g_layers.norm[1] = reinterpret_cast<NormFn>(f[1]);
    g_layers.norm_grad[0] = reinterpret_cast<NormGradFn>(f[2]);
    g_layers.norm_grad[1] = reinterpret_cast<NormGradFn>(f[3]);
    g_layers.sums_bytes = reinterpret_cast<SumsBytesFn>(f[4]);
    g_layers.checkpoint = reinterpret_cast<CheckpointFn>(f[5]);
    g_layers.checkpoint_grad = reinterpret_cast<CheckpointGradFn>(f[6]);
    g_layers.checkpoint_wgrad = reinterpret_cast<CheckpointWgradFn>(f[7]);
    g_layers.wgrad_bytes = reinterpret_cast<WgradBytesFn>(f[8]);
    g_layers.row_bytes = reinterpret_cast<WidthFn>(f[9]);
    g_layers.blocks = reinterpret_cast<WidthFn>(f[10]);
}

// Rows of `width` values with a row stride that the kernels take.
bool fits_rows(const at::Tensor& t, c10::ScalarType dtype, c10::Device device, int64_t n, int64_t width)
{
    return t.scalar_type() == dtype && t.device() == device && t.dim() == 2 && t.size(0) == n && t.size(1) == width &&
           (width == 1 || t.stride(1) == 1) && (n <= 1 || t.stride(0) >= width);
}
long long row_stride(const at::Tensor& t) { return std::max<long long>(t.size(0) > 1 ? t.stride(0) : 0, t.size(1)); }

struct Rows {
    int acs[4] = {};
    bool grouped = false;      // counts of four elements were given, and parameters for each
    int groups() const { return grouped ? 4 : 1; }
};
bool read_rows(py::handle acs, int64_t n, Rows* r)
{
    if (n > INT32_MAX) return false;
    if (acs.is_none()) {
        r->acs[0] = (int)n;
        return true;
    }
    r->grouped = true;
    if (!read_counts(acs.ptr(), r->acs)) return false;
    int64_t sum = 0;
    for (int c : r->acs) {
        if (c < 0) return false;
        sum += c;
    }
    return sum == n;
}

// One vector of `width` values, or four of them where the rows are grouped.
bool read_vectors(py::handle given, const Rows& r, c10::ScalarType dtype, c10::Device device, int64_t width, const void** out)
{
    auto one = [&](py::handle h, int t) {
        if (!THPVariable_Check(h.ptr())) return false;
        const at::Tensor& v = THPVariable_Unpack(h.ptr());
        if (!fits(v, dtype, device) || v.dim() != 1 || v.numel() != width) return false;
        out[t] = v.data_ptr();
        return true;
    };
    if (!r.grouped) return one(given, 0);
    if (!PyList_Check(given.ptr()) && !PyTuple_Check(given.ptr())) return false;
    const py::sequence s = py::reinterpret_borrow<py::sequence>(given);
    if (s.size() != 4) return false;
    for (int t = 0; t < 4; t++)
        if (!one(s[t], t)) return false;
    return true;
}

at::Tensor new_tensor(at::IntArrayRef shape, c10::ScalarType dtype, c10::Device device)
{
    return at::detail::empty_cuda(shape, dtype, device, std::nullopt);
}
at::Tensor workspace(size_t bytes, c10::Device device)
{
    return bytes ? new_tensor({(int64_t)bytes}, c10::kByte, device) : at::Tensor();
}
void* place(const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
void* stream_of(c10::Device d) { return at::cuda::getCurrentCUDAStream(d.index()).stream(); }

// Sums per element: [width] or [4, width], and the addresses of the rows.
at::Tensor new_sums(const Rows& r, int64_t width, c10::ScalarType dtype, c10::Device device, void** rows)
{
    at::Tensor t = r.grouped ? new_tensor({4, width}, dtype, device) : new_tensor({width}, dtype, device);
    for (int k = 0; k < r.groups(); k++) rows[k] = static_cast<char*>(t.data_ptr()) + k * width * t.element_size();
    return t;
}

py::object layer_norm(const at::Tensor& x, py::handle gain, py::handle bias, py::handle acs, double eps)
{
    const auto dtype = x.scalar_type();
    const auto device = x.device();
    Rows r;
    const void *g[4] = {}, *b[4] = {};
    if (!device.is_cuda() || (dtype != c10::kFloat && dtype != c10::kDouble) || x.dim() != 2) return py::none();
    const int64_t n = x.size(0), w = x.size(1);
    if (w < 1 || w > kMaxWidth || !fits_rows(x, dtype, device, n, w) || !read_rows(acs, n, &r) ||
        !read_vectors(gain, r, dtype, device, w, g) || !read_vectors(bias, r, dtype, device, w, b))
        return py::none();
    const c10::cuda::CUDAGuard guard(device);
    at::Tensor y = new_tensor({n, w}, dtype, device), mean = new_tensor({n}, dtype, device), rstd = new_tensor({n}, dtype, device);
    const int rc = g_layers.norm[dtype == c10::kDouble](data(x), row_stride(x), g, b, (int)w, eps, r.acs, data(y), data(mean),
                                                        data(rstd), stream_of(device));
    if (rc) return py::int_(rc);
    return py::make_tuple(y, mean, rstd);
}

py::object layer_norm_grad(const at::Tensor& grad, const at::Tensor& x, py::handle gain, const at::Tensor& mean,
                           const at::Tensor& rstd, py::handle acs)
{
    const auto dtype = x.scalar_type();
    const auto device = x.device();
    Rows r;
    const void* g[4] = {};
    if (!device.is_cuda() || (dtype != c10::kFloat && dtype != c10::kDouble) || x.dim() != 2) return py::none();
    const int64_t n = x.size(0), w = x.size(1);
    if (w < 1 || w > kMaxWidth || !fits_rows(x, dtype, device, n, w) || !fits_rows(grad, dtype, device, n, w) ||
        !fits(mean, dtype, device) || mean.numel() != n || !fits(rstd, dtype, device) || rstd.numel() != n ||
        !read_rows(acs, n, &r) || !read_vectors(gain, r, dtype, device, w, g))
        return py::none();
    const c10::cuda::CUDAGuard guard(device);
    void *dg[4] = {}, *db[4] = {};
    at::Tensor dx = new_tensor({n, w}, dtype, device), dgain = new_sums(r, w, dtype, device, dg), dbias = new_sums(r, w, dtype, device, db);
    at::Tensor ws = workspace(g_layers.sums_bytes((int)w, r.acs, 2, (int)x.element_size()), device);
    const int rc = g_layers.norm_grad[dtype == c10::kDouble](data(grad), row_stride(grad), data(x), row_stride(x), g, data(mean),
                                                             data(rstd), (int)w, r.acs, data(dx), dg, db, place(ws),
                                                             stream_of(device));
    if (rc) return py::int_(rc);
    return py::make_tuple(dx, dgain, dbias);
}

// A checkpoint: the tensors of its parts, or one buffer that holds them one behind the other (what checkpoint_activation
// returns: an allocation costs as much host time as half a launch).
struct Kept {
    const unsigned char* codes = nullptr;
    const float *blocks = nullptr, *mean = nullptr, *rstd = nullptr;
    int64_t n = 0, width = 0;
    c10::Device device = c10::Device(c10::DeviceType::CPU);
};
int64_t kept_bytes(int64_t n, int64_t width, bool norm)
{
    return n * (g_layers.row_bytes((int)width) + 8 * g_layers.blocks((int)width) + (norm ? 8 : 0));
}
Kept kept_in(const at::Tensor& buffer, int64_t n, int64_t width, bool norm)
{
    Kept k;
    k.n = n;
    k.width = width;
    k.device = buffer.device();
    if (n == 0) return k;
    k.codes = data<unsigned char>(buffer);
    k.blocks = reinterpret_cast<const float*>(k.codes + n * g_layers.row_bytes((int)width));
    if (norm) {
        k.mean = k.blocks + 2 * n * g_layers.blocks((int)width);
        k.rstd = k.mean + n;
    }
    return k;
}
// `rows` and `normed` are the checkpoint's own, n and norm what the call is about: the size of one buffer does not tell them
// (three normalised rows of 16 columns take as many bytes as four that are not).
bool read_kept(const at::Tensor& codes, py::handle blocks_or_none, py::handle mean, py::handle rstd, int64_t rows, bool normed,
               int64_t n, int64_t width, bool norm, Kept* k)
{
    k->device = codes.device();
    if (rows != n || normed != norm || !k->device.is_cuda() || width < 1 || width > kMaxWidth || !fits(codes, c10::kByte, k->device)) return false;
    if (blocks_or_none.is_none()) {
        if (codes.dim() != 1 || codes.numel() != kept_bytes(n, width, norm)) return false;
        *k = kept_in(codes, n, width, norm);
        return true;
    }
    if (!THPVariable_Check(blocks_or_none.ptr())) return false;
    const at::Tensor& blocks = THPVariable_Unpack(blocks_or_none.ptr());
    k->n = n;
    k->width = width;
    if (codes.dim() != 2 || codes.size(0) != n || codes.size(1) != g_layers.row_bytes((int)width) || blocks.dim() != 3 ||
        !fits(blocks, c10::kFloat, k->device) || blocks.size(0) != n || blocks.size(1) != g_layers.blocks((int)width) ||
        blocks.size(2) != 2 || norm == mean.is_none() || norm == rstd.is_none())
        return false;
    k->codes = data<unsigned char>(codes);
    k->blocks = data<float>(blocks);
    if (!norm) return true;
    if (!THPVariable_Check(mean.ptr()) || !THPVariable_Check(rstd.ptr())) return false;
    const at::Tensor &m = THPVariable_Unpack(mean.ptr()), &s = THPVariable_Unpack(rstd.ptr());
    if (!fits(m, c10::kFloat, k->device) || m.numel() != n || !fits(s, c10::kFloat, k->device) || s.numel() != n) return false;
    k->mean = data<float>(m);
    k->rstd = data<float>(s);
    return true;
}

py::object checkpoint_activation(const at::Tensor& z, int act, py::handle gain, py::handle bias, py::handle acs, double eps)
{
    const auto device = z.device();
    Rows r;
    const void *g[4] = {}, *b[4] = {};
    if (!device.is_cuda() || z.scalar_type() != c10::kFloat || z.dim() != 2) return py::none();
    const int64_t n = z.size(0), w = z.size(1);
    const bool norm = !gain.is_none();
    if (w < 1 || w > kMaxWidth || !fits_rows(z, c10::kFloat, device, n, w) || !read_rows(acs, n, &r) || norm == bias.is_none() ||
        (norm && (!read_vectors(gain, r, c10::kFloat, device, w, g) || !read_vectors(bias, r, c10::kFloat, device, w, b))))
        return py::none();
    const c10::cuda::CUDAGuard guard(device);
    at::Tensor a = new_tensor({n, w}, c10::kFloat, device), buffer = new_tensor({kept_bytes(n, w, norm)}, c10::kByte, device);
    const Kept k = kept_in(buffer, n, w, norm);
    const int rc = g_layers.checkpoint(data<float>(z), row_stride(z), norm ? g : nullptr, norm ? b : nullptr, (int)w, eps, act,
                                       r.acs, data<float>(a), const_cast<unsigned char*>(k.codes), const_cast<float*>(k.blocks),
                                       const_cast<float*>(k.mean), const_cast<float*>(k.rstd), stream_of(device));
    if (rc) return py::int_(rc);
    return py::make_tuple(a, buffer);
}

py::object checkpoint_activation_grad(const at::Tensor& codes, py::handle blocks, py::handle mean, py::handle rstd,
                                      int64_t rows, bool normed, int64_t width, int act, const at::Tensor& grad,
                                      py::handle gain, py::handle bias, py::handle acs)
{
    Rows r;
    Kept k;
    const void *g[4] = {}, *b[4] = {};
    const bool norm = !gain.is_none();
    if (grad.dim() != 2 || !read_kept(codes, blocks, mean, rstd, rows, normed, grad.size(0), width, norm, &k) || !read_rows(acs, k.n, &r) ||
        norm == bias.is_none() || !fits_rows(grad, c10::kFloat, k.device, k.n, width) ||
        (norm && (!read_vectors(gain, r, c10::kFloat, k.device, width, g) || !read_vectors(bias, r, c10::kFloat, k.device, width, b))))
        return py::none();
    const c10::cuda::CUDAGuard guard(k.device);
    void *ds[4] = {}, *dg[4] = {}, *db[4] = {};
    at::Tensor dz = new_tensor({k.n, width}, c10::kFloat, k.device), dsum = new_sums(r, width, c10::kFloat, k.device, ds), dgain, dbias;
    if (norm) {
        dgain = new_sums(r, width, c10::kFloat, k.device, dg);
        dbias = new_sums(r, width, c10::kFloat, k.device, db);
    }
    at::Tensor ws = workspace(g_layers.sums_bytes((int)width, r.acs, 3, 4), k.device);
    const int rc = g_layers.checkpoint_grad(k.codes, k.blocks, k.mean, k.rstd, data<float>(grad), row_stride(grad),
                                            norm ? g : nullptr, norm ? b : nullptr, (int)width, act, r.acs, data<float>(dz), ds,
                                            dg, db, place(ws), stream_of(k.device));
    if (rc) return py::int_(rc);
    return py::make_tuple(dz, dsum, norm ? py::cast(dgain) : py::none(), norm ? py::cast(dbias) : py::none());
}

py::object checkpoint_weight_grad(const at::Tensor& codes, py::handle blocks, py::handle mean, py::handle rstd,
                                  int64_t rows, bool normed, int64_t width, int act, const at::Tensor& grad,
                                  py::handle gain, py::handle bias, py::handle acs)
{
    Rows r;
    Kept k;
    const void *g[4] = {}, *b[4] = {};
    const bool norm = !gain.is_none();
    if (grad.dim() != 2 || grad.size(1) < 1 || grad.size(1) > kMaxWidth) return py::none();
    const int64_t out = grad.size(1);
    if (!read_kept(codes, blocks, mean, rstd, rows, normed, grad.size(0), width, norm, &k) || !read_rows(acs, k.n, &r) ||
        norm == bias.is_none() || !fits_rows(grad, c10::kFloat, k.device, k.n, out) ||
        (norm && (!read_vectors(gain, r, c10::kFloat, k.device, width, g) || !read_vectors(bias, r, c10::kFloat, k.device, width, b))))
        return py::none();
    const c10::cuda::CUDAGuard guard(k.device);
    at::Tensor dw = r.grouped ? new_tensor({4, width, out}, c10::kFloat, k.device) : new_tensor({width, out}, c10::kFloat, k.device);
    void* places[4] = {};
    for (int t = 0; t < r.groups(); t++) places[t] = data<float>(dw) + t * width * out;
    at::Tensor ws = workspace(g_layers.wgrad_bytes((int)width, (int)out, r.acs), k.device);
    const int rc = g_layers.checkpoint_wgrad(k.codes, k.blocks, k.mean, k.rstd, norm ? g : nullptr, norm ? b : nullptr, (int)width,
                                             act, data<float>(grad), row_stride(grad), (int)out, r.acs, places, place(ws),
                                             stream_of(k.device));
    if (rc) return py::int_(rc);
    return py::cast(dw);
}

}  // namespace
