"""ctypes binding of the C ABI: device tensors and one method per operator.

Every method launches asynchronously on the device's stream; ``DeviceTensor.numpy()`` and
``Backend.synchronize()`` wait.  Shapes follow the reference: NCHW activations, OIHW filters,
[in, out] dense weights, all float32.
"""
import ctypes

import numpy as np

from . import _lib


class EddlHipError(RuntimeError):
    """A C ABI call returned a negative code; the text is eddlhip_last_error()."""


# bytes of an element, and the numpy type that host copies have (bfloat16 travels as its 16 bits)
_TYPES = {"float32": (4, np.float32), "int32": (4, np.int32), "bfloat16": (2, np.uint16)}


def _host(a, dtype):
    """``a`` as a contiguous array of the numpy type of ``dtype``; numbers that the type does not hold are refused where it is not float32."""
    a, kind = np.asarray(a), _TYPES[dtype][1]
    if dtype == "bfloat16" and a.size and a.dtype != np.uint16:
        raise ValueError("bfloat16 numbers travel as their 16 bits, uint16, not as %s" % a.dtype)
    if dtype == "int32" and a.size and (a.dtype.kind not in "iub" or a.min() < -2 ** 31 or a.max() >= 2 ** 31):
        raise ValueError("no int32 numbers: %s of %s" % (a.dtype, a.shape))
    return np.ascontiguousarray(a, dtype=kind)


class DeviceTensor:
    """A float32 tensor in HBM owned by this object (freed when collected)."""
    dtype = "float32"

    def __init__(self, backend, shape):
        self._describe(backend, shape)
        self.ptr = backend._malloc(self.nbytes)

    def _describe(self, backend, shape):
        self.backend = backend
        self.shape = tuple(int(d) for d in shape)
        self.size = int(np.prod(self.shape)) if len(self.shape) else 1
        self.nbytes = self.size * _TYPES[self.dtype][0]

    @property
    def address(self):
        return self.ptr

    def __del__(self):
        try:
            if getattr(self, "ptr", None):
                self.backend._free(self.ptr)
                self.ptr = None
        except Exception:
            pass

    def numpy(self):
        out = np.empty(self.shape, _TYPES[self.dtype][1])
        self.backend._check(self.backend.lib.eddlhip_memcpy_d2h(self.backend.dev, out.ctypes.data, self.address, self.nbytes))
        return out

    def copy_from(self, host):
        host = _host(host, self.dtype)
        if host.size != self.size:
            raise ValueError("size mismatch: %s vs %s" % (host.shape, self.shape))
        self.backend._check(self.backend.lib.eddlhip_memcpy_h2d(self.backend.dev, self.address, host.ctypes.data, self.nbytes))
        return self

    def reshape(self, shape):
        """A view with another shape sharing the storage (the reference's reshape_)."""
        view = object.__new__(_View)
        view.backend, view.ptr, view.nbytes, view.size = self.backend, self.ptr, self.nbytes, self.size
        view.shape = tuple(int(d) for d in shape)
        if int(np.prod(view.shape)) != self.size:
            raise ValueError("reshape changes the size")
        view._base = self  # keeps the owner alive
        return view

    def columns(self, start, stop):
        """Columns ``start`` .. ``stop - 1`` of a matrix [rows, columns], for the operators that take rows of any distance."""
        if len(self.shape) != 2 or not 0 <= start < stop <= self.shape[1]:
            raise ValueError("columns %d to %d of a tensor of shape %s" % (start, stop, self.shape))
        return Columns(self, start, stop)


class _View(DeviceTensor):
    def __del__(self):  # storage belongs to the base tensor
        pass


class TypedTensor(DeviceTensor):
    """A tensor of int32 or bfloat16 numbers, for the operators that ask for them; the others take float32 tensors only, and find no ``ptr`` here."""

    def __init__(self, backend, shape, dtype, owner=None, address=None):
        if dtype not in _TYPES or dtype == "float32":
            raise ValueError("no tensors of type %s: %s" % (dtype, ", ".join(_TYPES)))
        self.dtype = dtype
        self._describe(backend, shape)
        self._owner, self._address = owner, backend._malloc(self.nbytes) if owner is None else address

    @property
    def address(self):
        return self._address

    @property
    def ptr(self):
        raise TypeError("this operator takes float32 tensors, not %s" % self.dtype)

    def __del__(self):
        try:
            if self._owner is None and self._address:
                self.backend._free(self._address)
                self._address = None
        except Exception:
            pass

    def reshape(self, shape):
        if int(np.prod(shape)) != self.size:
            raise ValueError("reshape changes the size")
        return TypedTensor(self.backend, shape, self.dtype, self, self._address)

    def columns(self, start, stop):
        raise TypeError("columns are those of float32 matrices, not %s" % self.dtype)


class Columns:
    """Some columns of a float32 matrix: its rows lie ``ld`` floats apart (``DeviceTensor.columns``).  Not a DeviceTensor: the operators
    that walk whole tensors do not take it."""

    def __init__(self, base, start, stop):
        self._base = base  # keeps the owner alive
        self.at, self.ld, self.shape = base.ptr + 4 * start, base.shape[1], (base.shape[0], stop - start)


class PinnedArray:
    """A float32 numpy array over page-locked host memory of the library (``.array``)."""

    def __init__(self, backend, shape):
        self.backend = backend
        self.shape = tuple(int(d) for d in shape)
        n = int(np.prod(self.shape)) if len(self.shape) else 1
        self.nbytes = n * 4
        p = ctypes.c_void_p()
        backend._check(backend.lib.eddlhip_host_malloc(backend.dev, ctypes.byref(p), max(self.nbytes, 4)))
        self.ptr = p.value
        self.array = np.ctypeslib.as_array((ctypes.c_float * max(n, 1)).from_address(self.ptr))[:n].reshape(self.shape)

    def __del__(self):
        try:
            if getattr(self, "ptr", None):
                self.array = None
                self.backend.lib.eddlhip_host_free(self.backend.dev, self.ptr)
                self.ptr = None
        except Exception:
            pass


class Event:
    def __init__(self, backend):
        self.backend = backend
        h = ctypes.c_void_p()
        backend._check(backend.lib.eddlhip_event_create(backend.dev, ctypes.byref(h)))
        self.handle = h

    def record(self):
        self.backend._check(self.backend.lib.eddlhip_event_record(self.backend.dev, self.handle))
        return self

    def synchronize(self):
        self.backend._check(self.backend.lib.eddlhip_event_synchronize(self.backend.dev, self.handle))

    def elapsed_ms(self, stop):
        ms = ctypes.c_float()
        self.backend._check(self.backend.lib.eddlhip_event_elapsed_ms(self.backend.dev, self.handle, stop.handle, ctypes.byref(ms)))
        return ms.value

    def __del__(self):
        try:
            self.backend.lib.eddlhip_event_destroy(self.backend.dev, self.handle)
        except Exception:
            pass


class Graph:
    """A recorded sequence of launches (``Backend.record``); ``launch()`` replays it on the device's stream."""

    def __init__(self, backend, handle):
        self.backend, self.handle = backend, handle

    def launch(self):
        self.backend._check(self.backend.lib.eddlhip_graph_launch(self.backend.dev, self.handle))

    def __del__(self):
        try:
            if self.handle:
                self.backend.lib.eddlhip_graph_destroy(self.backend.dev, self.handle)
                self.handle = None
        except Exception:
            pass


def _ptr(t):
    return None if t is None else t.ptr


def _rows(t, what):
    """(pointer, distance of two rows, shape) of a float32 matrix or some of its columns."""
    if isinstance(t, Columns):
        return t.at, t.ld, t.shape
    if len(t.shape) != 2 or t.dtype != "float32":
        raise ValueError("%s takes float32 matrices [rows, columns], not %s %s" % (what, t.dtype, t.shape))
    return t.ptr, t.shape[1], t.shape


class Backend:
    """One device of libeddlhip.so."""

    def __init__(self, dev=0):
        self.lib = _lib.load()
        self.dev = int(dev)
        self._deferred_free = []  # pointers whose free was refused (a graph was being recorded)
        self._check(self.lib.eddlhip_init(self.dev))

    # ---- plumbing
    def _check(self, rc):
        if rc != 0:
            raise EddlHipError("%s (code %d)" % (self.lib.eddlhip_last_error().decode(), rc))

    def _malloc(self, nbytes):
        p = ctypes.c_void_p()
        self._check(self.lib.eddlhip_malloc(self.dev, max(nbytes, 4), ctypes.byref(p)))
        return p.value

    def _free(self, ptr):
        """Frees device memory; a free is refused while a graph is being recorded (``record``), so such a pointer is
        kept and freed when the recording has ended."""
        if self.lib.eddlhip_free(self.dev, ptr) != 0:
            self._deferred_free.append(ptr)

    def _free_deferred(self):
        pending, self._deferred_free = self._deferred_free, []
        for ptr in pending:
            if self.lib.eddlhip_free(self.dev, ptr) != 0:
                self._deferred_free.append(ptr)

    def workspace_bytes(self):
        n = ctypes.c_size_t()
        self._check(self.lib.eddlhip_workspace_bytes(self.dev, ctypes.byref(n)))
        return n.value

    def workspace_trim(self):
        """Releases the library's workspace; it grows back to what the calls from now on need (after a plan search)."""
        self._check(self.lib.eddlhip_workspace_trim(self.dev))

    def record(self, fn):
        """Records the launches ``fn()`` makes into a Graph instead of running them.  ``fn`` must have
        run once before (workspace at its final size) and may only launch kernels."""
        self._check(self.lib.eddlhip_graph_begin(self.dev))
        h = ctypes.c_void_p()
        try:
            fn()
        except BaseException:
            self.lib.eddlhip_graph_end(self.dev, ctypes.byref(h))  # leaves recording mode; the first error is the one to report
            if h.value:
                self.lib.eddlhip_graph_destroy(self.dev, h)
            self._free_deferred()
            raise
        rc = self.lib.eddlhip_graph_end(self.dev, ctypes.byref(h))
        self._free_deferred()
        self._check(rc)
        return Graph(self, h)

    @property
    def name(self):
        buf = ctypes.create_string_buffer(256)
        self._check(self.lib.eddlhip_device_name(self.dev, buf, 256))
        return buf.value.decode()

    def synchronize(self):
        self._check(self.lib.eddlhip_synchronize(self.dev))

    def event(self):
        return Event(self)

    # ---- batch staging (upload and download streams)
    def pinned(self, shape):
        return PinnedArray(self, shape)

    def h2d_async(self, dst, pinned, done=None):
        self._check(self.lib.eddlhip_memcpy_h2d_async(self.dev, dst.ptr, pinned.ptr, dst.nbytes, done.handle if done else None))

    def d2h_async(self, pinned, src, done=None):
        self._check(self.lib.eddlhip_memcpy_d2h_async(self.dev, pinned.ptr, src.ptr, src.nbytes, done.handle if done else None))

    def stream_wait(self, event):
        self._check(self.lib.eddlhip_stream_wait_event(self.dev, event.handle))

    def upload_wait(self, event):
        self._check(self.lib.eddlhip_upload_wait_event(self.dev, event.handle))

    def download_wait(self, event):
        self._check(self.lib.eddlhip_download_wait_event(self.dev, event.handle))

    def _probe_lib(self):
        """The device probes live in a library of their own (libeddlhip_probe.so), loaded on first use."""
        if getattr(self, "_probe", None) is None:
            from . import _lib
            self._probe = _lib.load_probe()
        return self._probe

    def probe_mfma_f32(self, vary_operands=True, launches=40):
        """Sustained fp32 MFMA rate of the device with nothing else running: (mean, best launch, worst launch) TFLOP/s."""
        mean, best, worst = ctypes.c_float(), ctypes.c_float(), ctypes.c_float()
        self._check(self._probe_lib().eddlhip_probe_mfma_f32(self.dev, int(vary_operands), launches, ctypes.byref(mean), ctypes.byref(best),
                                                    ctypes.byref(worst)))
        return mean.value, best.value, worst.value

    def probe_hbm(self, nbytes=1 << 30):
        """What plain streams over device memory sustain with nothing else running: (read, write, copy) GB/s over
        two buffers of ``nbytes`` each; copy counts bytes read plus bytes written."""
        r, w, c = ctypes.c_float(), ctypes.c_float(), ctypes.c_float()
        self._check(self._probe_lib().eddlhip_probe_hbm(self.dev, int(nbytes), ctypes.byref(r), ctypes.byref(w), ctypes.byref(c)))
        return r.value, w.value, c.value

    def empty(self, shape, dtype="float32"):
        return DeviceTensor(self, shape) if dtype == "float32" else TypedTensor(self, shape, dtype)

    def wrap(self, owner, dtype=None):
        """Device memory that another library holds (an object with ``__cuda_array_interface__``, contiguous) as a tensor, without a copy; keeps
        ``owner`` alive.  ``dtype`` says what the memory holds where the interface has no name for it ("bfloat16").

        The operators read and write it on this backend's stream: the caller sees to it that other libraries' work on the memory has ended
        by then, or is ordered before and behind it; where the interface names the null stream (1), the call waits for that.  Refused are memory of
        another device, read-only or masked memory (a tensor may be any operator's output), and an interface that names another stream, on which the
        memory may still be written."""
        spec = owner.__cuda_array_interface__
        if spec["data"][1] or spec.get("mask") is not None:
            raise ValueError("a wrapped tensor may be written: not read-only or masked memory")
        lib, device = _lib.load(), ctypes.c_int(-1)
        if spec.get("stream") is not None and (spec["stream"] != 1 or lib.hipStreamSynchronize(None) != 0):  # (of the runtime that the library runs on)
            raise ValueError("the memory may still be written on stream %s: synchronize it, and pass an object that names none" % spec["stream"])
        if lib.eddlhip_pointer_device(spec["data"][0], ctypes.byref(device)) == 0 and device.value not in (-1, self.dev):
            raise ValueError("the memory lies on device %d, not on device %d" % (device.value, self.dev))
        kind = dtype or {"<f4": "float32", "<i4": "int32"}.get(spec["typestr"])
        shape = tuple(int(d) for d in spec["shape"])
        if kind not in _TYPES or _TYPES[kind][0] != int(spec["typestr"][2:]):
            raise ValueError("no tensors of type %s over elements of %s" % (kind, spec["typestr"]))
        steps, expect = spec.get("strides"), _TYPES[kind][0]
        for d, step in reversed(list(zip(shape, steps or ()))):
            if d > 1 and step != expect:
                raise ValueError("the memory of a wrapped tensor is contiguous: shape %s, strides %s" % (shape, steps))
            expect *= d
        if kind != "float32":
            return TypedTensor(self, shape, kind, owner, spec["data"][0])
        t = object.__new__(_View)
        t._describe(self, shape)
        t._base, t.ptr = owner, spec["data"][0]
        return t

    def array(self, host, dtype="float32"):
        if dtype not in _TYPES:
            raise ValueError("no tensors of type %s: %s" % (dtype, ", ".join(_TYPES)))
        host = _host(host, dtype)
        return self.empty(host.shape, dtype).copy_from(host)

    def full(self, shape, v):
        t = DeviceTensor(self, shape)
        self.fill_(t, v)
        return t

    def set_conv_algo(self, algo):
        self._check(self.lib.eddlhip_conv2d_set_algo({"auto": 0, "mfma": 1, "direct": 2, "mfma_staged": 3, "mfma_lds": 4, "ksplit_off": 5, "ksplit_on": 6, "winograd": 7, "winograd_off": 8, "winograd_never": 9}.get(algo, algo)))

    def force_conv_plan(self, tile=-1, slices=1):
        """Override the convolution launch planner (tile 0..3, K slices; tile 4 .. 7: the Winograd forms where they apply;
        8 / 9: the upsampled-input form of a 2x2 filter; 16 .. 19: the split form; 32: the one-launch Winograd form and
        33 / 34 the upsampled-input form in the split arithmetic; 40 / 41: the split form for few tiles); tile -1 restores it."""
        self._check(self.lib.eddlhip_conv2d_force_plan(tile, slices))

    def last_conv_kernel(self):
        return self.lib.eddlhip_conv2d_last_kernel().decode()

    def conv_profile(self, collect):
        """Start (True) or stop (False) bracketing every convolution-kernel launch with events."""
        self._check(self.lib.eddlhip_conv2d_profile(int(bool(collect))))

    def conv_profile_read(self):
        """(launches, total milliseconds) of the convolution-kernel launches since collection started."""
        n, ms = ctypes.c_int(), ctypes.c_float()
        self._check(self.lib.eddlhip_conv2d_profile_read(ctypes.byref(n), ctypes.byref(ms)))
        return n.value, ms.value

    def conv_autotune(self, on=True):
        """Search the launch plans on the first call of every new convolution geometry (True), stop using what was found
        (False), or also forget it (-1)."""
        self._check(self.lib.eddlhip_conv2d_autotune(int(on)))

    def conv_tuned_plans(self):
        return self.lib.eddlhip_conv2d_tuned_plans(self.dev)

    def conv_tuned_save(self, path):
        """Write the plans found so far to a text file."""
        self._check(self.lib.eddlhip_conv2d_tuned_save(self.dev, str(path).encode()))

    def conv_tuned_load(self, path):
        """Merge a file written by ``conv_tuned_save`` into the table (used while the plan search is on)."""
        self._check(self.lib.eddlhip_conv2d_tuned_load(self.dev, str(path).encode()))

    def conv_trace(self, workgroups):
        """Per-workgroup timeline records of the next convolution launches (at most `workgroups` workgroups each);
        returns the device tensor that receives them (two floats hold one 64-bit word), or switches tracing off with 0."""
        if not workgroups:
            self._check(self.lib.eddlhip_conv2d_trace(None, 0))
            return None
        buf = self.full((int(workgroups) * 16,), 0.0)
        self._check(self.lib.eddlhip_conv2d_trace(buf.ptr, int(workgroups)))
        return buf

    # ---- operators (names follow the reference's gpu_* functions)
    def fill_(self, A, v):
        self._check(self.lib.eddlhip_fill(self.dev, A.ptr, A.size, v))

    # ---- parameter initialisation on the device (gpu_rand_*, gpu_mult / gpu_add with a scalar)
    def rand_uniform(self, A, v, seed):
        self._check(self.lib.eddlhip_rand_uniform(self.dev, A.ptr, A.size, v, seed))

    def rand_signed_uniform(self, A, v, seed):
        self._check(self.lib.eddlhip_rand_signed_uniform(self.dev, A.ptr, A.size, v, seed))

    def rand_binary(self, A, v, seed):
        self._check(self.lib.eddlhip_rand_binary(self.dev, A.ptr, A.size, v, seed))

    def rand_normal(self, A, mean, stddev, seed):
        self._check(self.lib.eddlhip_rand_normal(self.dev, A.ptr, A.size, mean, stddev, seed))

    def rand_words(self, n, seed, first_block=0, counter_hi=0):
        """The generator's raw 32-bit words as a numpy uint32 array (known-answer tests)."""
        t = self.empty((n,))
        self._check(self.lib.eddlhip_rand_words(self.dev, t.ptr, n, seed, first_block, counter_hi))
        return t.numpy().view(np.uint32)

    def mult_scalar(self, A, B, v):
        self._check(self.lib.eddlhip_mult_scalar(self.dev, A.ptr, B.ptr, A.size, v))

    def add_scalar(self, A, B, v):
        self._check(self.lib.eddlhip_add_scalar(self.dev, A.ptr, B.ptr, A.size, v))

    def conv2D(self, I, K, bias, O, sr, sc, padrt, padcl, bn=None, residual=None, relu=False, second=None, upsample=None, pool=None,
               keep=True):
        """``bn`` = (g, b, mean, var, eps) device tensors (g, b may be None) or None.  ``second``: the other half
        of the input channels as a tensor of its own (a channel Concat of ``I`` and ``second`` folded into the call).
        ``upsample`` = (rows, columns): whole factors of a nearest-neighbour UpSampling2D of ``I`` folded into the call
        (paddings and the output size then refer to the enlarged image).  ``pool`` = (pooled, indX, indY): the 2x2,
        stride-2 max-pool of the output in the same call (``eddlhip_conv2d_fwd_maxpool``); ``keep=False``: the
        unpooled output ``O`` is scratch space whose contents nobody reads afterwards."""
        N, C, H, W = I.shape
        Kf, C2, R, S = K.shape
        if second is not None:
            if tuple(second.shape) != tuple(I.shape):
                raise ValueError("the two input tensors differ in shape: %s, %s" % (I.shape, second.shape))
            C = 2 * C
        if C2 != C:
            raise ValueError("filter depth %d != input channels %d" % (C2, C))
        if O.shape[0] != N or O.shape[1] != Kf:
            raise ValueError("output shape %s does not match" % (O.shape,))
        g = b = mean = var = None
        eps = 0.0
        if bn is not None:
            g, b, mean, var, eps = bn
        tail = (K.ptr, _ptr(bias), O.ptr, N, C, H, W, Kf, R, S, sr, sc, padrt, padcl, O.shape[2], O.shape[3], _ptr(g), _ptr(b),
                _ptr(mean), _ptr(var), eps, _ptr(residual), int(relu))
        if second is not None and upsample is not None:
            raise ValueError("a two-tensor input and an upsampled input do not combine")
        if pool is not None:
            up = upsample if upsample is not None else (1, 1)
            PO, IX, IY = pool
            if tuple(PO.shape) != (N, Kf, O.shape[2] // 2, O.shape[3] // 2) or tuple(IX.shape) != tuple(PO.shape) or tuple(IY.shape) != tuple(PO.shape):
                raise ValueError("pooled shapes %s %s %s do not match output %s" % (PO.shape, IX.shape, IY.shape, O.shape))
            self._check(self.lib.eddlhip_conv2d_fwd_maxpool(self.dev, I.ptr, _ptr(second), int(up[0]), int(up[1]), *tail, PO.ptr, IX.ptr, IY.ptr,
                                                            int(bool(keep))))
        elif upsample is not None:
            self._check(self.lib.eddlhip_conv2d_fwd_upsampled(self.dev, I.ptr, int(upsample[0]), int(upsample[1]), *tail))
        elif second is None:
            self._check(self.lib.eddlhip_conv2d_fwd(self.dev, I.ptr, *tail))
        else:
            self._check(self.lib.eddlhip_conv2d_fwd_concat(self.dev, I.ptr, second.ptr, *tail))

    def cache_conv_filters(self, K):
        """Keep the kernels' repacked copy of filter tensor ``K`` (fixed between calls) in the library."""
        Kf, C, R, S = K.shape
        self._check(self.lib.eddlhip_conv2d_cache_filters(self.dev, K.ptr, Kf, C, R, S))

    def uncache_conv_filters(self, K=None):
        self._check(self.lib.eddlhip_conv2d_uncache_filters(self.dev, _ptr(K)))

    def batchnorm_inference(self, x, y, opa, gmean, gvar, g, b, variance, eps):
        N, C = x.shape[0], x.shape[1]
        rc = x.size // (N * C) if N * C else 1
        self._check(self.lib.eddlhip_batchnorm_inference(self.dev, N, C, rc, x.ptr, y.ptr, _ptr(opa), gmean.ptr, gvar.ptr, _ptr(g),
                                                         _ptr(b), variance.ptr, eps))

    def relu(self, A, B):
        self._check(self.lib.eddlhip_relu(self.dev, A.ptr, B.ptr, A.size))

    def sigmoid(self, A, B):
        self._check(self.lib.eddlhip_sigmoid(self.dev, A.ptr, B.ptr, A.size))

    def full_softmax(self, A, B, axis, stable=True):
        outer = int(np.prod(A.shape[:axis])) if axis > 0 else 1
        inner = int(np.prod(A.shape[axis + 1:])) if axis + 1 < len(A.shape) else 1
        self._check(self.lib.eddlhip_softmax(self.dev, A.ptr, B.ptr, outer, A.shape[axis], inner, int(stable)))

    def pool_out_dims(self, H, W, k, stride, pads):
        lp, lq = ctypes.c_int(), ctypes.c_int()
        self._check(self.lib.eddlhip_pool2d_out_dims(H, W, k[0], k[1], stride[0], stride[1], *pads, ctypes.byref(lp), ctypes.byref(lq)))
        return lp.value, lq.value

    def mpool2D(self, I, O, indX, indY, k, stride, pads):
        N, C, H, W = I.shape
        self._check(self.lib.eddlhip_maxpool2d(self.dev, I.ptr, O.ptr, indX.ptr, indY.ptr, N, C, H, W, k[0], k[1], stride[0],
                                               stride[1], *pads))

    def avgpool2D(self, I, O, k, stride, pads):
        N, C, H, W = I.shape
        self._check(self.lib.eddlhip_avgpool2d(self.dev, I.ptr, O.ptr, N, C, H, W, k[0], k[1], stride[0], stride[1], *pads))

    def scale(self, A, B, new_shape):
        N, C, H, W = A.shape
        self._check(self.lib.eddlhip_scale_nearest(self.dev, A.ptr, B.ptr, N, C, H, W, B.shape[2], B.shape[3], new_shape[0],
                                                   new_shape[1]))

    def concat(self, out, ts, axis):
        outer = int(np.prod(out.shape[:axis])) if axis > 0 else 1
        inner = int(np.prod(out.shape[axis + 1:])) if axis + 1 < len(out.shape) else 1
        ptrs = (ctypes.c_void_p * len(ts))(*[t.ptr for t in ts])
        ext = (ctypes.c_int * len(ts))(*[t.shape[axis] for t in ts])
        if sum(t.shape[axis] for t in ts) != out.shape[axis]:
            raise ValueError("The dimension of the output tensor is incorrect")
        self._check(self.lib.eddlhip_concat(self.dev, out.ptr, ptrs, ext, len(ts), outer, inner))

    def add(self, scA, A, scB, B, C, incC=0):
        self._check(self.lib.eddlhip_add(self.dev, scA, A.ptr, scB, B.ptr, C.ptr, incC, A.size))

    def inc(self, A, B):
        self._check(self.lib.eddlhip_inc(self.dev, A.ptr, B.ptr, A.size))

    def pad(self, A, B, pads):
        N, C, H, W = A.shape
        self._check(self.lib.eddlhip_pad(self.dev, A.ptr, B.ptr, N, C, H, W, *pads))

    def mult2D(self, A, B, C, incC=0):
        m, k = A.shape
        k2, n = B.shape
        if k != k2 or C.shape != (m, n):
            raise ValueError("mult2D shapes %s x %s -> %s" % (A.shape, B.shape, C.shape))
        self._check(self.lib.eddlhip_mult2d(self.dev, A.ptr, B.ptr, C.ptr, m, k, n, incC))

    def dense(self, A, W, bias, C, relu=False):
        """C = A W (+ bias per column) (then ReLU): LDense::forward (+ a following ReLU) in one call."""
        m, k = A.shape
        k2, n = W.shape
        if k != k2 or C.shape != (m, n):
            raise ValueError("dense shapes %s x %s -> %s" % (A.shape, W.shape, C.shape))
        self._check(self.lib.eddlhip_dense_fwd(self.dev, A.ptr, W.ptr, _ptr(bias), C.ptr, m, k, n, int(relu)))

    def sum2D_rowwise(self, A, B, C):
        self._check(self.lib.eddlhip_sum2d_rowwise(self.dev, A.ptr, B.ptr, C.ptr, A.shape[0], A.shape[1]))

    # ---- attention blocks (eddl_amd.attention holds the cache, the batch and the plan that these take)
    def rotary_axes(self, X, Y, plan, positions):
        """Rotary positions: ``X``, ``Y`` [rows, heads * head_dim] (``Y`` may be ``X``), ``plan`` a RotaryPlan, ``positions`` [rows, axes]."""
        (x, ldx, shape), (y, ldy, yshape) = _rows(X, "rotary_axes"), _rows(Y, "rotary_axes")
        if shape != yshape or shape[1] % plan.head_dim or positions.shape != (shape[0], plan.axes) or positions.dtype != "float32":
            raise ValueError("rotary_axes shapes %s -> %s, heads of %d, positions %s" % (shape, yshape, plan.head_dim, positions.shape))
        self._check(self.lib.eddlhip_rotary_axes(self.dev, x, ldx, y, ldy, shape[0], shape[1] // plan.head_dim, plan.head_dim, positions.ptr,
                                                 *plan.arguments))

    def paged_append(self, Q, K, V, Qout, cache, batch, rotary=None, positions=None):
        """Writes the new tokens' keys (turned by ``rotary``, a RotaryPlan, or as they are) and values into ``cache`` and the turned queries
        into ``Qout`` (``Q`` and ``Qout`` may be None, or the same)."""
        (k, ldk, shape), (v, ldv, vshape) = _rows(K, "paged_append"), _rows(V, "paged_append")
        q, ldq, qshape = _rows(Q, "paged_append") if Q is not None else (None, 0, (shape[0], 0))
        o, ldo, oshape = _rows(Qout, "paged_append") if Qout is not None else (None, 0, (shape[0], 0))
        if shape != vshape or shape[1] != cache.kv_heads * cache.head_dim or qshape != oshape or qshape[0] != shape[0] or qshape[1] % cache.head_dim:
            raise ValueError("paged_append shapes q %s -> %s, k %s, v %s, %d heads of %d" % (qshape, oshape, shape, vshape, cache.kv_heads, cache.head_dim))
        if (rotary is None) != (positions is None):
            raise ValueError("paged_append: a rotary plan and positions come together")
        if rotary is not None and (rotary.head_dim != cache.head_dim or positions.shape != (shape[0], rotary.axes) or positions.dtype != "float32"):
            raise ValueError("paged_append: a plan for heads of %d and positions %s for %s rows" % (rotary.head_dim, positions.shape, shape[0]))
        self._check(self.lib.eddlhip_paged_append(self.dev, q, ldq, o, ldo, k, ldk, v, ldv, shape[0], qshape[1] // cache.head_dim, cache.kv_heads,
                                                  cache.head_dim, _ptr(positions), *(rotary.arguments if rotary is not None else (0, 0, 0, None, None)),
                                                  *cache.arguments, *batch.arguments, batch.max_new))

    def paged_attention(self, Q, O, cache, batch, scale=None, causal=True, window=0):
        """Attention of the new tokens ``Q`` -> ``O`` [rows, heads * head_dim] over the cache; ``scale`` is 1 / sqrt(head_dim) unless given."""
        (q, ldq, shape), (o, ldo, oshape) = _rows(Q, "paged_attention"), _rows(O, "paged_attention")
        if shape != oshape or shape[1] % (cache.kv_heads * cache.head_dim):
            raise ValueError("paged_attention shapes %s -> %s, %d key heads of %d" % (shape, oshape, cache.kv_heads, cache.head_dim))
        self._check(self.lib.eddlhip_paged_attention(self.dev, q, ldq, o, ldo, shape[0], *cache.arguments, shape[1] // cache.head_dim, cache.kv_heads,
                                                     cache.head_dim, *batch.arguments, batch.max_new, batch.max_length,
                                                     cache.head_dim ** -0.5 if scale is None else scale, int(causal), window))

    def norm_residual(self, X, R, S, H, post=(None, None, None, 0.0), pre=(None, None, None, 0.0), gate=None, residual_scale=1.0, mod=None, shift=None,
                      group_rows=None):
        """S = residual_scale * R + gate * post(X), H = pre(S) * (1 + mod) + shift.  ``post`` and ``pre``: (kind, weight, bias, eps), kind
        None, "layer" or "rms", weight and bias [columns] or None.
        ``gate`` [groups, columns] (or one row for all), ``mod``, ``shift`` [groups, columns] belong to ``group_rows`` rows side by side (all, unless
        given).  R, S, H may be None."""
        x, ldx, shape = _rows(X, "norm_residual")
        r, ldr, rs = _rows(R, "norm_residual") if R is not None else (None, 0, shape)
        s, lds, ss = _rows(S, "norm_residual") if S is not None else (None, 0, shape)
        h, ldh, hs = _rows(H, "norm_residual") if H is not None else (None, 0, shape)
        if not rs == ss == hs == shape:
            raise ValueError("norm_residual shapes x %s, residual %s, sum %s, normed %s" % (shape, rs, ss, hs))
        if group_rows is None:
            group_rows = shape[0] or 1
        cols, grouped = shape[1], (-(-shape[0] // group_rows) if group_rows > 0 else 0) * shape[1]
        for t in (post[1], post[2], pre[1], pre[2]):
            if t is not None and (t.size != cols or t.dtype != "float32"):
                raise ValueError("norm_residual: weights %s %s for %d columns" % (t.dtype, t.shape, cols))
        for t in (gate, mod, shift):
            if t is not None and (t.dtype != "float32" or t.size < grouped and not (t is gate and t.size == cols)):
                raise ValueError("norm_residual: gate, mod or shift %s for groups of %d rows of %s" % (t.shape, group_rows, shape))
        self._check(self.lib.eddlhip_norm_residual(self.dev, x, ldx, r, ldr, residual_scale, s, lds, h, ldh, shape[0], shape[1], _NORMS[post[0]], _ptr(post[1]),
                                                   _ptr(post[2]), post[3], _ptr(gate), gate.size // shape[1] if gate is not None else 0, _NORMS[pre[0]],
                                                   _ptr(pre[1]), _ptr(pre[2]), pre[3], _ptr(mod), _ptr(shift), group_rows))

    # ---- group norm and state space blocks (eddl_amd.state_space holds the batch that the last two take)
    def group_norm(self, X, Y, groups, weight=None, bias=None, eps=1e-5, activation=None, mod=None, shift=None, image_rows=None):
        """Y = act(n (1 + mod) + shift), n the norm of ``groups`` groups of channels over the pixels of an image, its ``weight`` and ``bias`` [channels].
        ``X``, ``Y``: maps [images, channels, height, width], or rows of tokens [rows, channels], ``image_rows`` rows an image (all, unless
        given); ``Y`` may be ``X``.  ``activation`` None, "relu" (NaN stays), "relu_layer" (as ``Backend.relu``, which makes 0 of it) or "silu"; ``mod``,
        ``shift`` [images, channels] or None."""
        if len(X.shape) == 4 and len(Y.shape) == 4 and image_rows is None:
            if X.dtype != "float32" or X.shape != Y.shape:
                raise ValueError("group_norm shapes %s -> %s" % (X.shape, Y.shape))
            images, channels, pixels, last = X.shape[0], X.shape[1], X.shape[2] * X.shape[3], 0
            x, ldx, y, ldy = X.ptr, channels, Y.ptr, channels
        else:
            (x, ldx, shape), (y, ldy, yshape) = _rows(X, "group_norm"), _rows(Y, "group_norm")
            pixels, channels, last = shape[0] if image_rows is None else int(image_rows), shape[1], 1
            if shape != yshape or pixels < 0 or (shape[0] % pixels if pixels else shape[0]):
                raise ValueError("group_norm: rows %s -> %s in images of %s rows" % (shape, yshape, image_rows))
            images, pixels = (shape[0] // pixels, pixels) if shape[0] else (0, 1)
        _ints("group_norm", images, channels, pixels, groups)
        for t, size in ((weight, channels), (bias, channels), (mod, images * channels), (shift, images * channels)):
            if t is not None and (t.size != size or t.dtype != "float32"):
                raise ValueError("group_norm: weight, bias, mod or shift %s %s for %d images of %d channels" % (t.dtype, t.shape, images, channels))
        self._check(self.lib.eddlhip_group_norm(self.dev, x, ldx, y, ldy, images, channels, pixels, last, groups, _ptr(weight), _ptr(bias), eps, _ptr(mod), _ptr(shift),
                                                _activation(activation, _NORM_ACTIVATIONS)))

    def causal_conv(self, X, W, bias, Y, batch, states=None, activation=None, reverse=False):
        """The short convolution of every channel along the tokens of a ragged batch: ``X`` -> ``Y`` [rows, channels], ``W`` [channels, width],
        ``bias`` [channels] or None, ``batch`` a StateBatch, ``states`` [slots, width - 1, channels] or None (every sequence begins with its new tokens)."""
        (x, ldx, shape), (y, ldy, yshape) = _rows(X, "causal_conv"), _rows(Y, "causal_conv")
        channels = shape[1]
        if shape != yshape or len(W.shape) != 2 or W.shape[0] != channels or W.dtype != "float32" or bias is not None and (bias.size != channels or bias.dtype != "float32"):
            raise ValueError("causal_conv shapes %s -> %s, weights %s, bias %s" % (shape, yshape, W.shape, getattr(bias, "shape", None)))
        pool, slots = _pool(states, batch, W.shape[1] - 1, channels, "causal_conv")
        _ints("causal_conv", *shape, W.shape[1], slots)
        self._check(self.lib.eddlhip_causal_conv(self.dev, x, ldx, W.ptr, _ptr(bias), y, ldy, shape[0], channels, W.shape[1], _activation(activation), 1 if reverse else 0,
                                                 pool, slots, *batch.arguments))

    def selective_scan(self, X, dt, A, B, C, Y, batch, states=None, skip=None, gate=None, dt_bias=None, softplus=True, reverse=False):
        """The selective scan along the tokens of a ragged batch: ``X``, ``dt``, ``Y`` and ``gate`` (or None) [rows, channels], ``A`` [channels, n], ``B`` and ``C``
        [rows, groups * n], ``skip`` and ``dt_bias`` [channels] or None, ``batch`` a StateBatch, ``states`` [slots, channels, n] or None (every
        sequence begins with its new tokens)."""
        (x, ldx, shape), (d, lddt, dshape), (y, ldy, yshape) = _rows(X, "selective_scan"), _rows(dt, "selective_scan"), _rows(Y, "selective_scan")
        (b, ldb, bshape), (c, ldc, cshape) = _rows(B, "selective_scan"), _rows(C, "selective_scan")
        g, ldg, gshape = _rows(gate, "selective_scan") if gate is not None else (None, 0, shape)
        rows, channels = shape
        n = A.shape[1] if len(A.shape) == 2 and A.dtype == "float32" else 0
        if not shape == dshape == yshape == gshape or bshape != cshape or bshape[0] != rows or A.shape[0] != channels or not n or bshape[1] % n:
            raise ValueError("selective_scan shapes x %s, dt %s, gate %s -> %s, A %s, B %s, C %s" % (shape, dshape, gshape, yshape, A.shape, bshape, cshape))
        if skip is not None and (skip.size != channels or skip.dtype != "float32") or dt_bias is not None and (dt_bias.size != channels or dt_bias.dtype != "float32"):
            raise ValueError("selective_scan: skip or dt_bias not float32 numbers of %d channels" % channels)
        pool, slots = _pool(states, batch, channels, n, "selective_scan")
        _ints("selective_scan", *shape, bshape[1], slots)
        self._check(self.lib.eddlhip_selective_scan(self.dev, x, ldx, d, lddt, A.ptr, b, ldb, c, ldc, None if skip is None else skip.ptr, g, ldg,
                                                    None if dt_bias is None else dt_bias.ptr, y, ldy, rows, channels, n, bshape[1] // n, 1 if softplus else 0,
                                                    1 if reverse else 0, pool, slots, *batch.arguments))


_NORMS = {None: 0, "layer": 1, "rms": 2}
_ACTIVATIONS = {None: 0, "relu": 1, "silu": 2}
_NORM_ACTIVATIONS = dict(_ACTIVATIONS, relu_layer=4)


def _activation(name, known=_ACTIVATIONS):
    if name not in known:
        raise ValueError("no activation %r: %s" % (name, ", ".join(map(repr, known))))
    return known[name]


def _ints(what, *sizes):
    """Refuses sizes that the library's ints do not hold: they would arrive as other ones."""
    if any(not -2 ** 31 <= size < 2 ** 31 for size in sizes):
        raise ValueError("%s: a size of %s is out of range" % (what, max(sizes, key=abs)))


def _pool(states, batch, rows, cols, what):
    """(pointer, slots) of a pool of states [rows, cols]."""
    if states is None:
        return None, 0
    shape = states.shape
    if len(shape) != 3 or shape[1] != rows or shape[2] != cols or states.dtype != "float32" or batch.slots is None:
        raise ValueError("%s: states are float32 [slots, %d, %d] with a batch that names lengths and slots, not %s %s" % (what, rows, cols, states.dtype, shape))
    return states.ptr, shape[0]
