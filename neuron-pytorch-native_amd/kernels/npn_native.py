"""ctypes binding of libnpn_spec_verify.so (the C ABI declared in include/npn_spec_verify.h).

This is the only place Python crosses into native code. Each op module calls
``call(name, *args)``: tensors are passed as raw device pointers, ints as C ints,
and a non-zero npn_status becomes a RuntimeError carrying the library's text.
There is no fallback: if the library is missing the first call raises.
"""
import array
import ctypes
import operator
import os

import torch
from torch.autograd import forward_ad
from torch.autograd.graph import increment_version

PKG_DIR = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LIB_PATH = os.path.join(PKG_DIR, "libnpn_spec_verify.so")

_P = ctypes.c_void_p
_I = ctypes.c_int
_F = ctypes.c_float
_Z = ctypes.c_size_t

# name -> (restype, argtypes); mirrors include/npn_spec_verify.h one to one.
SIGNATURES = {
    "npn_status_string": (ctypes.c_char_p, [_I]),
    "npn_abi_version": (_I, []),
    "npn_deltanet_full_batched": (_I, [_P] * 14 + [_I, _I, _I, _P]),
    "npn_deltanet_verify": (_I, [_P, _P, _I] + [_P] * 12 + [_I, _I, _I, _I, _P]),
    "npn_deltanet_rollback": (_I, [_P] * 6 + [_I, _I, _I, _I, _P]),
    "npn_gqa_tail": (_I, [_P] * 9 + [_I, _I, _I, _P]),
    "npn_gqa_tail_workspace_size": (_Z, [_I] * 3),
    "npn_gqa_tail_split": (_I, [_P] * 9 + [_I, _I, _I, _P, _Z, _P]),
    "npn_gqa_tail_verify_workspace_size": (_Z, [_I] * 5),
    "npn_gqa_tail_verify": (_I, [_P] * 9 + [_I] * 5 + [_P, _Z, _P]),
    "npn_gqa_kv_append": (_I, [_P] * 8 + [_I] * 4 + [_P]),
    "npn_gqa_tail_verify_append": (_I, [_P] * 8 + [_I] + [_P] * 4 + [_I] * 5 + [_P, _Z, _P]),
    "npn_fp8_matmul_workspace_size": (_Z, [_I] * 3),
    "npn_fp8_matmul": (_I, [_P] * 4 + [_I] * 3 + [_P, _Z, _P]),
    "npn_accept_workspace_size": (_Z, [_I] * 3),
    "npn_accept_greedy": (_I, [_P] * 4 + [_I] * 3 + [_P, _Z, _P]),
    "npn_accept_rejection": (_I, [_P] * 5 + [_F] + [_P] * 2 + [_I] * 3 + [_P, _Z, _P]),
    "npn_accept_rejection_noalloc": (_I, [_P] * 5 + [_F] + [_P] * 2 + [_I] * 3 + [_P]),
    "npn_residual_rmsnorm": (_I, [_P] * 5 + [_I, _I, _F, _P]),
    "npn_silu_mul": (_I, [_P, _P, _I, _I, _P]),
    "npn_deltanet_split": (_I, [_P, _I] + [_P] * 4 + [_I] * 4 + [_P]),
    "npn_gqa_split": (_I, [_P, _I] + [_P] * 4 + [_I] * 4 + [_P]),
    "npn_fp8_matmul_split_k": (_I, [_I] * 3),
    "npn_fp8_matmul_plan": (_I, [_I] * 3 + [_P]),
    "npn_fp8_matmul_partials": (_I, [_P] * 3 + [_I] * 3 + [_P]),
    "npn_residual_rmsnorm_partials": (_I, [_P, _P, _I] + [_P] * 4 + [_I, _I, _F, _P]),
    "npn_residual_add_partials": (_I, [_P, _P, _I, _P, _P, _I, _I, _P]),
    "npn_deltanet_split_partials": (_I, [_P, _I, _P, _I] + [_P] * 4 + [_I] * 4 + [_P]),
    "npn_gqa_split_partials": (_I, [_P, _I, _P, _I] + [_P] * 4 + [_I] * 4 + [_P]),
    "npn_rope_rows": (_I, [_P, _P, _I] + [_P] * 3 + [_I] * 3 + [_P]),
    "npn_spec_commit": (_I, [_P] * 4 + [_I, _P]),
    "npn_deltanet_rollback_commit": (_I, [_P, _P, _I] + [_P] * 4 + [_I] * 4 + [_P]),
    "npn_fp8_matmul_argmax_groups": (_I, [_I] * 3),
    "npn_fp8_matmul_argmax": (_I, [_P] * 4 + [_I] * 3 + [_P]),
    "npn_argmax_parts": (_I, [_P, _I, _P, _P, _I, _P]),
    "npn_accept_greedy_parts": (_I, [_P, _I] + [_P] * 3 + [_I, _I, _P]),
    "npn_fp8_matmul_swiglu_workspace_size": (_Z, [_I] * 3),
    "npn_fp8_matmul_swiglu": (_I, [_P] * 4 + [_I] * 3 + [_P, _Z, _P]),
    "npn_fp8_matmul_rowmax": (_I, [_P] * 5 + [_I] * 3 + [_P]),
    "npn_accept_rejection_lm_head_workspace_size": (_Z, [_I] * 4),
    "npn_accept_rejection_lm_head": (_I, [_P] * 7 + [_F] + [_P] * 3 + [_I] * 4 + [_P, _Z, _P]),
    "npn_deltanet_chunked_workspace_size": (_Z, [_I, _I]),
    "npn_deltanet_chunked_prefill": (_I, [_P] * 8 + [_I, _I, _P, _Z, _P]),
    "npn_paged_update_blocks": (_I, [_P] * 8 + [_I] * 5 + [_P]),
    "npn_gqa_kv_append_paged": (_I, [_P] * 5 + [_I] + [_P] * 6 + [_I] * 5 + [_P]),
    "npn_gqa_tail_verify_paged_workspace_size": (_Z, [_I] * 6),
    "npn_gqa_tail_verify_paged": (_I, [_P] * 5 + [_I] + [_P] * 8 + [_I] * 7 + [_P, _Z, _P]),
    "npn_gqa_tree_verify_paged_workspace_size": (_Z, [_I] * 6),
    "npn_gqa_tree_verify_paged": (_I, [_P] * 8 + [_I] + [_P] * 10 + [_I] * 7 + [_P, _Z, _P]),
    "npn_gqa_compact_paged": (_I, [_P] * 6 + [_I] * 6 + [_P]),
    "npn_deltanet_verify_tree": (_I, [_P] * 14 + [_I] * 4 + [_P]),
    "npn_deltanet_commit_tree": (_I, [_P] * 4 + [_I, _P] + [_I] * 4 + [_P]),
    "npn_accept_tree": (_I, [_P] * 7 + [_I] * 2 + [_P]),
    "npn_sample_workspace_size": (_Z, [_I] * 2),
    "npn_sample": (_I, [_P, _I] + [_P] * 6 + [_I] * 2 + [_P, _Z, _P]),
    "npn_deltanet_full_fp8_workspace_size": (_Z, [_I] * 3),
    "npn_deltanet_full_fp8": (_I, [_P] * 19 + [_I] * 3 + [_P, _Z, _P]),
}

_INT_MAX = 2 ** 31 - 1
_lib = None
_libraries = []  # registrations last as long as these
_PLAIN = frozenset((torch.Tensor, torch.nn.Parameter, int))  # of tensors, a kernel sees all there is


def lib():
    """Load the library once and declare every entry point's C signature."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise RuntimeError(
                f"{LIB_PATH} is not built: run `make -C {PKG_DIR}` (hipcc, gfx950) first")
        handle = ctypes.CDLL(LIB_PATH)
        for name, (res, args) in SIGNATURES.items():
            fn = getattr(handle, name)
            fn.restype = res
            fn.argtypes = args
        _lib = handle
    return _lib


def _arg(a):
    if isinstance(a, torch.Tensor):
        return a.data_ptr()
    return a


def stream_of(t):
    """Handle of torch's current HIP stream on t's device (the caller's stream)."""
    return torch.cuda.current_stream(t.device).cuda_stream


def call(name, *args):
    """Call an npn_* entry point; raise RuntimeError on a non-zero status.

    Every tensor argument must sit on one device: the kernels dereference the raw pointers
    on the device of the stream they are launched on."""
    devices = {a.device for a in args if isinstance(a, torch.Tensor)}
    if len(devices) > 1:
        raise RuntimeError(f"{name}: tensor arguments span devices {sorted(map(str, devices))}")
    status = getattr(lib(), name)(*[_arg(a) for a in args])
    if status != 0:
        text = lib().npn_status_string(status).decode()
        raise RuntimeError(f"{name} failed with status {status}: {text}")


def _refuse_gradients(name, tensors):
    """Raise if a backward pass (t requires grad while gradients are on) or a forward one (t has a
    tangent) is expected through an op that has none."""
    if torch.is_grad_enabled():
        for arg, t in tensors:
            if t.requires_grad:
                raise RuntimeError(f"{arg} requires grad, but {name} has no backward pass: call it under "
                                   "torch.no_grad() or with detached inputs")
    if forward_ad._current_level >= 0:
        for arg, t in tensors:
            if forward_ad.unpack_dual(t).tangent is not None:
                raise RuntimeError(f"{arg} has a tangent, but {name} has no forward-mode derivative")


def register(qualname, schema, fake):
    """Decorator: registers the function as torch.ops.<qualname> for HIP tensors with `schema` and
    the shape propagation `fake`. Like torch.library.custom_op, minus its autograd wrapper, which
    costs 8 us a call: more than these ops' kernels take at their smallest sizes. In the wrapper's
    place a kernel above the op's own refuses inputs that a gradient is expected of, in eager, compiled
    and torch.func code alike, and calls the function at once where nothing else (a mode, a
    transform, a tensor subclass) has a part in the call; tensors that the op writes count as written."""
    namespace, name = qualname.split("::")

    def wrap(fn):
        torch.library.define(qualname, schema)
        torch.library.register_fake(qualname, fake)
        op = getattr(getattr(torch.ops, namespace), name).default
        specs = op._schema.arguments
        names = [(i, a.name) for i, a in enumerate(specs) if str(a.type) == "Tensor"]
        lists = [(i, a.name) for i, a in enumerate(specs) if str(a.type) == "List[Tensor]"]
        first = names[0][0]
        written = [i for i, a in enumerate(specs) if a.alias_info is not None and a.alias_info.is_write]

        def flat(args):
            """The arguments with the lists' tensors in the lists' places (as they are, of an op without lists)."""
            if not lists:
                return args
            out = []
            for a in args:
                if isinstance(a, list):
                    out += a
                else:
                    out.append(a)
            return out

        def count_as_written(args):
            tensors = flat([args[i] for i in written])
            try:
                increment_version(tensors)
            except RuntimeError:  # inference tensors among them, which have no version
                increment_version([t for t in tensors if not t.is_inference()])

        def below_autograd(keyset, *args):
            count_as_written(args)
            return op.redispatch(keyset & torch._C._after_ADInplaceOrView_keyset, *args)

        def autograd(*args):
            if torch._C._any_requires_grad(*args) or forward_ad._current_level >= 0:
                _refuse_gradients(qualname, [(arg, args[i]) for i, arg in names] +
                                  [(arg, t) for i, arg in lists for t in args[i]])
            plain = (args[first].is_cuda and _PLAIN.issuperset(map(type, flat(args)))
                     and torch._C._len_torch_dispatch_stack() == 0
                     and torch._C._functorch.peek_interpreter_stack() is None)
            if plain:
                if written:
                    count_as_written(args)
                return fn(*args)
            with torch._C._AutoDispatchBelowAutograd():
                return op(*args)

        torch.library.impl(qualname, "cuda", fn)
        library = torch.library.Library(namespace, "FRAGMENT")
        library.impl(name, autograd, "Autograd")
        if written:
            library.impl(name, below_autograd, "ADInplaceOrView", with_keyset=True)
        _libraries.append(library)
        return fn
    return wrap


def check_all(dev, *specs):
    """specs: (tensor, name, dtype, shape, or a number of elements in any shape). `require` for all
    of them, and that they are on `dev`."""
    index = dev.index
    for t, name, dtype, shape in specs:
        if not ((t.numel() if type(shape) is int else t.shape) == shape and t.dtype is dtype
                and t.get_device() == index and t.is_contiguous()):
            require(t, name, dtype, **({"numel": shape} if isinstance(shape, int) else {"shape": shape}))
            raise RuntimeError(f"{name} must be on {dev}, got {t.device}")


class Addresses:
    """Host array of device pointers, as an argument of `launch`."""

    def __init__(self, tensors):
        pointers = array.array("Q", map(torch.Tensor.data_ptr, tensors))
        self.pointers = pointers if pointers else array.array("Q", (0,))

    def data_ptr(self):
        return self.pointers.buffer_info()[0]


_DTYPE = operator.attrgetter("dtype")
_SHAPE = operator.attrgetter("shape")


def check_lists(dev, *specs):
    """specs: (list of tensors, name, dtype, shape, or a number of elements in any shape), one tensor a layer:
    `check_all` for each, all of a list's at once where they are as they have to be. Returns their `Addresses`."""
    out = []
    for ts, name, dtype, shape in specs:
        if ts:
            sizes = set(map(torch.Tensor.numel if type(shape) is int else _SHAPE, ts))
            if not (sizes == {shape} and set(map(_DTYPE, ts)) == {dtype}
                    and set(map(torch.Tensor.get_device, ts)) == {dev.index}
                    and all(map(torch.Tensor.is_contiguous, ts))):
                check_all(dev, *[(t, f"{name}[{i}]", dtype, shape) for i, t in enumerate(ts)])
        out.append(Addresses(ts))
    return out


def launch(dev, name, *args):
    """`call` of an entry point that ends with a stream, on dev's current stream and with dev as the
    current device; the tensors' devices have been checked. Arguments: tensors, ints and `Addresses`."""
    raw = [a if type(a) is int else a.data_ptr() for a in args]
    fn = getattr(lib(), name)
    if dev.index == torch.cuda.current_device():
        status = fn(*raw, torch._C._cuda_getCurrentRawStream(dev.index))
    else:
        with torch.cuda.device(dev):
            status = fn(*raw, torch._C._cuda_getCurrentRawStream(dev.index))
    if status != 0:
        text = lib().npn_status_string(status).decode()
        raise RuntimeError(f"{name} failed with status {status}: {text}")


def query(name, *args):
    """Call a size-query entry point and return its value; 0 (unsupported) for sizes past a C int,
    which ctypes would take modulo 2^32."""
    if max(args) > _INT_MAX:
        return 0
    return int(getattr(lib(), name)(*args))


def require(t, name, dtype, numel=None, shape=None):
    """Reference-style argument checks: CUDA device, dtype, contiguity, size."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a tensor")
    if t.device.type != "cuda":
        raise RuntimeError(f"{name} must be on a HIP device, got {t.device}")
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    if not t.is_contiguous():
        raise RuntimeError(f"{name} must be contiguous")
    if numel is not None and t.numel() != numel:
        raise RuntimeError(f"{name} must have {numel} elements, got {t.numel()} {tuple(t.shape)}")
    if shape is not None and tuple(t.shape) != tuple(shape):
        raise RuntimeError(f"{name} must have shape {tuple(shape)}, got {tuple(t.shape)}")
