"""ctypes binding of the C ABI declared in `include/difflut_b200.h`.

There is no CPU fallback: if the shared library is missing, `lib()` raises.  Every wrapper
passes raw device pointers plus the current CUDA stream and turns a negative return code
into RuntimeError (the reference's bindings raise RuntimeError through TORCH_CHECK,
difflut/nodes/cuda/efd_cuda.cpp:18-40).
"""

import contextlib
import ctypes
import os

import torch
from torch.autograd import forward_ad

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_HERE, "_lib", "libdifflut_b200.so")

# signature strings: p = pointer, l = int64, i = int, f = float, d = double; the trailing
# stream argument is implicit for every entry marked with a final 's'.
SIGNATURES = {
    "dl_thermo_rows": "ppplll s",
    "dl_thermo_pack_t": "pppllll s",
    "dl_thermo_pack_s": "pppllll s",
    "dl_thermo_pack_rows": "ppplll s",
    "dl_pack_rows_to_t": "pplllf s",
    "dl_pack_t_to_t": "ppllllf s",
    "dl_f32_rows_to_t": "pplll s",
    "dl_f32_t_to_rows": "pplll s",
    "dl_bits_t_to_rows": "pplll s",
    "dl_bits_rows_to_t": "ppllll s",
    "dl_gather_rows": "pppllll s",
    "dl_gather_rows_bwd": "ppppllll s",
    "dl_gather_rows_bwd_ell": "pplpllll s",
    "dl_unfold_rows": "ppllllllllll s",
    "dl_unfold_pack_t": "ppllllllllllfl s",
    "dl_fold_rows": "ppllllllllll s",
    "dl_fold_t": "pplllllllllll s",
    "dl_dwn_prepare": "pppllff s",
    "dl_dwn_prepare_weighted": "pppllfp s",
    "dl_dwn_prepare_full": "ppllff s",
    "dl_dwn_fwd_bits_t": "pppplll s",
    "dl_dwn_fwd_vals_t": "ppppplll s",
    "dl_dwn_bwd_tables_t": "ppplfpplll s",
    "dl_dwn_bwd_input_t": "pplfpppplll s",
    "dl_dwn_bwd_input_disjoint_t": "pplfpppllll s",
    "dl_dwn_bwd_fused_t": "pplfpllpppppppllll s",
    "dl_sum_groups": "pplll s",
    "dl_dwn_mapped_fwd": "ppplllli s",
    "dl_dwn_mapped_bwd": "pppppllll s",
    "dl_dwn_stable_mapped_bwd_input": "ppppfpllll s",
    "dl_hybrid_mapped_bwd": "pppppllll s",
    "dl_prob_fwd_t": "pppfpllll s",
    "dl_prob_fwd_groupsum_t": "pppfpppllllfl s",
    "dl_prob_bwd_t": "pppfplfpplllll s",
    "dl_hybrid_bwd_t": "pppplfpplllll s",
    "dl_seg_sum_t": "ppppll s",
    "dl_gemm_bf16_tn": "ppplllp s",
    "dl_gemm_bf16_tn_bits": "pppllllfp s",
    "dl_softmax_rows_bf16": "pfpplll s",
    "dl_softmax_rows_centered_bf16": "pfplllll s",
    "dl_row_sum_split_bf16": "pllllfl s",
    "dl_softmax_bwd_rows": "ppfpll s",
    "dl_f32_to_bf16": "pppllli s",
    "dl_bf16_transpose": "ppllll s",
    "dl_groupsum_rows": "pplllf s",
    "dl_groupsum_rows_bwd": "pplllf s",
    "dl_groupsum_t": "ppllfl s",
    "dl_dwn_fwd_groupsum_t": "ppppplllfl s",
    "dl_dwn_fwd_groupsum_s": "ppppplllfl s",
    "dl_dwn_fwd_groupsum_ce_s": "pppppppplllflll s",
    "dl_dwn_bwd_fused_s": "pplfpllpppppppllll s",
    "dl_bits_swizzle_t": "ppll s",
    "dl_dwn_fwd_groupsum_noalloc_t": "pppplllfl s",
    "dl_flip_rows": "pplfl s",
    "dl_bits_flip_t": "plllfl s",
    "dl_flip_at": "pppll s",
    "dl_bits_flip_at_t": "ppllll s",
    "dl_grad_rescale": "ppllififp s",
    "dl_p2p_barrier": "pllpl s",
    "dl_p2p_reduce_adam": "pppppplllfffff s",
    "dl_p2p_exchange_adam": "pppppppllllllllfffffl s",
    "dl_p2p_wait_done": "ppllll s",
    "dl_popcount_groupsum_t": "ppllll s",
    "dl_ce_t": "pppppllll s",
    "dl_loss_sum": "ppll s",
    "dl_adam_step": "ppppplfffff s",
    "dl_adam_advance": "pff s",
    "dl_adam_apply": "ppppplfffff s",
    "dl_adam_step_groups": "ppllpppplfffff s",
    "dl_dropout": "pplldllp s",
    "dl_counter_draw": "pp s",
    "dl_embedding_order_bytes": "llll",
    "dl_embedding": "plppllllflp s",
    "dl_embedding_bwd_scratch_bytes": "llll",
    "dl_embedding_bwd": "pppllllfp s",
    "dl_group_norm_scratch_bytes": "lllll",
    "dl_group_norm": "ppppppplllllllf s",
    "dl_group_norm_bwd_scratch_bytes": "lllll",
    "dl_group_norm_bwd": "pppppppppplllllll s",
    "dl_sample_rows": "plplpdplpdpdplll s",
}

_CT = {"p": ctypes.c_void_p, "l": ctypes.c_int64, "i": ctypes.c_int, "f": ctypes.c_float, "d": ctypes.c_double}

_lib = None


def lib():
    """Load the shared library once; raise (never fall back) when it is absent."""
    global _lib
    if _lib is not None:
        return _lib
    if not os.path.exists(LIB_PATH):
        raise RuntimeError(
            f"difflut_b200: CUDA library not found at {LIB_PATH}. Build it with "
            "`python -m difflut_b200.build` (needs nvcc, targets sm_100a). There is no CPU fallback."
        )
    handle = ctypes.CDLL(LIB_PATH)
    for name, sig in SIGNATURES.items():
        fn = getattr(handle, name)
        sig = sig.replace(" ", "")
        args = [_CT[c] for c in sig if c != "s"]
        if sig.endswith("s"):
            args.append(ctypes.c_void_p)
        fn.argtypes = args
        fn.restype = ctypes.c_int
    handle.dl_group_norm_scratch_bytes.restype = ctypes.c_int64
    handle.dl_group_norm_bwd_scratch_bytes.restype = ctypes.c_int64
    handle.dl_embedding_order_bytes.restype = ctypes.c_int64
    handle.dl_embedding_bwd_scratch_bytes.restype = ctypes.c_int64
    handle.dl_version.restype = ctypes.c_int
    handle.dl_error_string.restype = ctypes.c_char_p
    handle.dl_error_string.argtypes = [ctypes.c_int]
    handle.dl_padded_batch.restype = ctypes.c_int64
    handle.dl_padded_batch.argtypes = [ctypes.c_int64]
    handle.dl_dwn_groupsum_splits.restype = ctypes.c_int64
    handle.dl_dwn_groupsum_splits.argtypes = [ctypes.c_int64, ctypes.c_int64]
    handle.dl_dwn_bwd_groups.restype = ctypes.c_int64
    handle.dl_dwn_bwd_groups.argtypes = [ctypes.c_int64]
    handle.dl_prob_groupsum_splits.restype = ctypes.c_int64
    handle.dl_prob_groupsum_splits.argtypes = [ctypes.c_int64, ctypes.c_int64]
    handle.dl_grad_rescale_scratch_doubles.restype = ctypes.c_int64
    handle.dl_grad_rescale_scratch_doubles.argtypes = []
    handle.dl_p2p_enable_peer.restype = ctypes.c_int
    handle.dl_p2p_enable_peer.argtypes = [ctypes.c_int64]
    handle.dl_swizzled_words.restype = ctypes.c_int64
    handle.dl_swizzled_words.argtypes = [ctypes.c_int64]
    handle.dl_unfold_positions.restype = ctypes.c_int64
    handle.dl_unfold_positions.argtypes = [ctypes.c_int64] * 4
    _lib = handle
    return _lib


def available() -> bool:
    return os.path.exists(LIB_PATH)


def padded_batch(B: int) -> int:
    return (int(B) + 127) // 128 * 128


def _ptr(a):
    if a is None:
        return None
    if isinstance(a, torch.Tensor):
        if not a.is_cuda:
            raise RuntimeError("difflut_b200 kernels take CUDA tensors only (no CPU fallback)")
        if not a.is_contiguous():
            raise RuntimeError("difflut_b200 kernels take contiguous tensors")
        return a.data_ptr()
    return int(a)


# element types of the entry points that take more than fp32 (DL_DTYPE_* of the header)
DTYPE_CODES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def dtype_code(t: torch.Tensor, what: str) -> int:
    code = DTYPE_CODES.get(t.dtype)
    if code is None:
        raise TypeError(f"{what} must be float32, bfloat16 or float16, got {t.dtype}")
    return code


def require_cuda(what: str, *tensors) -> None:
    """Every given tensor is on one CUDA device (None is skipped); RuntimeError otherwise."""
    device = -1
    for t in tensors:
        if t is None:
            continue
        if not t.is_cuda:
            raise RuntimeError(f"difflut_b200.{what} runs on CUDA tensors only (no CPU fallback)")
        index = t.get_device()
        if device < 0:
            device = index
        elif index != device:
            raise RuntimeError(f"difflut_b200.{what}: tensors are on devices {device} and {index}")


def followed(*tensors) -> bool:
    """Whether autograd follows a call on these tensors, so that it has to go through its Function (None is skipped).

    A tensor with a forward-mode tangent need not require a gradient; the Function then says that it has no forward
    derivative, where a bare launch would read as a tangent of zero."""
    if forward_ad._current_level >= 0:
        return True
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return False


def refuse_tangents(*grads) -> None:
    """For a backward pass by bare launches: its incoming gradients carry no forward-mode tangents."""
    if forward_ad._current_level >= 0:
        for g in grads:
            if g is not None and forward_ad.unpack_dual(g).tangent is not None:
                raise NotImplementedError("the backward pass has no forward derivative (jvp): it cannot take a gradient that "
                                          "carries a tangent")


def once_differentiable_backward(backward):
    """A Function's backward whose result cannot be differentiated again: an error says so if it is.  torch's own wrapper
    costs several microseconds a call and only matters while a graph of the backward pass is being built."""
    from torch.autograd.function import once_differentiable

    guarded = once_differentiable(backward)

    def chosen(ctx, *grads):
        refuse_tangents(*grads)
        return guarded(ctx, *grads) if torch.is_grad_enabled() else backward(ctx, *grads)

    return chosen


_SAME_DEVICE = contextlib.nullcontext()


def device_of(t: torch.Tensor):
    """Context in which the device of CUDA tensor t is the current one (free when it already is)."""
    return _SAME_DEVICE if torch._C._cuda_getDevice() == t.get_device() else torch.cuda.device(t.device)


def host_floats(values):
    """ctypes float array for entry points that take a small HOST array; pass `ctypes.addressof(arr)`
    (keep `arr` alive until the call returns)."""
    return (ctypes.c_float * len(values))(*[float(v) for v in values])


_CALL_PLANS = {}


def _call_plan(name: str):
    """(function, argument kinds, takes a stream) of entry `name`, resolved once."""
    plan = _CALL_PLANS.get(name)
    if plan is None:
        sig = SIGNATURES[name].replace(" ", "")
        plan = (getattr(lib(), name), tuple(c for c in sig if c != "s"), sig.endswith("s"))
        _CALL_PLANS[name] = plan
    return plan


_ENTRIES = {}


def entry(name: str):
    """Entry `name` as a function of plain addresses (0 or None: null) and numbers that appends the current stream and
    raises on an error code: `call` without its conversions (a third of a short call), for callers that have checked
    device, type and contiguity of their tensors themselves."""
    found = _ENTRIES.get(name)
    if found is None:
        fn = _call_plan(name)[0]

        def found(*args):
            code = fn(*args, torch._C._cuda_getCurrentRawStream(torch._C._cuda_getDevice()))
            if code != 0:
                raise RuntimeError(f"{name} failed: {lib().dl_error_string(code).decode()} (code {code})")

        _ENTRIES[name] = found
    return found


def call(name: str, *args, stream=None):
    """Invoke C-ABI entry `name`; tensors become device pointers, the stream is appended."""
    fn, kinds, has_stream = _call_plan(name)
    if len(kinds) != len(args):
        raise TypeError(f"{name}: expected {len(kinds)} arguments, got {len(args)}")
    conv = [_ptr(a) if kind == "p" else (int(a) if kind in ("l", "i") else float(a)) for kind, a in zip(kinds, args)]
    if has_stream:
        # the current stream of the current device, without building a Stream object around it (3 us of a call)
        conv.append(torch._C._cuda_getCurrentRawStream(torch.cuda.current_device()) if stream is None else stream)
    code = fn(*conv)
    if code != 0:
        raise RuntimeError(f"{name} failed: {lib().dl_error_string(code).decode()} (code {code})")
