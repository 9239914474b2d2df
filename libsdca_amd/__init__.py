"""libsdca_amd - MI355X (gfx950) batched prox operators and evaluation pass.

Python host side of the C ABI in include/sdca_hip.h.  The functions keep the
names and argument meaning of libsdca's batched C++ API
(include/sdca/prox/*.h, the `dim` overloads) and of the Matlab front end's
operator table (src/matlab/mex_prox.cpp:145-172):

    prox_knapsack_eq(dim, A, lo=0, hi=1, rhs=1)
    prox_knapsack_le(dim, A, lo=0, hi=1, rhs=1)
    prox_topk_simplex(dim, A, k=1, rhs=1)
    prox_topk_cone(dim, A, k=1)
    prox_entropy(dim, A, hi=1, rhs=1)
    prox_entropy_norm(dim, A, hi=1, rhs=1)
    prox_topk_entropy(dim, A, k=1)
    prox_two_simplex(dim, p, A, rhs=1)
    prox_knapsack_le_biased(dim, A, lo=0, hi=1, rhs=1, rho=1)
    prox_topk_simplex_biased(dim, A, k=1, rhs=1, rho=1)
    prox_topk_cone_biased(dim, A, k=1, rho=1)
    prox_topk_entropy_biased(dim, A, k=1, alpha=1)
    prox_two_simplex_sort(dim, p, A, rhs=1)
    prox_two_entropy(dim, p, A, alpha=1)
    lambert_w_exp(A)

and the answers of a trained model, which the reference does not have:

    quantize_i8(A)
    scores_i8(X, W, w_scales)
    sample(S, u, temperature=1, top_k=0, top_p=1, min_p=0)
    log_probs(S, labels, temperature=1, top=0)
    log_probs_grad(S, labels, g)
    scores_adapted(X, W, w_scales, A, B, index, scale=1)
    scores_adapted_grad(G, X, A, B, index, scale=1)

`A` holds n columns of length dim, contiguous (a C-contiguous (n, dim) array
or tensor, i.e. the column-major dim x n matrix of the reference).  A torch
CUDA tensor is processed in place on the device (stream-ordered on torch's
current stream); a numpy array is staged through device memory and updated in
place.  There is no CPU fallback: without the built HIP library every call
raises.
"""
import ctypes
import os
import sys

import numpy as np

__all__ = [
    "SdcaError", "library", "prox", "prox_knapsack_eq", "prox_knapsack_le",
    "prox_topk_simplex", "prox_topk_cone", "prox_entropy", "prox_entropy_norm",
    "prox_topk_entropy", "prox_two_simplex", "prox_knapsack_le_biased",
    "prox_topk_simplex_biased", "prox_topk_cone_biased", "prox_topk_entropy_biased",
    "prox_two_simplex_sort", "prox_two_entropy", "lambert_w_exp", "OPS", "F32", "F64",
    "OBJECTIVES", "objective", "scores", "eval_features", "eval_kernel", "eval_scores",
    "recompute_primal", "epoch_order", "epoch_features", "epoch_kernel", "BRANCHES",
    "quantize_i8", "scores_i8", "sample", "log_probs", "log_probs_grad",
    "scores_adapted", "scores_adapted_grad",
]

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "libsdca_hip.so")

F32, F64, LONG_DOUBLE = 0, 1, 2
HOST_PTR = 1
OPS = {
    "knapsack_eq": 0, "knapsack": 0, "knapsack_le": 1, "topk_simplex": 2,
    "topk_cone": 3, "entropy": 4, "entropy_norm": 5, "topk_entropy": 6,
    "two_simplex": 7, "lambert_w_exp": 8, "knapsack_le_biased": 9,
    "topk_simplex_biased": 10, "topk_cone_biased": 11,
    "topk_entropy_biased": 12, "two_simplex_sort": 13, "two_entropy": 14,
}
# sdca_prox_branch (include/sdca_hip.h): the return of the threshold
# function that produced a record.
BRANCHES = {
    0: "search", 1: "inactive", 2: "zero", 3: "constant", 4: "knapsack", 5: "scan",
    6: "default", 7: "u_empty", 8: "u_grown", 9: "below_rhs",
}
STATUS = {
    0: "OK", 1: "ARG_NULL", 2: "ARG_RANGE", 3: "PRECISION", 4: "NOT_IMPLEMENTED",
    5: "OUT_OF_MEMORY", 6: "HIP", 7: "PROX", 8: "LABELS",
}


class SdcaError(RuntimeError):
    """A failed C ABI call; .status is the sdca_status code."""

    def __init__(self, status, message):
        super().__init__(f"{STATUS.get(status, status)}: {message}")
        self.status = status


class ProxParams(ctypes.Structure):
    _fields_ = [("lo", ctypes.c_double), ("hi", ctypes.c_double),
                ("rhs", ctypes.c_double), ("rho", ctypes.c_double),
                ("alpha", ctypes.c_double), ("k", ctypes.c_int64),
                ("p", ctypes.c_int64)]


class Thresholds(ctypes.Structure):
    _fields_ = [("t", ctypes.c_double), ("lo", ctypes.c_double), ("hi", ctypes.c_double)]


class Objective(ctypes.Structure):
    _fields_ = [("kind", ctypes.c_int32), ("reserved", ctypes.c_int32),
                ("c", ctypes.c_double), ("gamma", ctypes.c_double), ("k", ctypes.c_int64)]


class EvalRecord(ctypes.Structure):
    _fields_ = [("primal", ctypes.c_double), ("dual", ctypes.c_double),
                ("primal_loss", ctypes.c_double), ("dual_loss", ctypes.c_double),
                ("primal_regularizer", ctypes.c_double),
                ("dual_regularizer", ctypes.c_double), ("rank_loss", ctypes.c_double)]


class SampleParams(ctypes.Structure):
    _fields_ = [("temperature", ctypes.c_double), ("top_p", ctypes.c_double),
                ("min_p", ctypes.c_double), ("top_k", ctypes.c_int64)]


class SampleColumns(ctypes.Structure):
    _fields_ = [("temperature", ctypes.c_void_p), ("top_p", ctypes.c_void_p),
                ("min_p", ctypes.c_void_p), ("top_k", ctypes.c_void_p)]


class Adapters(ctypes.Structure):
    _fields_ = [("count", ctypes.c_int64), ("rank", ctypes.c_int64), ("A", ctypes.c_void_p),
                ("B", ctypes.c_void_p), ("index", ctypes.c_void_p), ("scale", ctypes.c_void_p),
                ("factor", ctypes.c_double)]


# Objectives of the evaluation pass, named after the reference's makers
# (objective.h:55-160: make_objective_l2_hinge_topk, ...).
OBJECTIVES = {
    "l2_hinge_topk": 0, "l2_hinge_topk_smooth": 1, "l2_topk_hinge": 2,
    "l2_topk_hinge_smooth": 3, "l2_entropy": 4, "l2_entropy_topk": 5,
    "l2_multilabel_hinge": 6, "l2_multilabel_hinge_smooth": 7,
    "l2_multilabel_entropy": 8,
}


def objective(name, c=1.0, gamma=1.0, k=1):
    """An objective for eval_features / eval_scores (c = 1 / (lambda n))."""
    return (name, float(c), float(gamma), int(k))


_lib = None


def library():
    """The loaded libsdca_hip.so (raises if it was not built)."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise SdcaError(6, f"{LIB_PATH} is missing: build it with "
                               "`python -c 'import __graft_entry__ as g; g.build()'`")
        # torch ships its own HIP runtime under the same soname; loading torch
        # first makes the library bind to it, so that a process that uses both
        # holds one runtime (two runtimes in one process leave the second
        # without a device).
        try:
            import torch  # noqa: F401
        except ImportError:
            pass
        lib = ctypes.CDLL(LIB_PATH)
        lib.sdca_prox.restype = ctypes.c_int
        lib.sdca_prox_with_sets.restype = ctypes.c_int
        lib.sdca_prox.argtypes = [
            ctypes.c_int, ctypes.c_int, ctypes.c_int, ctypes.c_int64, ctypes.c_int64,
            ctypes.c_void_p, ctypes.c_void_p, ctypes.POINTER(ProxParams), ctypes.c_void_p,
            ctypes.c_void_p, ctypes.c_uint, ctypes.c_void_p]
        i32, i64, ptr, u32 = ctypes.c_int, ctypes.c_int64, ctypes.c_void_p, ctypes.c_uint
        lib.sdca_quantize_i8.argtypes = [i32, i64, i64, ptr, i64, ptr, i64, ptr, u32, ptr]
        lib.sdca_scores_i8.argtypes = [i32, i32, i64, i64, i64, ptr, i64, ptr, ptr, i64, ptr, ptr,
                                       i64, u32, ptr]
        lib.sdca_sample.argtypes = [i32, i64, i64, ptr, i64, ptr, ctypes.POINTER(SampleParams),
                                    ctypes.POINTER(SampleColumns), ptr, ptr, ptr, u32, ptr]
        f64, size = ctypes.c_double, ctypes.c_size_t
        lib.sdca_log_probs_work.argtypes, lib.sdca_log_probs_work.restype = [i32, i64, i64, i64], size
        lib.sdca_log_probs.argtypes = [i32, i64, i64, ptr, i64, ptr, f64, i64, ptr, ptr, ptr, ptr, ptr,
                                       ptr, u32, ptr]
        lib.sdca_log_probs_grad_work.argtypes, lib.sdca_log_probs_grad_work.restype = [i32, i64, i64, ptr], size
        lib.sdca_log_probs_grad.argtypes = [i32, i64, i64, ptr, i64, ptr, ptr, ptr, ptr, f64, ptr, i64,
                                            ptr, ptr, u32, ptr]
        ads = ctypes.POINTER(Adapters)
        lib.sdca_scores_adapted_work.argtypes = [i32, i64, i64, i64, ptr, i64, i64, i64]
        lib.sdca_scores_adapted_work.restype = size
        lib.sdca_scores_adapted.argtypes = [i32, i32, i64, i64, i64, ptr, i64, ptr, i64, ptr, ads, ptr, i64,
                                            ptr, u32, ptr]
        lib.sdca_scores_adapted_grad_work.argtypes = [i32, i32, i64, i64, i64, i64, i64]
        lib.sdca_scores_adapted_grad_work.restype = size
        lib.sdca_scores_adapted_grad.argtypes = [i32, i32, i64, i64, i64, ptr, i64, ptr, i64, ads, ptr, ptr,
                                                 ptr, u32, ptr]
        lib.sdca_last_error.restype = ctypes.c_char_p
        lib.sdca_abi_version.restype = ctypes.c_int
        _lib = lib
    return _lib


def check(rc):
    if rc != 0:
        msg = library().sdca_last_error().decode(errors="replace")
        raise SdcaError(rc, msg)


_torch_types = {}  # a small call asks some forty times


def _is_torch(x):
    t = type(x)
    known = _torch_types.get(t)
    if known is None:
        known = _torch_types[t] = t.__module__.startswith("torch")
    return known


def _dtype_code(x):
    if _is_torch(x):
        import torch
        return {torch.float32: F32, torch.float64: F64}.get(x.dtype, -1)
    return {np.dtype(np.float32): F32, np.dtype(np.float64): F64}.get(x.dtype, -1)


def _need(x, name, shape, like):
    """Checks that x can be handed to the C ABI beside `like`: the same kind
    (numpy array, or tensor on like's device), like's element type, the given
    shape, contiguous.  The library reads and writes through raw pointers, so
    a mismatch here would otherwise become an out-of-bounds access."""
    if x is None:
        return
    if _is_torch(x) != _is_torch(like):
        raise SdcaError(2, f"{name}: numpy arrays and torch tensors cannot be mixed in one call")
    if _is_torch(x):
        if x.device != like.device:
            raise SdcaError(2, f"{name} is on {x.device}, expected {like.device}")
        contiguous = x.is_contiguous()
    else:
        contiguous = x.flags.c_contiguous
    if x.dtype != like.dtype:
        raise SdcaError(3, f"{name} has element type {x.dtype}, expected {like.dtype}")
    if tuple(int(v) for v in x.shape) != tuple(shape):
        raise SdcaError(2, f"{name} has shape {tuple(x.shape)}, expected {tuple(shape)}")
    if not contiguous:
        raise SdcaError(2, f"{name} must be contiguous")


def _label_arrays(labels, offsets, n, like):
    """int64 label (and CSR offset) arrays of the kind of `like`, with the
    lengths the C ABI reads: n labels, or n + 1 offsets and offsets[n] labels."""
    if _is_torch(like):
        import torch
        lab = torch.as_tensor(labels, dtype=torch.int64, device=like.device).contiguous().reshape(-1)
        off = None if offsets is None else torch.as_tensor(
            offsets, dtype=torch.int64, device=like.device).contiguous().reshape(-1)
    else:
        lab = np.ascontiguousarray(labels, dtype=np.int64).reshape(-1)
        off = None if offsets is None else np.ascontiguousarray(offsets, dtype=np.int64).reshape(-1)
    if off is None:
        if lab.shape[0] != n:
            raise SdcaError(8, f"{lab.shape[0]} labels for {n} examples")
    else:
        if off.shape[0] != n + 1:
            raise SdcaError(8, f"{off.shape[0]} offsets for {n} examples (need n + 1)")
        if int(off[-1]) != lab.shape[0]:
            raise SdcaError(8, f"offsets end at {int(off[-1])} but {lab.shape[0]} labels are given")
        if int(off[0]) != 0:
            raise SdcaError(8, f"offsets start at {int(off[0])}, not 0")
        if n > 0 and bool((off[1:] < off[:-1]).any()):
            raise SdcaError(8, "offsets decrease")
    return lab, off


def _stream_ptr():
    import torch
    return ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)


def prox(op, A, out=None, result=None, lo=0.0, hi=1.0, rhs=1.0, rho=1.0,
         alpha=1.0, k=1, p=1, col_p=None, thresholds=False, check_col_p=True, sets=False):
    """Batched prox over the rows of A (each row is one column of the
    reference's dim x n matrix).  Returns out (A itself when out is None) and,
    with thresholds=True, an (n, 3) (or (2n, 3) for the two-block operators) array of
    (t, lo, hi) per column/block; with sets=True also an int64 array of the
    same shape of (n_hi, n_mid, branch) per record (sdca_prox_with_sets: the
    sizes of the record's set at hi and free set, and its sdca_prox_branch).
    A device col_p is checked against [1, dim - 1] here (one
    synchronisation) unless check_col_p=False, for callers that validated it
    already (the kernels clamp it into range either way)."""
    lib = library()
    code = OPS[op] if isinstance(op, str) else int(op)
    data = _dtype_code(A)
    if data < 0:
        raise SdcaError(3, f"unsupported element type {A.dtype}")
    res = data if result is None else ({"float": F32, "single": F32, "double": F64,
                                        "long double": LONG_DOUBLE}.get(result, result))
    if A.ndim == 1:
        A = A.reshape(1, -1)
        if out is not None:
            out = out.reshape(1, -1)
    if A.ndim != 2:
        raise SdcaError(2, f"A must be 1-D or 2-D (got {A.ndim} dimensions)")
    n, m = int(A.shape[0]), int(A.shape[1])
    if out is None:
        out = A
    _need(A, "A", (n, m), A)
    _need(out, "out", (n, m), A)
    params = ProxParams(lo, hi, rhs, rho, alpha, int(k), int(p))
    nthr = 2 * n if code in (OPS["two_simplex"], OPS["two_simplex_sort"],
                             OPS["two_entropy"]) else n
    if _is_torch(A):
        import torch
        if not A.is_cuda:
            raise SdcaError(2, "torch inputs must be CUDA tensors")
        thr = torch.zeros((nthr, 3), dtype=torch.float64, device=A.device) if thresholds else None
        # sdca_prox_sets is {int64, int64, int32, int32}: the third int64 word
        # reads as the branch (the reserved half is 0).
        st = torch.zeros((nthr, 3), dtype=torch.int64, device=A.device) if sets else None
        cp = None
        if col_p is not None:
            cp = torch.as_tensor(col_p, dtype=torch.int64, device=A.device).contiguous().reshape(-1)
            if cp.shape[0] != n:
                raise SdcaError(2, f"col_p has {cp.shape[0]} entries for {n} columns")
            if check_col_p and n > 0:
                lo_p, hi_p = torch.aminmax(cp)
                if int(lo_p) < 1 or int(hi_p) > m - 1:
                    raise SdcaError(2, f"col_p must lie in [1, {m - 1}] (got {int(lo_p)}..{int(hi_p)})")
        if st is not None:
            check(lib.sdca_prox_with_sets(
                code, data, res, ctypes.c_int64(m), ctypes.c_int64(n), ctypes.c_void_p(A.data_ptr()),
                ctypes.c_void_p(out.data_ptr()), ctypes.byref(params),
                ctypes.c_void_p(cp.data_ptr() if cp is not None else None),
                ctypes.c_void_p(thr.data_ptr() if thr is not None else None),
                ctypes.c_void_p(st.data_ptr()), ctypes.c_uint(0), _stream_ptr()))
        else:
            check(lib.sdca_prox(code, data, res, m, n, A.data_ptr(), out.data_ptr(),
                                ctypes.byref(params), cp.data_ptr() if cp is not None else None,
                                thr.data_ptr() if thr is not None else None, 0, _stream_ptr()))
        return _prox_result(out, thr, st, thresholds, sets)
    thr = np.zeros((nthr, 3), dtype=np.float64) if thresholds else None
    st = np.zeros((nthr, 3), dtype=np.int64) if sets else None
    cp = None if col_p is None else np.ascontiguousarray(col_p, dtype=np.int64).reshape(-1)
    if cp is not None and cp.shape[0] != n:
        raise SdcaError(2, f"col_p has {cp.shape[0]} entries for {n} columns")
    if st is not None:
        check(lib.sdca_prox_with_sets(
            code, data, res, ctypes.c_int64(m), ctypes.c_int64(n), ctypes.c_void_p(A.ctypes.data),
            ctypes.c_void_p(out.ctypes.data), ctypes.byref(params),
            ctypes.c_void_p(cp.ctypes.data if cp is not None else None),
            ctypes.c_void_p(thr.ctypes.data if thr is not None else None),
            ctypes.c_void_p(st.ctypes.data), ctypes.c_uint(HOST_PTR), None))
    else:
        check(lib.sdca_prox(code, data, res, m, n, A.ctypes.data, out.ctypes.data,
                            ctypes.byref(params), cp.ctypes.data if cp is not None else None,
                            thr.ctypes.data if thr is not None else None, HOST_PTR, None))
    return _prox_result(out, thr, st, thresholds, sets)


def _prox_result(out, thr, st, thresholds, sets):
    res = (out,) + ((thr,) if thresholds else ()) + ((st,) if sets else ())
    return res if len(res) > 1 else out


def _rows(dim, A):
    if A.ndim == 2 and A.shape[1] == dim:
        return A
    return A.reshape(-1, dim)


# The reference's batched overloads (`dim` first).  Result follows the
# reference: deduced from the floating parameter's type in C++; here the
# element type unless `result` is given.  prox_topk_cone, prox_topk_entropy
# and prox_topk_entropy_biased default to double, as their C++ templates do
# (topk_cone.h:187-199, topk_entropy.h:106-118, topk_entropy_biased.h:302-315).
def prox_knapsack_eq(dim, A, lo=0.0, hi=1.0, rhs=1.0, result=None):
    return prox("knapsack_eq", _rows(dim, A), lo=lo, hi=hi, rhs=rhs, result=result)


def prox_knapsack_le(dim, A, lo=0.0, hi=1.0, rhs=1.0, result=None):
    return prox("knapsack_le", _rows(dim, A), lo=lo, hi=hi, rhs=rhs, result=result)


def prox_topk_simplex(dim, A, k=1, rhs=1.0, result=None):
    return prox("topk_simplex", _rows(dim, A), k=k, rhs=rhs, result=result)


def prox_topk_cone(dim, A, k=1, result="double"):
    return prox("topk_cone", _rows(dim, A), k=k, result=result)


def prox_entropy(dim, A, hi=1.0, rhs=1.0, result=None):
    return prox("entropy", _rows(dim, A), hi=hi, rhs=rhs, result=result)


def prox_entropy_norm(dim, A, hi=1.0, rhs=1.0, result=None):
    return prox("entropy_norm", _rows(dim, A), hi=hi, rhs=rhs, result=result)


def prox_topk_entropy(dim, A, k=1, result="double"):
    return prox("topk_entropy", _rows(dim, A), k=k, result=result)


def prox_two_simplex(dim, p, A, rhs=1.0, result=None):
    return prox("two_simplex", _rows(dim, A), p=p, rhs=rhs, result=result)


def prox_knapsack_le_biased(dim, A, lo=0.0, hi=1.0, rhs=1.0, rho=1.0, result=None):
    return prox("knapsack_le_biased", _rows(dim, A), lo=lo, hi=hi, rhs=rhs, rho=rho, result=result)


def prox_topk_simplex_biased(dim, A, k=1, rhs=1.0, rho=1.0, result=None):
    return prox("topk_simplex_biased", _rows(dim, A), k=k, rhs=rhs, rho=rho, result=result)


def prox_topk_cone_biased(dim, A, k=1, rho=1.0, result=None):
    return prox("topk_cone_biased", _rows(dim, A), k=k, rho=rho, result=result)


def prox_topk_entropy_biased(dim, A, k=1, alpha=1.0, result="double"):
    return prox("topk_entropy_biased", _rows(dim, A), k=k, alpha=alpha, result=result)


def prox_two_entropy(dim, p, A, alpha=1.0, result=None):
    """Batched form of prox_two_entropy(p, first, last, aux, alpha)
    (two_entropy.h:280-292), which the reference has per column only."""
    return prox("two_entropy", _rows(dim, A), p=p, alpha=alpha, result=result)


def prox_two_simplex_sort(dim, p, A, rhs=1.0, result=None):
    return prox("two_simplex_sort", _rows(dim, A), p=p, rhs=rhs, result=result)


def lambert_w_exp(A):
    """Elementwise W(exp(x)) in place (apply(dim, ..., lambert_w_exp_map))."""
    return prox("lambert_w_exp", A if A.ndim == 2 else A.reshape(1, -1))


# ---------------------------------------------------------------------------
# Evaluation pass (evaluate_dataset, eval.h:15-51, for feature input).
# X: (n, d) examples, W: (m, d) classes, S/A: (n, m); all C-contiguous, i.e.
# the reference's column-major d x n, d x m and m x n matrices.
# ---------------------------------------------------------------------------
def _objs(objs):
    arr = (Objective * len(objs))()
    for i, (name, c, gamma, k) in enumerate(objs):
        arr[i] = Objective(OBJECTIVES[name], 0, c, gamma, k)
    return arr


def _ptr(x):
    if x is None:
        return None
    return x.data_ptr() if _is_torch(x) else x.ctypes.data


def scores(X, W, out=None):
    """S = X W^T (scores of every example for every class)."""
    lib = library()
    n, d = int(X.shape[0]), int(X.shape[1])
    m = int(W.shape[0])
    data = _dtype_code(X)
    _need(X, "X", (n, d), X)
    _need(W, "W", (m, d), X)
    _need(out, "out", (n, m), X)
    if _is_torch(X):
        import torch
        S = out if out is not None else torch.empty((n, m), dtype=X.dtype, device=X.device)
        check(lib.sdca_scores(data, ctypes.c_int64(d), ctypes.c_int64(m), ctypes.c_int64(n),
                              ctypes.c_void_p(X.data_ptr()), ctypes.c_void_p(W.data_ptr()),
                              ctypes.c_void_p(S.data_ptr()), ctypes.c_uint(0), _stream_ptr()))
        return S
    S = out if out is not None else np.zeros((n, m), dtype=X.dtype)
    check(lib.sdca_scores(data, ctypes.c_int64(d), ctypes.c_int64(m), ctypes.c_int64(n),
                          ctypes.c_void_p(X.ctypes.data), ctypes.c_void_p(W.ctypes.data),
                          ctypes.c_void_p(S.ctypes.data), ctypes.c_uint(HOST_PTR), None))
    return S


def epoch_order(n, epoch):
    """The reference solver's example order for epoch `epoch` (0-based) of a
    solve over n examples (solver.h:75-112): int64 numpy array."""
    lib = library()
    out = np.zeros(int(n), dtype=np.int64)
    lib.sdca_epoch_order.restype = ctypes.c_int
    rc = lib.sdca_epoch_order(ctypes.c_int64(int(n)), ctypes.c_int64(int(epoch)),
                              ctypes.c_void_p(out.ctypes.data))
    if rc != 0:
        raise SdcaError(rc, lib.sdca_last_error().decode())
    return out


def epoch_features(obj, X, W, A, labels, order=None, norms=None, result=None, offsets=None):
    """One SDCA epoch on feature input (update_variables for each example of
    `order`, update.h:52-85) for an objective (name, c, gamma, k):
    X (n, d), W (m, d), A (n, m), W and A updated in place and returned.
    CUDA tensors run on torch's current stream; numpy arrays (C-contiguous,
    X's dtype) go through the host-staging path.  order: example indices
    (None: 0..n-1), e.g. epoch_order(n, e); norms: (n,) squared row norms of
    X, or None; offsets: (n + 1,) CSR row starts into labels for the
    multilabel objectives."""
    lib = library()
    n, d = int(X.shape[0]), int(X.shape[1])
    m = int(W.shape[0])
    objarr = _objs([obj])
    lib.sdca_epoch_features.restype = ctypes.c_int
    if _is_torch(X):
        if not X.is_cuda:
            raise SdcaError(2, "epoch_features takes CUDA tensors or numpy arrays")
        import torch
        _need(X, "X", (n, d), X)
        _need(W, "W", (m, d), X)
        _need(A, "A", (n, m), X)
        _need(norms, "norms", (n,), X)
        od = None
        if order is not None:
            od = torch.as_tensor(order, dtype=torch.int64, device=X.device).contiguous().reshape(-1)
        flags, stream = 0, _stream_ptr()
        ptr = _ptr
    else:
        for name, a, shape in (("X", X, (n, d)), ("W", W, (m, d)), ("A", A, (n, m)),
                               ("norms", norms, (n,))):
            if a is None:
                continue
            if (not isinstance(a, np.ndarray) or a.dtype != X.dtype or tuple(a.shape) != shape
                    or not a.flags.c_contiguous):
                raise SdcaError(2, f"{name}: expected a C-contiguous {X.dtype} array {shape}")
        od = None if order is None else np.ascontiguousarray(order, dtype=np.int64).reshape(-1)
        flags, stream = HOST_PTR, None

        def ptr(a):
            return None if a is None else a.ctypes.data
    data = _dtype_code(X)
    res = data if result is None else ({"float": F32, "single": F32, "double": F64}.get(result, result))
    # n labels, or n + 1 offsets from 0, non-decreasing, ending at len(labels)
    lab, off = _label_arrays(labels, offsets, n, X)
    count = n if od is None else int(od.shape[0])
    rc = lib.sdca_epoch_features(objarr, ctypes.c_int(data), ctypes.c_int(res), ctypes.c_int64(d),
                                 ctypes.c_int64(m), ctypes.c_int64(n), ctypes.c_void_p(ptr(X)),
                                 ctypes.c_void_p(ptr(W)), ctypes.c_void_p(ptr(A)),
                                 ctypes.c_void_p(ptr(lab)), ctypes.c_void_p(ptr(off)),
                                 ctypes.c_void_p(ptr(od)),
                                 ctypes.c_int64(count), ctypes.c_void_p(ptr(norms)),
                                 ctypes.c_uint(flags), stream)
    if rc != 0:
        raise SdcaError(rc, lib.sdca_last_error().decode())
    return W, A


def epoch_kernel(obj, K, A, labels, order=None, result=None, offsets=None):
    """One SDCA epoch on kernel input (the kernel form of update_variables,
    update.h:88-107, for each example of `order`) for an objective (name, c,
    gamma, k): K (n, n) the symmetric training kernel matrix, A (n, m)
    updated in place and returned.  CUDA tensors run on torch's current
    stream; numpy arrays (C-contiguous, K's dtype) go through the
    host-staging path.  order, result and offsets: as epoch_features."""
    lib = library()
    n = int(K.shape[0])
    m = int(A.shape[1])
    objarr = _objs([obj])
    lib.sdca_epoch_kernel.restype = ctypes.c_int
    if _is_torch(K):
        if not K.is_cuda:
            raise SdcaError(2, "epoch_kernel takes CUDA tensors or numpy arrays")
        import torch
        _need(K, "K", (n, n), K)
        _need(A, "A", (n, m), K)
        od = None
        if order is not None:
            od = torch.as_tensor(order, dtype=torch.int64, device=K.device).contiguous().reshape(-1)
        flags, stream = 0, _stream_ptr()
        ptr = _ptr
    else:
        for name, a, shape in (("K", K, (n, n)), ("A", A, (n, m))):
            if (not isinstance(a, np.ndarray) or a.dtype != K.dtype or tuple(a.shape) != shape
                    or not a.flags.c_contiguous):
                raise SdcaError(2, f"{name}: expected a C-contiguous {K.dtype} array {shape}")
        od = None if order is None else np.ascontiguousarray(order, dtype=np.int64).reshape(-1)
        flags, stream = HOST_PTR, None

        def ptr(a):
            return None if a is None else a.ctypes.data
    data = _dtype_code(K)
    res = data if result is None else ({"float": F32, "single": F32, "double": F64}.get(result, result))
    lab, off = _label_arrays(labels, offsets, n, K)
    count = n if od is None else int(od.shape[0])
    rc = lib.sdca_epoch_kernel(objarr, ctypes.c_int(data), ctypes.c_int(res), ctypes.c_int64(m),
                               ctypes.c_int64(n), ctypes.c_void_p(ptr(K)), ctypes.c_void_p(ptr(A)),
                               ctypes.c_void_p(ptr(lab)), ctypes.c_void_p(ptr(off)),
                               ctypes.c_void_p(ptr(od)), ctypes.c_int64(count),
                               ctypes.c_uint(flags), stream)
    if rc != 0:
        raise SdcaError(rc, lib.sdca_last_error().decode())
    return A


def recompute_primal(X, A, W0=None, out=None):
    """W = W0 + A^T X (the reference's W = W0 + X A' of eval_recompute_primal,
    eval/core.h:148-182): X (n, d) features, A (n, m) dual variables, W0 and
    the result (m, d)."""
    lib = library()
    n, d = int(X.shape[0]), int(X.shape[1])
    m = int(A.shape[1])
    data = _dtype_code(X)
    _need(X, "X", (n, d), X)
    _need(A, "A", (n, m), X)
    _need(W0, "W0", (m, d), X)
    _need(out, "out", (m, d), X)
    lib.sdca_recompute_primal.restype = ctypes.c_int
    if _is_torch(X):
        import torch
        W = out if out is not None else torch.empty((m, d), dtype=X.dtype, device=X.device)
        check(lib.sdca_recompute_primal(data, ctypes.c_int64(d), ctypes.c_int64(m), ctypes.c_int64(n),
                                        ctypes.c_void_p(X.data_ptr()), ctypes.c_void_p(A.data_ptr()),
                                        ctypes.c_void_p(_ptr(W0)), ctypes.c_void_p(W.data_ptr()),
                                        ctypes.c_uint(0), _stream_ptr()))
        return W
    W = out if out is not None else np.zeros((m, d), dtype=X.dtype)
    check(lib.sdca_recompute_primal(data, ctypes.c_int64(d), ctypes.c_int64(m), ctypes.c_int64(n),
                                    ctypes.c_void_p(X.ctypes.data), ctypes.c_void_p(A.ctypes.data),
                                    ctypes.c_void_p(_ptr(W0)), ctypes.c_void_p(W.ctypes.data),
                                    ctypes.c_uint(HOST_PTR), None))
    return W


EVAL_TEST = 2  # SDCA_EVAL_TEST


EVAL_FUSED = 4  # SDCA_EVAL_FUSED


def _eval(fn_name, objs, lead_args, m, n, labels, offsets, A, result, per_example, torch_mode,
          data, tail_args=(), test=False, fused=False):
    lib = library()
    res = data if result is None else ({"float": F32, "single": F32, "double": F64}.get(result, result))
    objarr = _objs(objs)
    recs = (EvalRecord * len(objs))()
    acc = np.zeros(m, dtype=np.float64)
    pe = None
    lab, off = _label_arrays(labels, offsets, n, lead_args[0])
    if torch_mode:
        import torch
        dev = lead_args[0].device
        if per_example:
            pe = torch.zeros((n, len(objs), 2), dtype=torch.float64, device=dev)
        flags, stream = 0, _stream_ptr()
    else:
        if per_example:
            pe = np.zeros((n, len(objs), 2), dtype=np.float64)
        flags, stream = HOST_PTR, None
    if test:
        flags |= EVAL_TEST
    if fused:
        flags |= EVAL_FUSED
    fn = getattr(lib, fn_name)
    fn.restype = ctypes.c_int
    args = [objarr, ctypes.c_int(len(objs)), ctypes.c_int(data), ctypes.c_int(res)]
    args += list(lead_args[1])
    args += [ctypes.c_void_p(_ptr(A)), *tail_args, ctypes.c_void_p(_ptr(lab)),
             ctypes.c_void_p(_ptr(off)), recs, ctypes.c_void_p(acc.ctypes.data),
             ctypes.c_void_p(_ptr(pe)), ctypes.c_uint(flags), stream]
    check(fn(*args))
    records = [{f: getattr(r, f) for f, _ in EvalRecord._fields_} for r in recs]
    return records, acc, pe


def eval_features(objs, X, W, labels, A=None, W0=None, offsets=None, result=None,
                  per_example=False, test=False, fused=False):
    """evaluate_dataset for feature input.  objs: list of objective(...).
    Returns (records, accuracy, per_example): one eval record per objective
    (primal, dual, primal_loss, dual_loss, primal/dual regularizer, rank_loss),
    the top-(i+1) accuracies (multiclass) and optionally the (n, n_obj, 2)
    per-example (primal, dual) losses before the loss coefficient.
    test=True gives a test set's records (eval_test: primal loss and
    accuracy / rank loss only).  fused=True runs the one-kernel form where it
    applies (SDCA_EVAL_FUSED; slower on MI355X; bit-identical results below
    2^32 multiply-adds n m d or 512 classes, equal to score rounding above,
    where the two-kernel form's scores come from hipBLASLt)."""
    n, d = int(X.shape[0]), int(X.shape[1])
    m = int(W.shape[0])
    _need(X, "X", (n, d), X)
    _need(W, "W", (m, d), X)
    _need(A, "A", (n, m), X)
    _need(W0, "W0", (m, d), X)
    lead = (X, [ctypes.c_int64(d), ctypes.c_int64(m), ctypes.c_int64(n),
                ctypes.c_void_p(_ptr(X)), ctypes.c_void_p(_ptr(W))])
    return _eval("sdca_eval_features", objs, lead, m, n, labels, offsets, A, result, per_example,
                 _is_torch(X), _dtype_code(X), tail_args=(ctypes.c_void_p(_ptr(W0)),), test=test,
                 fused=fused)


def eval_kernel(objs, K, A, labels, offsets=None, result=None, per_example=False, test=False):
    """evaluate_dataset for kernel input (data/input.h:44-76): K is (n, n_train),
    row i the kernel column K_i of example i; A is (n_train, m), the dual
    variables (rows are the reference's columns); scores_i = A K_i.  For a
    training set (n == n_train) the dual losses come from A's rows and the
    dual regularizer is sum_i 0.5 <a_i, s_i>; test=True gives a test set's
    records."""
    n, n_train = int(K.shape[0]), int(K.shape[1])
    m = int(A.shape[1])
    _need(K, "K", (n, n_train), K)
    _need(A, "A", (n_train, m), K)
    lead = (K, [ctypes.c_int64(n_train), ctypes.c_int64(m), ctypes.c_int64(n),
                ctypes.c_void_p(_ptr(K))])
    return _eval("sdca_eval_kernel", objs, lead, m, n, labels, offsets, A, result, per_example,
                 _is_torch(K), _dtype_code(K), test=test)


def eval_scores(objs, S, labels, A=None, offsets=None, primal_regularizer=0.0,
                dual_regularizer=0.0, result=None, per_example=False):
    """The per-example part of evaluate_dataset on precomputed scores S."""
    n, m = int(S.shape[0]), int(S.shape[1])
    _need(S, "S", (n, m), S)
    _need(A, "A", (n, m), S)
    lib = library()
    res = _dtype_code(S) if result is None else ({"float": F32, "single": F32, "double": F64}.get(result, result))
    torch_mode = _is_torch(S)
    objarr = _objs(objs)
    recs = (EvalRecord * len(objs))()
    acc = np.zeros(m, dtype=np.float64)
    lab, off = _label_arrays(labels, offsets, n, S)
    if torch_mode:
        import torch
        pe = torch.zeros((n, len(objs), 2), dtype=torch.float64, device=S.device) if per_example else None
        flags, stream = 0, _stream_ptr()
    else:
        pe = np.zeros((n, len(objs), 2), dtype=np.float64) if per_example else None
        flags, stream = HOST_PTR, None
    lib.sdca_eval_scores.restype = ctypes.c_int
    check(lib.sdca_eval_scores(objarr, ctypes.c_int(len(objs)), ctypes.c_int(_dtype_code(S)),
                               ctypes.c_int(res), ctypes.c_int64(m), ctypes.c_int64(n),
                               ctypes.c_void_p(_ptr(S)), ctypes.c_void_p(_ptr(A)),
                               ctypes.c_void_p(_ptr(lab)), ctypes.c_void_p(_ptr(off)),
                               ctypes.c_double(primal_regularizer), ctypes.c_double(dual_regularizer),
                               recs, ctypes.c_void_p(acc.ctypes.data), ctypes.c_void_p(_ptr(pe)),
                               ctypes.c_uint(flags), stream))
    records = [{f: getattr(r, f) for f, _ in EvalRecord._fields_} for r in recs]
    return records, acc, pe


# ---------------------------------------------------------------------------
# Answering from a trained model: scores from 8-bit weights, and labels drawn
# from scores.  Matrices may have rows further apart than their length (a
# stride of 1 within a row); CUDA tensors run on torch's current stream,
# numpy arrays go through the host-staging path.
# ---------------------------------------------------------------------------
F16, BF16, I8 = 3, 4, 5
_answer_codes = None


def _answer_dtype(x):
    global _answer_codes
    if _answer_codes is None:
        _answer_codes = {np.dtype(np.float32): F32, np.dtype(np.float64): F64,
                         np.dtype(np.float16): F16, np.dtype(np.int8): I8}
        try:
            import torch
            _answer_codes.update({torch.float32: F32, torch.float64: F64, torch.float16: F16,
                                  torch.bfloat16: BF16, torch.int8: I8})
        except ImportError:
            pass
    return _answer_codes.get(x.dtype, -1)


def _pitch(x, name, shape=None):
    """The distance between the rows of the matrix x, in elements."""
    if x.ndim != 2:
        raise SdcaError(2, f"{name} must be 2-D (got {x.ndim} dimensions)")
    n, d = x.shape
    if shape is not None and (n, d) != shape:
        raise SdcaError(2, f"{name} has shape {(n, d)}, expected {shape}")
    if _is_torch(x):
        step, one = x.stride()
    else:
        step, one = (s // x.itemsize for s in x.strides)
        if not x.dtype.isnative or any(s % x.itemsize for s in x.strides):
            raise SdcaError(2, f"{name}: unsupported layout")
    if n <= 1:
        step = d
    if (one != 1 and d > 1) or step < d:
        raise SdcaError(2, f"{name}: the values of a row must be neighbours, and rows apart")
    return step


def _written(x, name):
    """The library writes through a raw pointer, so an array that numpy holds
    read-only (a view of bytes, of a file mapped for reading) is refused."""
    if not _is_torch(x) and not x.flags.writeable:
        raise SdcaError(2, f"{name} is read-only")


def _values(x, name, n, dtype, like):
    """Checks a vector of n values of the given element type beside `like`."""
    if _is_torch(x) != _is_torch(like):
        raise SdcaError(2, f"{name}: numpy arrays and torch tensors cannot be mixed in one call")
    if x.dtype != dtype:
        raise SdcaError(3, f"{name} has element type {x.dtype}, expected {dtype}")
    if tuple(x.shape) != (n,):
        raise SdcaError(2, f"{name} has shape {tuple(x.shape)}, expected {(n,)}")
    if not (x.is_contiguous() if _is_torch(x) else x.flags.c_contiguous):
        raise SdcaError(2, f"{name} must be contiguous")
    if _is_torch(x) and x.device != like.device:
        raise SdcaError(2, f"{name} is on {x.device}, expected {like.device}")
    return x


_raw_stream = None


def _torch_stream(device):
    """torch's current stream on a device, as the C ABI takes it."""
    global _raw_stream
    if _raw_stream is None:
        torch = sys.modules["torch"]
        # The number alone; a Stream object takes longer to make than a
        # small call to run.
        _raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
            lambda index: torch.cuda.current_stream(index).cuda_stream)
    return _raw_stream(device)


def _answer(x, name, fn, *args):
    """Calls fn(*args, flags, stream) for the tensor or array x: on torch's
    current stream of its device, or with host arrays."""
    if not _is_torch(x):
        return check(fn(*args, HOST_PTR, None))
    if not x.is_cuda:
        raise SdcaError(2, f"{name} takes CUDA tensors or numpy arrays")
    torch = sys.modules["torch"]
    device = x.get_device()
    if device == torch.cuda.current_device():
        return check(fn(*args, 0, _torch_stream(device)))
    with torch.cuda.device(device):
        return check(fn(*args, 0, _torch_stream(device)))


def _empty(shape, dtype, like):
    """dtype by its numpy name."""
    if _is_torch(like):
        torch = sys.modules["torch"]
        return torch.empty(shape, dtype=getattr(torch, dtype), device=like.device)
    return np.empty(shape, dtype=dtype)


def quantize_i8(A, out=None, scales=None):
    """(Q, scales): the rows of A (float32, float64, float16 or bfloat16) as
    8-bit integers with a float32 scale each, A[i] ~ Q[i] scales[i] with
    scales[i] = max |A[i]| (1 / 127) (sdca_quantize_i8).  Without `out`, Q's rows
    are a multiple of 16 bytes apart, which scores_i8 reads in place."""
    lib = library()
    data = _answer_dtype(A)
    if data < 0 or data == I8:
        raise SdcaError(3, f"unsupported element type {A.dtype}")
    lda = _pitch(A, "A")
    n, d = A.shape
    like = out if out is not None else A
    if _is_torch(like) != _is_torch(A) or (_is_torch(A) and like.device != A.device):
        raise SdcaError(2, "out: expected the same kind and device as A")
    Q = out if out is not None else _empty((n, (d + 15) // 16 * 16), "int8", A)[:, :d]
    if _answer_dtype(Q) != I8:
        raise SdcaError(3, f"out has element type {Q.dtype}, expected int8")
    ldq = _pitch(Q, "out", (n, d))
    _written(Q, "out")
    s = scales if scales is not None else _empty((n,), "float32", A)
    _values(s, "scales", n, _float32(A), A)
    _written(s, "scales")
    _answer(A, "quantize_i8", lib.sdca_quantize_i8, data, d, n, _ptr(A), lda, _ptr(Q), ldq, _ptr(s))
    return Q, s


def _float32(like):
    if _is_torch(like):
        return sys.modules["torch"].float32
    return np.float32


def scores_i8(X, W, w_scales, x_scales=None, out=None, dtype=None):
    """S = X W^T with W in 8 bits (scores for a quantised model):
    W (m, d) int8 with its m scales, as quantize_i8 gives them; X (n, d) int8
    with x_scales, or float32, float64, float16 or bfloat16 without, which is
    quantised row by row within the call.  S is (n, m) of `dtype` (float32 by
    default, float16 or bfloat16; a dtype of torch or numpy) or of out's."""
    lib = library()
    data = _answer_dtype(X)
    if data < 0:
        raise SdcaError(3, f"unsupported element type {X.dtype}")
    ldx = _pitch(X, "X")
    n, d = X.shape
    m = W.shape[0]
    if _is_torch(W) != _is_torch(X) or (_is_torch(X) and W.device != X.device):
        raise SdcaError(2, "W: expected the same kind and device as X")
    if _answer_dtype(W) != I8:
        raise SdcaError(3, f"W has element type {W.dtype}, expected int8")
    ldw = _pitch(W, "W", (m, d))
    f32 = _float32(X)
    _values(w_scales, "w_scales", m, f32, X)
    if (x_scales is None) == (data == I8):
        raise SdcaError(1, "x_scales go with int8 examples, and with them only")
    if x_scales is not None:
        _values(x_scales, "x_scales", n, f32, X)
    if out is None:
        if _is_torch(X):
            out = sys.modules["torch"].empty((n, m), dtype=dtype or f32, device=X.device)
        else:
            out = np.empty((n, m), dtype=dtype or f32)
    elif _is_torch(out) != _is_torch(X) or (_is_torch(X) and out.device != X.device):
        raise SdcaError(2, "out: expected the same kind and device as X")
    code = _answer_dtype(out)
    if code not in (F32, F16, BF16):
        raise SdcaError(3, f"scores cannot be {out.dtype}")
    lds = _pitch(out, "out", (n, m))
    _written(out, "out")
    _answer(X, "scores_i8", lib.sdca_scores_i8, data, code, d, m, n, _ptr(X), ldx, _ptr(x_scales),
            _ptr(W), ldw, _ptr(w_scales), _ptr(out), lds)
    return out


def _setting(v, name, n, kind, like):
    """A setting's array of n values beside `like`, or None for a number."""
    if isinstance(v, (float, int)) or not (_is_torch(v) or isinstance(v, (np.ndarray, list, tuple))):
        return None
    if _is_torch(like):
        torch = sys.modules["torch"]
        dtype = getattr(torch, kind)
        if not (_is_torch(v) and v.dtype == dtype and v.device == like.device and v.is_contiguous()):
            v = torch.as_tensor(v, dtype=dtype, device=like.device).contiguous()
    elif _is_torch(v):
        raise SdcaError(2, f"{name}: numpy arrays and torch tensors cannot be mixed in one call")
    else:
        v = np.ascontiguousarray(v, dtype=kind)
    if tuple(v.shape) != (n,):
        raise SdcaError(2, f"{name} has shape {tuple(v.shape)}, expected {(n,)}")
    return v


def sample(S, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, prob=False, kept=False):
    """Draws a label for each row of the scores S (n, m) (float32, float64,
    float16 or bfloat16) with the random numbers u (n float32 values in
    [0, 1)): int64 labels, -1 for a row that has none (sdca_sample).  The
    settings are numbers, or arrays of n values (float32; int64 for top_k).
    A row has at most 2^23 scores.
    With prob=True also the drawn labels' probabilities after the cuts, with
    kept=True also the number of labels that the cuts left."""
    lib = library()
    data = _answer_dtype(S)
    if data < 0 or data == I8:
        raise SdcaError(3, f"unsupported element type {S.dtype}")
    lds = _pitch(S, "S")
    n, m = S.shape
    _values(u, "u", n, _float32(S), S)
    T = _setting(temperature, "temperature", n, "float32", S)
    p = _setting(top_p, "top_p", n, "float32", S)
    q = _setting(min_p, "min_p", n, "float32", S)
    k = _setting(top_k, "top_k", n, "int64", S)
    params = SampleParams(1.0 if T is not None else temperature, 1.0 if p is not None else top_p,
                          0.0 if q is not None else min_p, 0 if k is not None else int(top_k))
    columns = SampleColumns(_ptr(T), _ptr(p), _ptr(q), _ptr(k))
    labels = _empty((n,), "int64", S)
    pr = _empty((n,), "float32", S) if prob else None
    kp = _empty((n,), "int64", S) if kept else None
    _answer(S, "sample", lib.sdca_sample, data, m, n, _ptr(S), lds, _ptr(u), params, columns,
            _ptr(labels), _ptr(pr), _ptr(kp))
    res = (labels,) + ((pr,) if prob else ()) + ((kp,) if kept else ())
    return res if len(res) > 1 else labels


def _scratch(x, size, *args):
    """Device scratch of size(*args) bytes for a call on the tensor x, from
    torch's allocator (a captured call's then belongs to its graph); None for
    numpy arrays, whose calls use the library's own."""
    if not _is_torch(x):
        return None
    n = size(*args)
    return sys.modules["torch"].empty(n, dtype=sys.modules["torch"].uint8, device=x.device) if n else None


def _label_values(labels, n, like):
    return _values(labels, "labels", n, sys.modules["torch"].int64 if _is_torch(like) else np.int64, like)


def _score_type(S):
    data = _answer_dtype(S)
    if data not in (F32, F16, BF16):
        raise SdcaError(3, f"unsupported element type {S.dtype}")
    return data


def log_probs(S, labels, temperature=1.0, top=0, entropy=False, stats=False):
    """The log-probability of a given label for each row of the scores S (n, m)
    (float32, float16 or bfloat16): float32, 0 for a label of -1, which asks for
    none (sdca_log_probs).  labels: n int64 in [-1, m).
    With entropy=True also the rows' entropies (n,), with stats=True also what
    log_probs_grad takes of them (n, 3): the largest score, the logarithm of the
    sum of the weights relative to it and the entropy; with top > 0 also the
    log-probabilities and the indices (int64) of each row's `top` largest
    scores, (n, top) each, ties by rising index, -inf and -1 where a row has
    fewer scores above -inf.  top is at most 64."""
    lib = library()
    data = _score_type(S)
    lds = _pitch(S, "S")
    n, m = S.shape
    _label_values(labels, n, S)
    top = int(top)
    logp = _empty((n,), "float32", S)
    ent = _empty((n,), "float32", S) if entropy else None
    st = _empty((n, 3), "float32", S) if stats else None
    best = _empty((n, max(top, 0)), "float32", S) if top else None
    at = _empty((n, max(top, 0)), "int64", S) if top else None
    work = _scratch(S, lib.sdca_log_probs_work, data, m, n, top)
    _answer(S, "log_probs", lib.sdca_log_probs, data, m, n, _ptr(S), lds, _ptr(labels), float(temperature), top,
            _ptr(logp), _ptr(ent), _ptr(st), _ptr(best), _ptr(at), _ptr(work))
    res = (logp,) + ((ent,) if entropy else ()) + ((st,) if stats else ()) + ((best, at) if top else ())
    return res if len(res) > 1 else logp


def log_probs_grad(S, labels, g, g_entropy=None, stats=None, temperature=1.0, out=None, logp=False):
    """The gradient of the scores S where g (n float32) is that of the labels'
    log-probabilities and g_entropy, if given, that of the rows' entropies
    (sdca_log_probs_grad): a matrix of S's type, or `out`, which may be S.
    A row of label -1 has none from g.  stats: what log_probs(stats=True) gave
    for the same S and temperature; without, they are computed here.  With
    logp=True also the labels' log-probabilities."""
    lib = library()
    data = _score_type(S)
    lds = _pitch(S, "S")
    n, m = S.shape
    f32 = _float32(S)
    _label_values(labels, n, S)
    _values(g, "g", n, f32, S)
    if g_entropy is not None:
        _values(g_entropy, "g_entropy", n, f32, S)
    if stats is not None:
        if len(stats.shape) != 2:
            raise SdcaError(2, f"stats has shape {tuple(stats.shape)}, expected {(n, 3)}")
        _values(stats.reshape(-1), "stats", 3 * n, f32, S)
        if tuple(stats.shape) != (n, 3) or not (
                stats.is_contiguous() if _is_torch(stats) else stats.flags.c_contiguous):
            raise SdcaError(2, f"stats must be a contiguous {(n, 3)} matrix")
    if out is None:
        out = sys.modules["torch"].empty((n, m), dtype=S.dtype, device=S.device) if _is_torch(S) else \
            np.empty((n, m), dtype=S.dtype)
    elif _is_torch(out) != _is_torch(S) or (_is_torch(S) and out.device != S.device):
        raise SdcaError(2, "out: expected the same kind and device as S")
    if out.dtype != S.dtype:
        raise SdcaError(3, f"out has element type {out.dtype}, expected {S.dtype}")
    ldd = _pitch(out, "out", (n, m))
    _written(out, "out")
    lp = _empty((n,), "float32", S) if logp else None
    work = _scratch(S, lib.sdca_log_probs_grad_work, data, m, n, _ptr(stats))
    _answer(S, "log_probs_grad", lib.sdca_log_probs_grad, data, m, n, _ptr(S), lds, _ptr(labels), _ptr(g),
            _ptr(g_entropy), _ptr(stats), float(temperature), _ptr(out), ldd, _ptr(lp), _ptr(work))
    return (out, lp) if logp else out


def _stack(x, name, shape, like):
    """Checks the matrices of all adapters, one behind the other."""
    if _is_torch(x) != _is_torch(like) or (_is_torch(x) and x.device != like.device):
        raise SdcaError(2, f"{name}: expected the same kind and device as X")
    if x.dtype != like.dtype:
        raise SdcaError(3, f"{name} has element type {x.dtype}, expected {like.dtype}")
    if tuple(x.shape) != shape:
        raise SdcaError(2, f"{name} has shape {tuple(x.shape)}, expected {shape}")
    if not (x.is_contiguous() if _is_torch(x) else x.flags.c_contiguous):
        raise SdcaError(2, f"{name} must be contiguous")


def _adapters(X, A, B, index, scale, m):
    """(the call's argument, what has to live as long) for the adapters A
    (count, rank, d), B (count, m, rank)."""
    n, d = X.shape
    if len(A.shape) != 3:
        raise SdcaError(2, f"A must be 3-D (got {len(A.shape)} dimensions)")
    count, rank = int(A.shape[0]), int(A.shape[1])
    _stack(A, "A", (count, rank, d), X)
    _stack(B, "B", (count, m, rank), X)
    _values(index, "index", n, sys.modules["torch"].int64 if _is_torch(X) else np.int64, X)
    each = _setting(scale, "scale", count, "float32", X)
    return Adapters(count, rank, _ptr(A), _ptr(B), _ptr(index), _ptr(each),
                    1.0 if each is not None else float(scale)), each


def scores_adapted(X, W, w_scales, A, B, index, scale=1.0, out=None, dtype=None):
    """S = scores_i8(X, W, w_scales) + scale[a] (X A[a]^T) B[a]^T with an adapter
    a = index[i] for each row of X, -1 for none (sdca_scores_adapted): the
    scores of many requests, each with a low-rank correction of the shared 8-bit
    weights.  X (n, d) float32, float16 or bfloat16; A (count, rank, d) and
    B (count, m, rank) contiguous and of X's type, rank at most 128; index n
    int64; scale a number or count values.  S as scores_i8 gives it."""
    lib = library()
    data = _score_type(X)
    ldx = _pitch(X, "X")
    n, d = X.shape
    if _is_torch(W) != _is_torch(X) or (_is_torch(X) and W.device != X.device):
        raise SdcaError(2, "W: expected the same kind and device as X")
    if _answer_dtype(W) != I8:
        raise SdcaError(3, f"W has element type {W.dtype}, expected int8")
    m = W.shape[0]
    ldw = _pitch(W, "W", (m, d))
    f32 = _float32(X)
    _values(w_scales, "w_scales", m, f32, X)
    adapters, each = _adapters(X, A, B, index, scale, m)
    if out is None:
        if _is_torch(X):
            out = sys.modules["torch"].empty((n, m), dtype=dtype or f32, device=X.device)
        else:
            out = np.empty((n, m), dtype=dtype or f32)
    elif _is_torch(out) != _is_torch(X) or (_is_torch(X) and out.device != X.device):
        raise SdcaError(2, "out: expected the same kind and device as X")
    code = _answer_dtype(out)
    if code not in (F32, F16, BF16):
        raise SdcaError(3, f"scores cannot be {out.dtype}")
    lds = _pitch(out, "out", (n, m))
    _written(out, "out")
    work = _scratch(X, lib.sdca_scores_adapted_work, data, d, m, n, _ptr(W), ldw,
                    adapters.count, adapters.rank)
    _answer(X, "scores_adapted", lib.sdca_scores_adapted, data, code, d, m, n, _ptr(X), ldx, _ptr(W), ldw,
            _ptr(w_scales), adapters, _ptr(out), lds, _ptr(work))
    return out


def scores_adapted_grad(G, X, A, B, index, scale=1.0):
    """(dA, dB): the gradients of the adapters where G (n, m) (float32, float16
    or bfloat16) is that of scores_adapted's scores, float32, laid out as A and
    B (sdca_scores_adapted_grad); zeros for an adapter that no row has.  The
    examples and the shared weights are fixed and have none."""
    lib = library()
    data = _score_type(X)
    ldx = _pitch(X, "X")
    n, d = X.shape
    if _is_torch(G) != _is_torch(X) or (_is_torch(X) and G.device != X.device):
        raise SdcaError(2, "G: expected the same kind and device as X")
    grad = _score_type(G)
    if G.ndim != 2:
        raise SdcaError(2, f"G must be 2-D (got {G.ndim} dimensions)")
    m = G.shape[1]
    ldg = _pitch(G, "G", (n, m))
    adapters, each = _adapters(X, A, B, index, scale, m)
    dA = _empty(tuple(A.shape), "float32", X)
    dB = _empty(tuple(B.shape), "float32", X)
    work = _scratch(X, lib.sdca_scores_adapted_grad_work, data, grad, d, m, n, adapters.count, adapters.rank)
    _answer(X, "scores_adapted_grad", lib.sdca_scores_adapted_grad, data, grad, d, m, n, _ptr(G), ldg, _ptr(X),
            ldx, adapters, _ptr(dA), _ptr(dB), _ptr(work))
    return dA, dB
