"""Operators on class scores that lie on the GPU, as torch tensors (tgbm_scores_*): what is known besides the model is put on
the scores (`adjust`), the best classes of every row are listed (`top`) or one is drawn (`sample`), and they
are held against a teacher's best scores (`distill`). Scores of a linear layer, as a larger model's last one, are a product in
8 bits (`linear`) of rows that `quantise` makes. torch is imported by the caller, never here.

Scores are [classes, rows], float32, float16 or bfloat16, in either order: the rows of a class side by side, as trainers and
predictors hold them, or the classes of a row side by side (`x.t()` of a [rows, classes] tensor). Everything is launched on
torch's current stream of the tensors' device; nothing waits, and calls can be captured into a graph. Wrong arguments
raise ValueError before anything is launched. The calls take no part in autograd: a tensor that requires a gradient is refused.
"""
import ctypes as C
import functools
import math
import operator
import sys

from . import _lib


class _Scores(C.Structure):
    _fields_ = [("data", C.c_void_p), ("class_stride", C.c_longlong), ("row_stride", C.c_longlong), ("type", C.c_int),
                ("classes", C.c_int), ("rows", C.c_int)]


class _Rules(C.Structure):
    _fields_ = [("bias", C.c_void_p), ("allowed", C.c_void_p), ("allowed_set", C.c_void_p), ("shown", C.c_void_p),
                ("shown_begin", C.c_void_p), ("n_shown", C.c_longlong), ("allowed_sets", C.c_int), ("repetition", C.c_float),
                ("frequency", C.c_float), ("presence", C.c_float)]


class _Sampling(C.Structure):
    _fields_ = [("temperature", C.c_void_p), ("p", C.c_void_p), ("min_p", C.c_void_p), ("k", C.c_void_p), ("temperature_all", C.c_float),
                ("p_all", C.c_float), ("min_p_all", C.c_float), ("k_all", C.c_int)]


class _Rows(C.Structure):
    _fields_ = [("data", C.c_void_p), ("scale", C.c_void_p), ("pitch", C.c_longlong), ("type", C.c_int), ("rows", C.c_int), ("features", C.c_int),
                ("padded", C.c_int)]


class _Teacher(C.Structure):
    _fields_ = [("classes", C.c_void_p), ("scores", C.c_void_p), ("lse", C.c_void_p), ("type", C.c_int), ("entries", C.c_int)]


_types = None


def _torch():
    """The caller's torch, and the numbers of the types."""
    global _types
    torch = sys.modules.get("torch")
    if torch is None:
        raise ValueError("the scores are torch tensors")
    if _types is None:
        _types = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
    return torch


def _on_gpu(torch, name, x):
    if not isinstance(x, torch.Tensor):
        raise ValueError("%s: a torch tensor is wanted, got %s" % (name, type(x).__name__))
    if not x.is_cuda:
        raise ValueError("%s: a tensor on the GPU is wanted" % name)
    if x.requires_grad:
        raise ValueError("%s requires a gradient: these operators take no part in autograd (detach it)" % name)


def _scores(torch, name, x):
    _on_gpu(torch, name, x)
    kind = _types.get(x.dtype)
    if kind is None:
        raise ValueError("%s: float32, float16 or bfloat16 is wanted, got %s" % (name, x.dtype))
    if x.dim() != 2:
        raise ValueError("%s: [classes, rows] is wanted, got %d dimensions" % (name, x.dim()))
    classes, rows = x.shape
    by_class, by_row = x.stride()
    if classes < 1 or classes > 1 << 22 or rows >= 1 << 31:
        raise ValueError("%s: %d classes, %d rows" % (name, classes, rows))
    if classes == 1:  # (the stride along a single class says nothing)
        by_class = max(by_class, rows, 1) if by_row == 1 else 1
    if rows <= 1:
        by_row = max(by_row, classes) if by_class == 1 else 1
    if not (by_row == 1 and by_class >= rows) and not (by_class == 1 and by_row >= classes):
        raise ValueError("%s: strides %s of a tensor %s: the rows of a class or the classes of a row lie side by side"
                         % (name, tuple(x.stride()), tuple(x.shape)))
    return _Scores(x.data_ptr(), by_class, by_row, kind, classes, rows)


def _plain(torch, name, x, like, dtype, shape):
    """The address of a contiguous tensor of one type, on the scores' device."""
    if (isinstance(x, torch.Tensor) and x.dtype is dtype and x.shape == shape and x.is_cuda and x.get_device() == like.get_device()
            and x.is_contiguous() and not x.requires_grad):
        return x.data_ptr()
    _on_gpu(torch, name, x)
    if x.dtype != dtype:
        raise ValueError("%s: %s is wanted, got %s" % (name, dtype, x.dtype))
    if x.device != like.device:
        raise ValueError("%s is on %s, the scores are on %s" % (name, x.device, like.device))
    if tuple(x.shape) != shape:
        raise ValueError("%s: the shape %s is wanted, got %s" % (name, shape, tuple(x.shape)))
    raise ValueError("%s: a contiguous tensor is wanted" % name)


def _rules(torch, scores, bias, allowed, allowed_set, shown, shown_begin, repetition, frequency, presence):
    classes, rows = scores.shape
    r = _Rules()
    if bias is not None:
        r.bias = _plain(torch, "bias", bias, scores, torch.float32, (classes,))
    if allowed is not None:
        _on_gpu(torch, "allowed", allowed)
        if allowed.dim() != 2 or allowed.shape[0] < 1:
            raise ValueError("allowed: [sets, (classes + 31) // 32] is wanted, got %s" % (tuple(allowed.shape),))
        sets = allowed.shape[0]
        r.allowed = _plain(torch, "allowed", allowed, scores, torch.int32, (sets, (classes + 31) // 32))
        r.allowed_sets = sets
        if allowed_set is not None:
            r.allowed_set = _plain(torch, "allowed_set", allowed_set, scores, torch.int32, (rows,))
        elif sets != 1 and sets != rows:
            raise ValueError("allowed: %d sets for %d rows: which one is a row's says allowed_set" % (sets, rows))
    elif allowed_set is not None:
        raise ValueError("allowed_set without allowed")
    if (shown is None) != (shown_begin is None):
        raise ValueError("shown and shown_begin belong together")
    if shown is not None:
        r.shown_begin = _plain(torch, "shown_begin", shown_begin, scores, torch.int64, (rows + 1,))
        if shown.dim() != 1:
            raise ValueError("shown: one dimension is wanted, got %d" % shown.dim())
        r.n_shown = shown.numel()
        # (an empty tensor has no address, and no list is like empty lists)
        r.shown = _plain(torch, "shown", shown, scores, torch.int32, (shown.numel(),)) if shown.numel() else None
        if not shown.numel():
            r.shown_begin = None
        if not (repetition > 0 and math.isfinite(repetition)):
            raise ValueError("repetition is %r: a number above 0 is wanted" % (repetition,))
        if not (math.isfinite(frequency) and math.isfinite(presence)):
            raise ValueError("frequency is %r, presence is %r: numbers are wanted" % (frequency, presence))
        r.repetition, r.frequency, r.presence = repetition, frequency, presence
    return r


def _rows(torch, name, x, scale=None, whole=False, floating=True):
    """Rows of numbers, [rows, features]; int8 ones with their scales."""
    if not isinstance(x, torch.Tensor) or not x.is_cuda or x.requires_grad:
        _on_gpu(torch, name, x)
    kind = _types.get(x.dtype) if floating else None
    if kind is None and whole and x.dtype == torch.int8:
        kind = 3
    if kind is None:
        raise ValueError("%s: %s is wanted, got %s" % (name, " or ".join((["float32, float16, bfloat16"] if floating else []) + (["int8"] if whole else [])), x.dtype))
    if x.dim() != 2 or not 1 <= x.shape[1] <= 65536 or x.shape[0] >= 1 << 31:
        raise ValueError("%s: [rows, features] with 1 to 65536 features is wanted, got %s" % (name, tuple(x.shape)))
    rows, features = x.shape
    pitch = x.stride(0) if rows > 1 else features
    if (features > 1 and x.stride(1) != 1) or pitch < features:
        raise ValueError("%s: strides %s of a tensor %s: the features of a row lie side by side" % (name, tuple(x.stride()), tuple(x.shape)))
    r = _Rows(x.data_ptr(), None, pitch, kind, rows, features, 0)
    if kind == 3:
        if scale is None:
            raise ValueError("%s: whole numbers go with a scale for each row" % name)
        r.scale = _plain(torch, name + "_scale", scale, x, torch.float32, (rows,))
        if features % 16:  # (whether the memory goes on behind the last row as it does behind the others)
            left = x.untyped_storage().nbytes() - x.storage_offset()
            if rows == 1 and left >= (features + 15) // 16 * 16:
                r.pitch = (features + 15) // 16 * 16
            r.padded = 1 if left >= rows * r.pitch else 0
    elif scale is not None:
        raise ValueError("%s_scale goes with whole numbers, %s is %s" % (name, name, x.dtype))
    return r


def _list_length(k):
    """How many classes are listed, as any type of integer."""
    try:
        n = operator.index(k)
    except TypeError:
        n = 0
    if not 1 <= n <= 128:
        raise ValueError("k is %r: 1 to 128 is wanted" % (k,))
    return n


_functions = {}


def _call(torch, scores, name, *args):
    """One call of the library on the current stream of the scores' device."""
    fn = _functions.get(name)
    if fn is None:
        fn = _functions[name] = getattr(_lib.load(), name)
    device = scores.get_device()
    if device == torch.cuda.current_device():
        rc = fn(*args, _stream(torch, device))
    else:
        with torch.cuda.device(device):
            rc = fn(*args, _stream(torch, device))
    if rc:
        raise (ValueError if rc == 1 else RuntimeError)("%s failed; it has said why on stderr" % name)


def _stream(torch, device):
    """The number of the current stream (3 us through torch's stream objects, as much as a launch)."""
    raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)
    return raw(device) if raw is not None else torch.cuda.current_stream(device).cuda_stream


@functools.lru_cache(maxsize=256)
def _top_workspace(by_class, by_row, classes, rows, k):
    return _lib.load().tgbm_scores_top_workspace(C.byref(_Scores(1, by_class, by_row, 0, classes, rows)), k)


@functools.lru_cache(maxsize=256)
def _sample_workspace(kind, by_class, by_row, classes, rows, shown, k):
    """shown: whether there are lists; k: the rows' common one, None where each has its own."""
    r, h = _Rules(repetition=1.0), _Sampling(None, None, None, 1 if k is None else None, 1.0, 1.0, 0.0, k or 0)  # (addresses stand for any)
    if shown:
        r.shown, r.shown_begin = 1, 1
    return _lib.load().tgbm_scores_sample_workspace(C.byref(_Scores(1, by_class, by_row, kind, classes, rows)), C.byref(r), C.byref(h))


@functools.lru_cache(maxsize=256)
def _linear_workspace(features, *rows):
    """rows: of x and of the weights, the place in 16 bytes, pitch, type, rows, padded."""
    x, w = (_Rows(16 + at, 16, pitch, kind, n, features, padded) for at, pitch, kind, n, padded in (rows[:5], rows[5:]))
    return _lib.load().tgbm_scores_linear_workspace(C.byref(x), C.byref(w))


@functools.lru_cache(maxsize=256)
def _distill_workspace(classes, rows, entries):
    return _lib.load().tgbm_scores_distill_workspace(C.byref(_Scores(1, max(rows, 1), 1, 0, classes, rows)), entries)


def adjust(scores, bias=None, allowed=None, allowed_set=None, shown=None, shown_begin=None, repetition=1.0, frequency=0.0,
           presence=0.0, out=None):
    """The scores with what is known besides them, in their type and order.

    bias: float32 [classes], added to every row's scores.
    shown, shown_begin: classes that the rows were shown before, int32 lists one behind the other, and where they begin, int64
      [rows + 1]. A score s of a class that the row was shown m times becomes (s / repetition if s > 0 else s * repetition) -
      frequency * m - presence. Numbers that are no classes are skipped.
    allowed: int32 [sets, (classes + 31) // 32], bit c % 32 of word c // 32 says whether class c is allowed; the others'
      scores become -inf. One set for all rows, one for each, or with allowed_set, int32 [rows], the rows' sets: a negative
      number allows everything, one that is no set's nothing.
    out: where the result goes; `scores` itself, or memory apart from it."""
    torch = _torch()
    s = _scores(torch, "scores", scores)
    r = _rules(torch, scores, bias, allowed, allowed_set, shown, shown_begin, repetition, frequency, presence)
    if out is None:
        # (in the scores' order, without the gaps that a part of a larger array has)
        if s.class_stride == 1 and s.rows > 1:
            out = torch.empty((s.rows, s.classes), dtype=scores.dtype, device=scores.device).t()
            o = _Scores(out.data_ptr(), 1, s.classes, s.type, s.classes, s.rows)
        else:
            out = torch.empty((s.classes, s.rows), dtype=scores.dtype, device=scores.device)
            o = _Scores(out.data_ptr(), max(s.rows, 1), 1, s.type, s.classes, s.rows)
        if s.rows:
            _call(torch, scores, "tgbm_scores_adjust", C.byref(s), C.byref(r), C.byref(o))
        return out
    if not isinstance(out, torch.Tensor) or out.dtype != scores.dtype or out.shape != scores.shape or out.device != scores.device:
        raise ValueError("out: a tensor of the scores' type, shape and device is wanted")
    o = _scores(torch, "out", out)
    if s.rows:
        if o.data == s.data:
            if (o.class_stride, o.row_stride) != (s.class_stride, s.row_stride):
                raise ValueError("out is the scores' memory in another order")
        else:
            size = scores.element_size()
            ends = [x.data + ((x.classes - 1) * x.class_stride + (x.rows - 1) * x.row_stride + 1) * size for x in (s, o)]
            # (two parts of one array may lie between each other's rows: what counts is that they have the same strides then)
            if o.data < ends[0] and s.data < ends[1] and not _apart(s, o, size):
                raise ValueError("out overlaps the scores")
        _call(torch, scores, "tgbm_scores_adjust", C.byref(s), C.byref(r), C.byref(o))
    return out


def top(scores, k, bias=None, allowed=None, allowed_set=None, shown=None, shown_begin=None, repetition=1.0, frequency=0.0,
        presence=0.0, temperature=1.0):
    """The k (1 to 128) best classes of every row, by the scores as `adjust` would leave them: values float32 [rows, k], classes int32
    [rows, k], lse float32 [rows].

    The best come first, of equal scores the lower class. A class whose score is -inf or NaN is not listed; a list that is
    not filled ends with class -1 and -inf. lse is the logarithm of the sum of exp(score / temperature) over all classes (-inf
    where nothing is allowed, NaN where a score is NaN), so that exp(values / temperature - lse[:, None]) are probabilities; lse being a 32-bit number, they
    are off by up to 2^-23 of values / temperature where that is large."""
    torch = _torch()
    s = _scores(torch, "scores", scores)
    r = _rules(torch, scores, bias, allowed, allowed_set, shown, shown_begin, repetition, frequency, presence)
    k = _list_length(k)
    if not 1e-6 <= temperature <= 1e6:
        raise ValueError("temperature is %r: 1e-6 to 1e6 is wanted" % (temperature,))
    n, device = s.rows, scores.device
    values = torch.empty((n, k), dtype=torch.float32, device=device)
    classes = torch.empty((n, k), dtype=torch.int32, device=device)
    lse = torch.empty(n, dtype=torch.float32, device=device)
    if n:
        size = _top_workspace(s.class_stride, s.row_stride, s.classes, n, k)
        # (torch keeps it until the stream's work that uses it is done, and a captured graph has its own)
        room = torch.empty(size, dtype=torch.uint8, device=device) if size else None
        _call(torch, scores, "tgbm_scores_top", C.byref(s), C.byref(r), k, temperature, values.data_ptr(), classes.data_ptr(), lse.data_ptr(),
              room.data_ptr() if size else None, size)
    return values, classes, lse


def distill(scores, classes, teacher, labels=None, teacher_lse=None, temperature=1.0, weight=1.0, gradient=True):
    """The loss of class scores z against a teacher's best scores, float32 [rows], and the gradient pairs for the trees of the
    next boosting round, float32 [classes, rows, 2] (None where `gradient` is false).

    scores: float32, the rows of a class side by side.
    classes, teacher: int32 and a floating type, [rows, entries] with 1 to 128 entries in any order, as `top` lists them.
      Entries whose class is negative or no class of the student, or whose score is -inf, are left out; entries that name
      the same class add up.
    teacher_lse: float32 [rows], the teacher's log of the sum of exp(score / temperature) over all its classes, as `top` gives it for
      the same temperature. With it q = exp(teacher / T - teacher_lse), and what is left, r = 1 - sum(q), belongs to the classes
      that are not named, taken together; without it the entries' q add up to 1.
    labels: float32 [rows], class numbers; a row whose label is none has no part in the second term.

    With p = softmax(z / T) and R its part on the classes that are not named:
      loss = weight * T^2 * (sum(q * (log q - log p)) + r * (log r - log R)) + (1 - weight) * -log softmax(z)[label]
      gradient = weight * T * (M * p - q) + (1 - weight) * (softmax(z) - [label]); q of a class that is not named is r * p / R
      hessian = max(2 * (weight * M * p * (1 - p) + (1 - weight) * s * (1 - s)), 1e-16), s = softmax(z), like multi:softmax's.
    M = sum(q) + r is 1, but for rows with a teacher_lse where every class is named or the others' scores are all -inf (no class can take r, the loss has
    no such part, and M = sum(q)), or where sum(q) is above 1.

    Everything is 32 bits: terms of the size of log(classes) cancel in the loss of a student that is near its teacher, so about T^2 * 1e-6 of it is rounding;
    with a teacher_lse, q is off by up to 2^-23 of teacher / T. A q below 1e-38 is not counted in the loss."""
    torch = _torch()
    s = _scores(torch, "scores", scores)
    if s.type != 0 or (s.row_stride != 1 and s.rows > 1):
        raise ValueError("scores: float32 with the rows of a class side by side is wanted")
    n, C_ = s.rows, s.classes
    _on_gpu(torch, "teacher", teacher)
    kind = _types.get(teacher.dtype)
    if kind is None:
        raise ValueError("teacher: float32, float16 or bfloat16 is wanted, got %s" % teacher.dtype)
    if teacher.dim() != 2 or not 1 <= teacher.shape[1] <= 128:
        raise ValueError("teacher: [rows, entries] with 1 to 128 entries is wanted, got %s" % (tuple(teacher.shape),))
    entries = teacher.shape[1]
    t = _Teacher(_plain(torch, "classes", classes, scores, torch.int32, (n, entries)), _plain(torch, "teacher", teacher, scores, teacher.dtype, (n, entries)),
                 None if teacher_lse is None else _plain(torch, "teacher_lse", teacher_lse, scores, torch.float32, (n,)), kind, entries)
    if not 1e-3 <= temperature <= 1e3:
        raise ValueError("temperature is %r: 1e-3 to 1e3 is wanted" % (temperature,))
    if not 0 <= weight <= 1:
        raise ValueError("weight is %r: 0 to 1 is wanted" % (weight,))
    if labels is None and weight != 1:
        raise ValueError("weight is %r, and there are no labels" % (weight,))
    y = None if labels is None else _plain(torch, "labels", labels, scores, torch.float32, (n,))
    loss = torch.empty(n, dtype=torch.float32, device=scores.device)
    pairs = torch.empty((C_, n, 2), dtype=torch.float32, device=scores.device) if gradient else None
    if n:
        size = _distill_workspace(C_, n, entries)
        room = torch.empty(size, dtype=torch.uint8, device=scores.device) if size else None
        _call(torch, scores, "tgbm_scores_distill", C.byref(s), C.byref(t), y, temperature, weight, loss.data_ptr(),
              pairs.data_ptr() if gradient else None, n, room.data_ptr() if size else None, size)
    return loss, pairs


# what a setting of `sample` may be, for all rows alike
_FINE = {"temperature": (lambda v: v == 0 or 1e-6 <= v <= 1e6, "0 or 1e-6 to 1e6"), "p": (lambda v: 1e-37 <= v <= 1, "above 0 and up to 1"),
         "min_p": (lambda v: 0 <= v <= 1, "0 to 1"), "k": (lambda v: v >= 0, "0 or more")}


def _one_setting(name, v, fine, wanted):
    try:
        number = operator.index(v) if name == "k" else float(v)
    except (TypeError, ValueError, OverflowError):
        number = None
    if number is None or not fine(number):
        raise ValueError("%s is %r: %s is wanted" % (name, v, wanted))
    return number


def _setting(torch, name, v, scores, dtype, fine, wanted):
    """A setting of `sample`: (address of the rows' own, 0) or (None, everybody's)."""
    if (type(v) is int or (type(v) is float and name != "k")) and fine(v):
        return None, v
    if isinstance(v, torch.Tensor):
        return _plain(torch, name, v, scores, dtype, (scores.shape[1],)), 0
    return None, _one_setting(name, v, fine, wanted)


def sample(scores, u, k=0, p=1.0, min_p=0.0, temperature=1.0, bias=None, allowed=None, allowed_set=None, shown=None, shown_begin=None,
           repetition=1.0, frequency=0.0, presence=0.0):
    """A class of every row, drawn from softmax(score / temperature) of the scores as `adjust` would leave them: classes int32 [rows], and the
    logarithm of each one's probability among those that were kept, float32 [rows].

    u: float32 [rows], random numbers from 0 up to 1, not included (what is beyond counts as the ends). With the classes in falling order of their scores, of
      equal scores the lower class first, the first one is drawn where the sum of the probabilities passes u: 0 draws the best class.
    k: so many of the best classes are kept; 0: all.
    min_p: of those, the ones with at least min_p (0 to 1) of the best one's probability.
    p: of those, the fewest best ones that have at least p (above 0, up to 1) of their probability together.
    temperature: 0 takes the best class; else 1e-6 to 1e6.
    Each of these may be a tensor [rows], int32 (k) or float32, with a number for each row: there a k below 0 is all, a p of 0 or below leaves the best class, what is
    above 1 is 1, a min_p below 0 is 0, temperatures below 1e-6 are 0 and above 1e6 are that.

    Classes whose score is -inf or NaN are never drawn. A row that nothing is left of gets class -1 and -inf, one with a NaN among its numbers class -1 and NaN.
    Sums are 64 bits, of probabilities that are rounded by about 2^-46 of themselves at most (beyond 2^16 classes by more, 2^-40 at 2^22), and the same call draws the same
    classes; a class with less than 2^-64 of the best one's probability counts as one without."""
    torch = _torch()
    s = _scores(torch, "scores", scores)
    r = _rules(torch, scores, bias, allowed, allowed_set, shown, shown_begin, repetition, frequency, presence)
    n = s.rows
    at = _plain(torch, "u", u, scores, torch.float32, (n,))
    h = _Sampling()
    h.temperature, h.temperature_all = _setting(torch, "temperature", temperature, scores, torch.float32, *_FINE["temperature"])
    h.p, h.p_all = _setting(torch, "p", p, scores, torch.float32, *_FINE["p"])
    h.min_p, h.min_p_all = _setting(torch, "min_p", min_p, scores, torch.float32, *_FINE["min_p"])
    h.k, k = _setting(torch, "k", k, scores, torch.int32, *_FINE["k"])
    h.k_all = k = min(k, s.classes)
    classes = torch.empty(n, dtype=torch.int32, device=scores.device)
    logp = torch.empty(n, dtype=torch.float32, device=scores.device)
    if n:
        size = _sample_workspace(s.type, s.class_stride, s.row_stride, s.classes, n, r.shown is not None, k if h.k is None else None)
        room = torch.empty(size, dtype=torch.uint8, device=scores.device) if size else None
        _call(torch, scores, "tgbm_scores_sample", C.byref(s), C.byref(r), C.byref(h), at, classes.data_ptr(), logp.data_ptr(),
              room.data_ptr() if size else None, size)
    return classes, logp


def quantise(x):
    """Rows of numbers in 8 bits: (q int8 [rows, features], scale float32 [rows]), x being about q * scale[:, None].

    x: float32, float16 or bfloat16 [rows, features], the features of a row side by side, 1 to 65536 of them.
    scale is the row's largest magnitude / 127 and q the nearest whole number (of two the even one) to x / scale, 0 where the scale is 0. A row that
    holds an infinity or a NaN gets the scale NaN and zeros. Rows of q begin at multiples of 128 bytes, with zeros behind their features: as `linear`
    takes them without copying."""
    torch = _torch()
    r = _rows(torch, "x", x)
    width = (r.features + 127) // 128 * 128
    q = torch.empty((r.rows, width), dtype=torch.int8, device=x.device)
    scale = torch.empty(r.rows, dtype=torch.float32, device=x.device)
    if r.rows:
        _call(torch, x, "tgbm_rows_quantise", C.byref(r), q.data_ptr(), width, width, scale.data_ptr())
    return q[:, :r.features], scale


def linear(x, weight, weight_scale, bias=None, x_scale=None, order="row", dtype=None):
    """Class scores of a linear layer in 8 bits, [classes, rows]: (sum of x[i] * weight[c] over the features) * x_scale[i] * weight_scale[c] + bias[c].

    x: [rows, features], int8 with x_scale float32 [rows], or float32, float16 or bfloat16, which are quantised first as `quantise` does.
    weight, weight_scale: int8 [classes, features] and float32 [classes], as `quantise` makes them of the layer's weights, once. Rows that begin at multiples of 16
      bytes are read as they lie; others (and int8 rows of x whose features are no multiple of 128) are copied at every call.
    bias: float32 [classes].
    order: "row": the classes of a row side by side, "class": the rows of a class, as the trainer's operators want them.
    dtype: of the scores, float32 (the default), float16 or bfloat16.
    The sum is exact; the steps behind it are 32 bits, rounded once to the scores' type. A row whose scale is NaN has scores that are."""
    torch = _torch()
    r = _rows(torch, "x", x, x_scale, whole=True)
    w = _rows(torch, "weight", weight, weight_scale, whole=True, floating=False)
    if weight.device != x.device:
        raise ValueError("weight is on %s, x is on %s" % (weight.device, x.device))
    if w.features != r.features:
        raise ValueError("%d features of x, %d of the weights" % (r.features, w.features))
    if not 1 <= w.rows <= 1 << 22:
        raise ValueError("weight: %d classes" % w.rows)
    dtype = torch.float32 if dtype is None else dtype
    kind = _types.get(dtype)
    if kind is None:
        raise ValueError("dtype: float32, float16 or bfloat16 is wanted, got %s" % (dtype,))
    if order not in ("row", "class"):
        raise ValueError("order is %r: \"row\" or \"class\" is wanted" % (order,))
    b = None if bias is None else _plain(torch, "bias", bias, x, torch.float32, (w.rows,))
    n, classes = r.rows, w.rows
    if order == "row":
        out = torch.empty((n, classes), dtype=dtype, device=x.device).t()
        o = _Scores(out.data_ptr(), 1, classes, kind, classes, n)
    else:
        out = torch.empty((classes, n), dtype=dtype, device=x.device)
        o = _Scores(out.data_ptr(), max(n, 1), 1, kind, classes, n)
    if n:
        size = _linear_workspace(r.features, r.data % 16, r.pitch, r.type, n, r.padded, w.data % 16, w.pitch, w.type, classes, w.padded)
        room = torch.empty(size, dtype=torch.uint8, device=x.device) if size else None
        _call(torch, x, "tgbm_scores_linear", C.byref(r), C.byref(w), b, C.byref(o), room.data_ptr() if size else None, size)
    return out


def _apart(s, o, size):
    """Whether two arrays whose memory is interleaved share no element: parts of one larger array, side by side."""
    if (s.class_stride, s.row_stride) != (o.class_stride, o.row_stride):
        return False
    pitch, width = (s.class_stride, s.rows) if s.row_stride == 1 else (s.row_stride, s.classes)
    at = abs(o.data - s.data) // size % pitch
    return width <= at <= pitch - width
