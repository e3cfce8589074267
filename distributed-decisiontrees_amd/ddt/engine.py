"""Host-side mirror of the engine interface above the C-ABI (include/ddt.h).

The reference has no host software; what a host program must do is fixed by its hardware contract:
write the run parameters (CSR 201-207, rtl/DTEngine/EngineCSR.sv:190-248), stream the model
(weights lines then feature-index lines, rtl/DTEngine/PCIeReceiver.sv:136-139,230-275), stream tuples,
read back result lines (rtl/DTEngine/ResultsCombiner.sv:136-160).  `Engine` is that sequence as an
object: Engine(device) -> load_model(params, weights_lines, findex_lines) -> score(tuple_lines).
PyTorch is used only for device memory and streams.
"""
from __future__ import annotations

import ctypes as C

import numpy as np

from . import _lib
from ._lib import Info, Params, Stats

MISSING_DEFAULT = 0x7FC00000


class DDTError(RuntimeError):
    def __init__(self, code: int, detail: str = ""):
        self.code = code
        msg = _lib.lib().ddt_strerror(code).decode()
        super().__init__(f"ddt error {code} ({msg}){': ' + detail if detail else ''}")


def weights_lines_per_tree(D: int) -> int:
    return ((1 << (D + 1)) - 1 + 3) // 4


def findex_lines_per_tree(D: int) -> int:
    return ((1 << D) - 1 + 7) // 8


def tuple_words(F: int) -> int:
    return (F + 3) // 4 * 4


def shard_bounds(T: int, G: int):
    """Contiguous shards of ceil(T/G) trees in stream order: the split ddt_load_model_shard applies (PCIeReceiver.sv:241-264)."""
    per = (T + G - 1) // G
    return [(min(g * per, T), min((g + 1) * per, T)) for g in range(G)]


def default_clusters(T: int) -> int:
    """Smallest C in {1,2,4,8} whose 8 PUs x 16 trees x C slots hold T trees (DTPU.sv:74, Core.sv:291-316)."""
    for c in (1, 2, 4, 8):
        if T <= 128 * c:
            return c
    return 8


def make_params(T: int, D: int, F: int, missing_bits: int = MISSING_DEFAULT, cmp_mode: int = 0,
                clusters: int | None = None, sum_mode: int = 0) -> Params:
    p = Params()
    p.num_trees, p.num_levels, p.num_features, p.missing_bits = T, D, F, missing_bits
    p.weights_lines_per_tree, p.findex_lines_per_tree = weights_lines_per_tree(D), findex_lines_per_tree(D)
    p.cmp_mode, p.sum_mode = cmp_mode, sum_mode
    p.clusters_per_tuple = default_clusters(T) if clusters is None else clusters
    return p


def synth_model(T: int, D: int, F: int, dist: int = 0):
    """Deterministic synthetic model of SURVEY.md 8(d) in the reference wire format -> (wlines u32, flines u16)."""
    w = np.zeros(T * weights_lines_per_tree(D) * 4, np.uint32)
    f = np.zeros(T * findex_lines_per_tree(D) * 8, np.uint16)
    rc = _lib.lib().ddt_synth_model(T, D, F, dist, w.ctypes.data, f.ctypes.data)
    if rc:
        raise DDTError(rc)
    return w, f


def make_sparse_params(T: int, max_depth: int, F: int, missing_bits: int = MISSING_DEFAULT, cmp_mode: int = 0,
                       clusters: int | None = None, sum_mode: int = 0) -> Params:
    """Parameters of a SPARSE (explicit-children) model: num_levels is the depth bound, no lines-per-tree fields."""
    p = Params()
    p.num_trees, p.num_levels, p.num_features, p.missing_bits = T, max_depth, F, missing_bits
    p.cmp_mode, p.sum_mode = cmp_mode, sum_mode
    p.clusters_per_tuple = default_clusters(T) if clusters is None else clusters
    return p


def synth_sparse_model(T: int, max_depth: int, F: int, full_levels: int, split_permille: int, dist: int = 0):
    """Deterministic random-forest-like sparse model (include/ddt.h ddt_synth_sparse_model)
    -> (node_lines uint32 [n, 4], tree_first_line uint64 [T + 1])."""
    L = _lib.lib()
    first = np.zeros(T + 1, np.uint64)
    n = L.ddt_synth_sparse_model(T, max_depth, F, full_levels, split_permille, dist, None, 0, first.ctypes.data)
    if n < 0:
        raise DDTError(int(n))
    lines = np.zeros((n, 4), np.uint32)
    L.ddt_synth_sparse_model(T, max_depth, F, full_levels, split_permille, dist, lines.ctypes.data, n, first.ctypes.data)
    return lines, first


def synth_tuples_host(row0: int, n: int, F: int, dist: int = 0, missing_bits: int = MISSING_DEFAULT) -> np.ndarray:
    out = np.zeros((n, tuple_words(F)), np.uint32)
    rc = _lib.lib().ddt_synth_tuples_host(out.ctypes.data, row0, n, F, dist, missing_bits)
    if rc:
        raise DDTError(rc)
    return out


_types = None


def _torch_types():
    """What the class-score calls use of torch, looked up once (torch is imported where it is needed)."""
    global _types
    if _types is None:
        import types

        import torch

        raw = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda d: torch.cuda.current_stream(d).cuda_stream)
        _types = types.SimpleNamespace(
            torch=torch, f32=torch.float32, i32=torch.int32, u32=torch.uint32, i64=torch.int64, raw_stream=raw,
            grad_enabled=torch.is_grad_enabled, wrote=torch.autograd.graph.increment_version,
            codes={torch.float32: 0, torch.float16: 1, torch.bfloat16: 2})
    return _types


_distill_cls = None


def _distill_function():
    """The torch.autograd.Function behind Engine.distill (made on first use: torch is imported where it is needed)."""
    global _distill_cls
    if _distill_cls is None:
        import torch

        class Distill(torch.autograd.Function):
            @staticmethod
            def forward(ctx, engine, student, ids, values, lse, temperature):
                ctx.engine, ctx.temperature = engine, temperature
                ctx.save_for_backward(student, ids, values, lse)
                return engine.distill_device(student, ids, values, lse, temperature)

            @staticmethod
            @torch.autograd.function.once_differentiable
            def backward(ctx, weight):
                student, ids, values, lse = ctx.saved_tensors
                # the loss comes out of the same pass once more (n floats); nothing but the inputs is kept between the passes
                _, grad = ctx.engine.distill_grad_device(student, ids, values, lse, weight, ctx.temperature)
                return None, grad, None, None, None, None

        _distill_cls = Distill
    return _distill_cls


class Engine:
    """One engine == one GPU (the analogue of one FPGA running DTInference)."""

    def __init__(self, device: int = 0):
        self._L = _lib.lib()
        h = C.c_void_p()
        rc = self._L.ddt_create(C.byref(h), device)
        if rc:
            raise DDTError(rc, "ddt_create")
        self._h = h
        self.device = device
        self.params = None
        self.num_classes = 1

    def close(self):
        if getattr(self, "_h", None):
            self._L.ddt_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def _check(self, rc: int):
        if rc:
            raise DDTError(rc, self._L.ddt_last_error(self._h).decode())

    # ---- model ------------------------------------------------------------------------------------
    def load_model(self, params: Params, wlines: np.ndarray, flines: np.ndarray, shard_index: int = 0,
                   shard_count: int = 1):
        w = np.ascontiguousarray(wlines).view(np.uint32).reshape(-1)
        f = np.ascontiguousarray(flines).view(np.uint16).reshape(-1)
        self._check(self._L.ddt_load_model_shard(self._h, C.byref(params), w.ctypes.data, w.size // 4,
                                                 f.ctypes.data, f.size // 8, shard_index, shard_count))
        self.params = params
        self.num_classes = 1
        return self

    def load_model_sparse(self, params: Params, node_lines: np.ndarray, tree_first_line: np.ndarray,
                          shard_index: int = 0, shard_count: int = 1, num_classes: int = 1, interleaved: bool = True):
        """Sparse (explicit-children) forest: one 128-bit line per internal node (include/ddt.h ddt_load_model_sparse);
        num_classes > 1: one-vs-all classes in the stream (ddt_load_model_sparse_multiclass), scored with classify*()."""
        nl = np.ascontiguousarray(node_lines).view(np.uint32).reshape(-1, 4)
        first = np.ascontiguousarray(tree_first_line, dtype=np.uint64).reshape(-1)
        if first.size != params.num_trees + 1:
            raise ValueError("tree_first_line must hold num_trees + 1 entries")
        self._check(self._L.ddt_load_model_sparse_multiclass(self._h, C.byref(params), nl.ctypes.data, nl.shape[0], first.ctypes.data,
                                                             num_classes, int(interleaved), shard_index, shard_count))
        self.params = params
        self.num_classes = num_classes
        return self

    def load_model_multiclass(self, params: Params, wlines: np.ndarray, flines: np.ndarray, num_classes: int,
                              interleaved: bool = True, shard_index: int = 0, shard_count: int = 1):
        """One-vs-all ensemble of `num_classes` classes (an extension of the reference)."""
        w = np.ascontiguousarray(wlines).view(np.uint32).reshape(-1)
        f = np.ascontiguousarray(flines).view(np.uint16).reshape(-1)
        self._check(self._L.ddt_load_model_multiclass(self._h, C.byref(params), w.ctypes.data, w.size // 4,
                                                      f.ctypes.data, f.size // 8, num_classes, int(interleaved),
                                                      shard_index, shard_count))
        self.params = params
        self.num_classes = num_classes
        return self

    def classify(self, tuple_lines: np.ndarray, want_scores: bool = False):
        """Host buffers -> int32 labels [n] (and fp32 class scores [K, n])."""
        t = np.ascontiguousarray(tuple_lines).view(np.uint32).reshape(-1, tuple_words(self.params.num_features))
        n = t.shape[0]
        labels = np.empty(n, np.int32)
        cs = np.empty((self.num_classes, n), np.float32) if want_scores else None
        self._check(self._L.ddt_classify(self._h, t.ctypes.data, n, labels.ctypes.data,
                                         cs.ctypes.data if want_scores else None))
        return (labels, cs) if want_scores else labels

    def classify_device(self, d_tuples, class_scores=None, labels=None, want_labels: bool = True, stream=None):
        """torch CUDA tuple lines -> (labels int32 [n] or None, class scores fp32 [K, n]); asynchronous."""
        import torch

        W = tuple_words(self.params.num_features)
        n = d_tuples.numel() // W
        if class_scores is None:
            class_scores = torch.empty((self.num_classes, n), dtype=torch.float32, device=d_tuples.device)
        if labels is None and want_labels:
            labels = torch.empty(n, dtype=torch.int32, device=d_tuples.device)
        s = torch.cuda.current_stream(d_tuples.device) if stream is None else stream
        self._check(self._L.ddt_classify_device(self._h, d_tuples.data_ptr(), n, class_scores.data_ptr(),
                                                labels.data_ptr() if labels is not None else None, s.cuda_stream))
        return labels, class_scores

    def argmax_device(self, class_scores, labels=None, stream=None):
        import torch

        K, n = class_scores.shape
        if labels is None:
            labels = torch.empty(n, dtype=torch.int32, device=class_scores.device)
        s = torch.cuda.current_stream(class_scores.device) if stream is None else stream
        self._check(self._L.ddt_argmax_device(self._h, class_scores.data_ptr(), K, n, labels.data_ptr(), s.cuda_stream))
        return labels

    # ---- class scores: after the trees ---------------------------------------------------------------
    # Matrices are torch tensors [num_classes, n] as classify_device returns them; row-major logits [n, num_classes] go in as
    # logits.t() (a view: the strides say which it is).  Everything is asynchronous on `stream` (default: the device's current
    # one); results that are not handed in are allocated on it, so another stream that reads them waits for it first.  The caller's
    # tensors may be let go right after a call: their memory is not given out again before `stream` is done with them.  The checks
    # are written for the calls that take less time on the device than in Python: no context, device or dtype object is made on the
    # way through.
    # No gradient goes through adjust_device, top_device and distill*_device (distill is the call with one): a result that autograd
    # would have to see written is refused, and every caller's tensor that is written counts as modified in place (_version), so that
    # a backward pass that saved it says so.
    def _tensor(self, t, what: str, dtype, shape=None) -> int:
        if not t.is_cuda or t.get_device() != self.device:
            raise ValueError(f"{what}: on {t.device}, the engine is on cuda:{self.device}")
        if t.dtype is not dtype:
            raise ValueError(f"{what}: {t.dtype}, must be {dtype}")
        if shape is not None and t.shape != shape:
            raise ValueError(f"{what}: shape {tuple(t.shape)}, must be {shape}")
        return t.data_ptr()

    def _packed(self, t, what: str, dtype, shape) -> int:
        p = self._tensor(t, what, dtype, shape)
        if not t.is_contiguous():
            raise ValueError(f"{what}: must be contiguous")
        return p

    @staticmethod
    def _result(t, what: str):
        """a caller's tensor that the call writes"""
        if t.requires_grad and _torch_types().grad_enabled():
            raise ValueError(f"{what}: requires grad and would be written without autograd's knowledge (torch.no_grad(), or detach it)")
        return t

    def _scores(self, t, what: str, rows: int = 1) -> _lib.Scores:
        """ddt_scores_t of a tensor whose dimension `rows` counts the rows"""
        code = _torch_types().codes.get(t.dtype)
        if code is None:
            raise ValueError(f"{what}: {t.dtype}, must be one of {list(_torch_types().codes)}")
        if t.dim() != 2:
            raise ValueError(f"{what}: {t.dim()} dimensions, must be 2")
        if not t.is_cuda or t.get_device() != self.device:
            raise ValueError(f"{what}: on {t.device}, the engine is on cuda:{self.device}")
        a, b = t.shape
        c, d = t.stride()
        return _lib.Scores(t.data_ptr(), b, d, c, a, code) if rows else _lib.Scores(t.data_ptr(), a, c, d, b, code)

    def _stream(self, stream, *used):
        """handle of the stream of a call, which uses these tensors"""
        if stream is None:
            return _torch_types().raw_stream(self.device)
        if stream.device_index != self.device:
            raise ValueError(f"stream: of cuda:{stream.device_index}, the engine is on cuda:{self.device}")
        for t in used:
            if t is not None:
                t.record_stream(stream)
        return stream.cuda_stream

    @staticmethod
    def _allocator(like, stream):
        """like.new_empty on the stream of the call"""
        if stream is None:
            return like.new_empty

        def on_stream(*args, **kw):
            with _torch_types().torch.cuda.stream(stream):
                return like.new_empty(*args, **kw)

        return on_stream

    def adjust_device(self, class_scores, bias=None, allowed=None, history=None, history_first=None, history_prompt=None,
                      repetition=None, frequency=None, presence=None, out=None, stream=None):
        """Penalties for repeated classes, biases and a mask on class scores [K, n] (fp32, fp16, bf16) -> adjusted scores, same type
        and layout (ddt_adjust_scores_device; `out` may be `class_scores`).

        bias            fp32 [K] (the base scores of an imported model, say) or [K, n], any strides
        allowed         int32 / uint32 bits, class c at bit c % 32 of word c // 32: [ceil(K / 32)] or [n, ceil(K / 32)]; others get -inf
        history         int32 classes; row r's are history[history_first[r] : history_first[r + 1]] (int64 [n + 1]), the first
                        history_prompt[r] (int32 [n]) of them its prompt part
        repetition      fp32 [n]: a class of the history: score / it if positive, else score * it
        frequency       fp32 [n]: minus it for every time the class stands behind the prompt part
        presence        fp32 [n]: minus it if it stands there at all"""
        T = _torch_types()
        s = self._scores(class_scores, "class_scores")
        K, n = s.num_classes, s.rows
        a = _lib.Adjust()
        if bias is not None:
            a.bias = self._tensor(bias, "bias", T.f32)
            if bias.shape == (K,):
                a.bias_class_stride = bias.stride(0)
            elif bias.shape == (K, n):
                a.bias_class_stride, a.bias_row_stride = bias.stride()
            else:
                raise ValueError(f"bias: shape {tuple(bias.shape)}, must be {(K,)} or {(K, n)}")
        if allowed is not None:
            words = (K + 31) // 32
            a.allowed = self._tensor(allowed, "allowed", T.u32 if allowed.dtype is T.u32 else T.i32)
            if allowed.shape != (words,) and allowed.shape != (n, words):
                raise ValueError(f"allowed: shape {tuple(allowed.shape)}, must be {(words,)} or {(n, words)}")
            if words > 1 and allowed.stride(-1) != 1:
                raise ValueError("allowed: the words of a row must be contiguous")
            a.allowed_row_stride = allowed.stride(0) if n > 1 and allowed.dim() == 2 else 0
        if history is not None:
            if history_first is None:
                raise ValueError("history without history_first")
            a.history_len = history.numel()
            a.history = self._packed(history, "history", T.i32, (a.history_len,))
            a.history_first = self._packed(history_first, "history_first", T.i64, (n + 1,))
            if history_prompt is not None:
                a.history_prompt = self._packed(history_prompt, "history_prompt", T.i32, (n,))
            if repetition is not None:
                a.repetition = self._packed(repetition, "repetition", T.f32, (n,))
            if frequency is not None:
                a.frequency = self._packed(frequency, "frequency", T.f32, (n,))
            if presence is not None:
                a.presence = self._packed(presence, "presence", T.f32, (n,))
        elif not (history_first is None and history_prompt is None and repetition is None and frequency is None and presence is None):
            raise ValueError("history_first, history_prompt and penalties need a history")
        given = out
        if out is None:
            row_major = s.class_stride == 1 and (s.row_stride >= K or n <= 1)
            new = self._allocator(class_scores, stream)
            out = new((n, K)).t() if row_major else new((K, n))
            o = _lib.Scores(out.data_ptr(), n, K if row_major else 1, 1 if row_major else n, K, s.dtype)
        else:
            o = self._scores(self._result(out, "out"), "out")
        self._check(self._L.ddt_adjust_scores_device(self._h, C.byref(s), C.byref(a), C.byref(o),
                                                     self._stream(stream, class_scores, bias, allowed, history, history_first, history_prompt, repetition,
                                                                  frequency, presence, out)))
        if given is not None:
            T.wrote(given)
        return out

    def top_device(self, class_scores, k: int, temperature: float = 1.0, ids=None, values=None, lse=None, stream=None):
        """The k best classes of each row of class scores [K, n], best first, equal scores in the order of the classes ->
        (ids int32 [n, k], values fp32 [n, k], lse fp32 [n] = log sum exp(score / temperature) over all classes): the class's
        probability is exp(values / temperature - lse).  Rows with fewer candidates (NaN and -inf are none) end in id -1, value
        -inf.  (ddt_top_scores_device)"""
        T = _torch_types()
        s = self._scores(class_scores, "class_scores")
        n = s.rows
        given = [t for t in (ids, values, lse) if t is not None]
        new = self._allocator(class_scores, stream)
        if ids is None:
            ids = new((n, k), dtype=T.i32)
            p_ids = ids.data_ptr()
        else:
            p_ids = self._packed(self._result(ids, "ids"), "ids", T.i32, (n, k))
        if values is None:
            values = new((n, k), dtype=T.f32)
            p_values = values.data_ptr()
        else:
            p_values = self._packed(self._result(values, "values"), "values", T.f32, (n, k))
        if lse is None:
            lse = new((n,), dtype=T.f32)
            p_lse = lse.data_ptr()
        else:
            p_lse = self._packed(self._result(lse, "lse"), "lse", T.f32, (n,))
        self._check(self._L.ddt_top_scores_device(self._h, C.byref(s), k, temperature, p_ids, p_values, p_lse,
                                                  self._stream(stream, class_scores, ids, values, lse)))
        if given:
            T.wrote(given)
        return ids, values, lse

    def top_classes_device(self, d_tuples, k: int, temperature: float = 1.0, stream=None, **adjust):
        """Tuple lines -> (ids, values, lse) of top_device: classify_device's class sums, adjust_device with the keywords given here
        (bias = an imported model's base scores, allowed, histories ...), top_device.  k = 1 is the label; a larger k is what a
        student network learns from (distill)."""
        import contextlib

        import torch

        self._stream(stream, d_tuples, *adjust.values())
        with contextlib.nullcontext() if stream is None else torch.cuda.stream(stream):
            _, scores = self.classify_device(d_tuples, want_labels=False)
            if adjust:
                self.adjust_device(scores, out=scores, **adjust)
            return self.top_device(scores, k, temperature)

    def _teacher(self, n, ids, values, lse, temperature) -> _lib.Teacher:
        T = _torch_types()
        k = ids.shape[-1] if ids.dim() else 0
        p, v = self._tensor(ids, "ids", T.i32, (n, k)), self._tensor(values, "values", T.f32, (n, k))
        by_row, by_entry = ids.stride()
        if n > 1 and by_row != values.stride(0) or k > 1 and (by_entry != 1 or values.stride(1) != 1):
            raise ValueError("ids, values: rows must be contiguous and stand equally far apart")
        return _lib.Teacher(p, v, by_row if n > 1 else k, None if lse is None else self._packed(lse, "lse", T.f32, (n,)), k, temperature)

    def distill_device(self, student, ids, values, lse=None, temperature: float = 1.0, loss=None, stream=None):
        """KL divergence of a student's softmax (scores [n, K], row-major) from a teacher's top scores (ids, values, lse of
        top_device at the same temperature) -> loss fp32 [n].  lse None: the teacher's probabilities are normalised over the
        listed classes; otherwise everything it does not list is one more outcome.  +inf where the teacher has a probability and the
        student, at -inf, has none.  (ddt_distill_device)"""
        T = _torch_types()
        s = self._scores(student, "student", rows=0)
        t = self._teacher(s.rows, ids, values, lse, temperature)
        given = loss
        if loss is None:
            loss = self._allocator(student, stream)((s.rows,), dtype=T.f32)
            p_loss = loss.data_ptr()
        else:
            p_loss = self._packed(self._result(loss, "loss"), "loss", T.f32, (s.rows,))
        self._check(self._L.ddt_distill_device(self._h, C.byref(s), C.byref(t), p_loss,
                                               self._stream(stream, student, ids, values, lse, loss)))
        if given is not None:
            T.wrote(given)
        return loss

    def distill_grad_device(self, student, ids, values, lse=None, row_weight=None, temperature: float = 1.0, loss=None, grad=None,
                            stream=None):
        """distill_device and, from the same pass over the student's scores, the gradient of sum(row_weight * loss) by them ->
        (loss fp32 [n], grad [n, K] of the student's type); row_weight fp32 [n] (any stride; None = 1), `grad` may be `student`.
        (ddt_distill_grad_device)"""
        T = _torch_types()
        s = self._scores(student, "student", rows=0)
        n = s.rows
        t = self._teacher(n, ids, values, lse, temperature)
        w, w_stride = None, 0
        if row_weight is not None:
            w, w_stride = self._tensor(row_weight, "row_weight", T.f32, (n,)), row_weight.stride(0) if n > 1 else 0
        given = [t for t in (loss, grad) if t is not None]
        new = self._allocator(student, stream)
        if loss is None:
            loss = new((n,), dtype=T.f32)
            p_loss = loss.data_ptr()
        else:
            p_loss = self._packed(self._result(loss, "loss"), "loss", T.f32, (n,))
        if grad is None:
            grad = new((n, s.num_classes))
            g = _lib.Scores(grad.data_ptr(), n, s.num_classes, 1, s.num_classes, s.dtype)
        else:
            g = self._scores(self._result(grad, "grad"), "grad", rows=0)
        self._check(self._L.ddt_distill_grad_device(self._h, C.byref(s), C.byref(t), w, w_stride, p_loss, C.byref(g),
                                                    self._stream(stream, student, ids, values, lse, row_weight, loss, grad)))
        if given:
            T.wrote(given)
        return loss, grad

    def distill(self, student, ids, values, lse=None, temperature: float = 1.0):
        """distill_device for training: loss fp32 [n] that autograd takes back to `student` (the teacher gets no gradient)."""
        return _distill_function().apply(self, student, ids, values, lse, temperature)

    def set_option(self, key: str, value: int):
        self._check(self._L.ddt_set_option(self._h, key.encode(), int(value)))

    # ---- scoring ----------------------------------------------------------------------------------
    def score(self, tuple_lines: np.ndarray, out: np.ndarray | None = None) -> np.ndarray:
        """Host buffers through the pinned, pipelined feeder (the PCIe tuple stream); buffers pinned with host_register skip the staging."""
        t = np.ascontiguousarray(tuple_lines).view(np.uint32)
        if self.params is None:  # let the library report DDT_ESTATE
            self._check(self._L.ddt_score(self._h, t.ctypes.data, 1, t.ctypes.data))
        W = tuple_words(self.params.num_features)
        t = t.reshape(-1, W)
        if out is None:
            out = np.empty(t.shape[0], np.float32)
        assert out.dtype == np.float32 and out.flags.c_contiguous and out.size >= t.shape[0]
        self._check(self._L.ddt_score(self._h, t.ctypes.data, t.shape[0], out.ctypes.data))
        return out

    def host_register(self, a: np.ndarray) -> bool:
        """Pin a host array for this engine's device (ddt_host_register): ddt_score then DMAs it directly.  -> is it pinned?  (A driver
        that does not pin memory that exists already leaves it to be staged like any other.)"""
        assert a.flags.c_contiguous
        self._check(self._L.ddt_host_register(self._h, a.ctypes.data, a.nbytes))
        return self.host_pinned(a)

    def host_pinned(self, a: np.ndarray) -> bool:
        """Does ddt_score move this array directly (ddt_host_pinned)?"""
        return self._L.ddt_host_pinned(self._h, a.ctypes.data, a.nbytes) == 1

    def host_unregister(self, a: np.ndarray):
        self._check(self._L.ddt_host_unregister(self._h, a.ctypes.data))

    def score_device(self, d_tuples, out=None, stream=None):
        """torch CUDA tensor of tuple lines ([n, W] int32/uint32/float32) -> torch float32 [n], asynchronous."""
        import torch

        W = tuple_words(self.params.num_features)
        assert d_tuples.is_cuda and d_tuples.is_contiguous() and d_tuples.element_size() == 4
        n = d_tuples.numel() // W
        if out is None:
            out = torch.empty(n, dtype=torch.float32, device=d_tuples.device)
        assert out.is_cuda and out.is_contiguous() and out.dtype == torch.float32 and out.numel() >= n
        s = torch.cuda.current_stream(d_tuples.device) if stream is None else stream
        self._check(self._L.ddt_score_device(self._h, d_tuples.data_ptr(), n, out.data_ptr(), s.cuda_stream))
        return out

    def chain_sum_device(self, parts, out=None, stream=None):
        """parts: torch float32 [G, n] -> out[n] = (((p0+p1)+p2)+...) in the reference's chain order."""
        import torch

        assert parts.is_cuda and parts.is_contiguous() and parts.dtype == torch.float32 and parts.dim() == 2
        G, n = parts.shape
        if out is None:
            out = torch.empty(n, dtype=torch.float32, device=parts.device)
        s = torch.cuda.current_stream(parts.device) if stream is None else stream
        self._check(self._L.ddt_chain_sum_device(self._h, parts.data_ptr(), G, n, out.data_ptr(), s.cuda_stream))
        return out

    def synth_tuples_device(self, row0: int, n: int, F: int, dist: int = 0, missing_bits: int = MISSING_DEFAULT,
                            out=None, stream=None):
        import torch

        W = tuple_words(F)
        if out is None:
            out = torch.empty((n, W), dtype=torch.int32, device=f"cuda:{self.device}")
        s = torch.cuda.current_stream(out.device) if stream is None else stream
        self._check(self._L.ddt_synth_tuples_device(self._h, out.data_ptr(), row0, n, F, dist, missing_bits,
                                                    s.cuda_stream))
        return out

    # ---- introspection ----------------------------------------------------------------------------
    def info(self) -> Info:
        i = Info()
        self._check(self._L.ddt_get_info(self._h, C.byref(i)))
        return i

    def stats(self) -> Stats:
        s = Stats()
        self._check(self._L.ddt_get_stats(self._h, C.byref(s)))
        return s


def variant_names():
    L = _lib.lib()
    out = []
    for v in range(L.ddt_num_variants()):
        b = C.create_string_buffer(64)
        L.ddt_variant_name(v, b, 64)
        out.append(b.value.decode())
    return out


COMBINE_ALLREDUCE, COMBINE_CHAIN = 0, 1
COMM_ID_BYTES = 128


def hybrid_rows(n: int, row_groups: int, row_group: int):
    """rows [lo, hi) of a row group of a hybrid job (ddt_hybrid_rows)"""
    lo, hi = C.c_size_t(), C.c_size_t()
    rc = _lib.lib().ddt_hybrid_rows(n, row_groups, row_group, C.byref(lo), C.byref(hi))
    if rc:
        raise DDTError(rc, "ddt_hybrid_rows")
    return lo.value, hi.value


def comm_unique_id() -> bytes:
    """ncclGetUniqueId through the C-ABI: rank 0 makes it, the launcher hands it to every rank."""
    buf = C.create_string_buffer(COMM_ID_BYTES)
    rc = _lib.lib().ddt_comm_get_unique_id(buf)
    if rc:
        raise DDTError(rc, "ddt_comm_get_unique_id")
    return buf.raw


class Comm:
    """One rank of a multi-GPU job: an RCCL communicator bound to an Engine (include/ddt.h ddt_comm_*).  The sharded
    calls are collective: every rank calls them with the same arguments."""

    def __init__(self, engine: Engine, rank: int, n_ranks: int, unique_id: bytes, tree_ranks: int = 0):
        """tree_ranks = 0: a plain communicator (tree-sharded over all ranks, or row-sharded replicas).  tree_ranks = Gt >= 1: the hybrid
        layout (ddt_comm_create_hybrid) -- row groups of Gt consecutive ranks, the engine must hold tree shard rank % Gt of Gt."""
        self._L, self.engine, self.rank, self.n_ranks, self.tree_ranks = _lib.lib(), engine, rank, n_ranks, tree_ranks
        assert len(unique_id) == COMM_ID_BYTES
        h = C.c_void_p()
        if tree_ranks:
            rc = self._L.ddt_comm_create_hybrid(C.byref(h), engine._h, rank, n_ranks, tree_ranks, unique_id)
        else:
            rc = self._L.ddt_comm_create(C.byref(h), engine._h, rank, n_ranks, unique_id)
        if rc:
            raise DDTError(rc, self._L.ddt_last_error(engine._h).decode())
        self._h = h

    def layout(self):
        lay = _lib.CommLayout()
        self._check(self._L.ddt_comm_layout(self._h, C.byref(lay)))
        return lay

    def abort(self):
        """A peer failed: free this rank's queued collectives (ddt_comm_abort); the communicator is dead afterwards."""
        self._check(self._L.ddt_comm_abort(self._h))

    def score_hybrid(self, d_tuples, out=None, combine: int = COMBINE_ALLREDUCE, gather: bool = True, stream=None):
        """Hybrid job: this rank's row group scores its slice of the rows against the group's tree shards; gather: all rows on every rank."""
        import torch

        n, s = self._args(d_tuples, stream)
        if out is None:
            out = torch.empty(n, dtype=torch.float32, device=d_tuples.device)
        self._check(self._L.ddt_score_hybrid_device(self._h, d_tuples.data_ptr(), n, out.data_ptr(), combine, 1 if gather else 0, s.cuda_stream))
        return out

    def classify_hybrid(self, d_tuples, combine: int = COMBINE_ALLREDUCE, gather: bool = True, want_labels: bool = True, stream=None,
                        class_scores=None, labels=None):
        import torch

        n, s = self._args(d_tuples, stream)
        cs = class_scores if class_scores is not None else torch.empty((self.engine.num_classes, n), dtype=torch.float32, device=d_tuples.device)
        if labels is None and want_labels:
            labels = torch.empty(n, dtype=torch.int32, device=d_tuples.device)
        want_labels = labels is not None
        self._check(self._L.ddt_classify_hybrid_device(self._h, d_tuples.data_ptr(), n, cs.data_ptr(), labels.data_ptr() if want_labels else None,
                                                       combine, 1 if gather else 0, s.cuda_stream))
        return labels, cs

    def close(self):
        if getattr(self, "_h", None):
            self._L.ddt_comm_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def _check(self, rc: int):
        if rc:
            raise DDTError(rc, self._L.ddt_comm_last_error(self._h).decode())

    def set_option(self, key: str, value: int):
        self._check(self._L.ddt_comm_set_option(self._h, key.encode(), int(value)))

    def _args(self, d_tuples, stream):
        import torch

        W = tuple_words(self.engine.params.num_features)
        assert d_tuples.is_cuda and d_tuples.is_contiguous() and d_tuples.element_size() == 4
        s = torch.cuda.current_stream(d_tuples.device) if stream is None else stream
        return d_tuples.numel() // W, s

    def score_sharded(self, d_tuples, out=None, combine: int = COMBINE_ALLREDUCE, stream=None):
        """Tree-sharded job: tuples replicated on every rank -> full fp32 scores on every rank (asynchronous)."""
        import torch

        n, s = self._args(d_tuples, stream)
        if out is None:
            out = torch.empty(n, dtype=torch.float32, device=d_tuples.device)
        self._check(self._L.ddt_score_sharded_device(self._h, d_tuples.data_ptr(), n, out.data_ptr(), combine, s.cuda_stream))
        return out

    def score(self, tuple_lines: np.ndarray, combine: int = COMBINE_ALLREDUCE) -> np.ndarray:
        """Host buffers (ddt_comm_score): with peers the tuples cross PCIe once (1/n per rank) and travel on over xGMI; every rank
        gets the combined scores.  Collective and synchronous."""
        t = np.ascontiguousarray(tuple_lines).view(np.uint32).reshape(-1, tuple_words(self.engine.params.num_features))
        out = np.empty(t.shape[0], np.float32)
        self._check(self._L.ddt_comm_score(self._h, t.ctypes.data, t.shape[0], out.ctypes.data, combine))
        return out

    def score_rowsharded(self, d_tuples, out=None, stream=None):
        """Row-sharded job ("replicas only"): every rank holds the whole ensemble and scores its slice of the rows."""
        import torch

        n, s = self._args(d_tuples, stream)
        if out is None:
            out = torch.empty(n, dtype=torch.float32, device=d_tuples.device)
        self._check(self._L.ddt_score_rowsharded_device(self._h, d_tuples.data_ptr(), n, out.data_ptr(), s.cuda_stream))
        return out

    def classify_sharded(self, d_tuples, combine: int = COMBINE_ALLREDUCE, want_labels: bool = True, stream=None,
                         class_scores=None, labels=None):
        """-> (labels int32 [n] or None, combined class scores fp32 [K, n])"""
        import torch

        n, s = self._args(d_tuples, stream)
        cs = class_scores if class_scores is not None else torch.empty((self.engine.num_classes, n), dtype=torch.float32, device=d_tuples.device)
        if labels is None and want_labels:
            labels = torch.empty(n, dtype=torch.int32, device=d_tuples.device)
        want_labels = labels is not None
        self._check(self._L.ddt_classify_sharded_device(self._h, d_tuples.data_ptr(), n, cs.data_ptr(),
                                                        labels.data_ptr() if want_labels else None, combine, s.cuda_stream))
        return labels, cs


class Group:
    """Single-process multi-GPU job (include/ddt.h ddt_group_*): n engines + one RCCL communicator over them."""

    def __init__(self, device_ids, tree_ranks: int = 0):
        """tree_ranks = Gt >= 1: the hybrid layout (row groups of Gt consecutive devices, ddt_group_create_hybrid)"""
        self._L = _lib.lib()
        ids = (C.c_int * len(device_ids))(*device_ids)
        h = C.c_void_p()
        rc = (self._L.ddt_group_create_hybrid(C.byref(h), len(device_ids), ids, tree_ranks) if tree_ranks
              else self._L.ddt_group_create(C.byref(h), len(device_ids), ids))
        if rc:
            raise DDTError(rc, "ddt_group_create")
        self._h, self.n, self.params = h, len(device_ids), None

    def close(self):
        if getattr(self, "_h", None):
            self._L.ddt_group_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def _check(self, rc: int):
        if rc:
            raise DDTError(rc, self._L.ddt_group_last_error(self._h).decode())

    def load_model(self, params: Params, wlines: np.ndarray, flines: np.ndarray):
        w = np.ascontiguousarray(wlines).view(np.uint32).reshape(-1)
        f = np.ascontiguousarray(flines).view(np.uint16).reshape(-1)
        self._check(self._L.ddt_group_load_model(self._h, C.byref(params), w.ctypes.data, w.size // 4, f.ctypes.data, f.size // 8))
        self.params = params
        return self

    def load_model_sparse(self, params: Params, node_lines: np.ndarray, tree_first_line: np.ndarray):
        nl = np.ascontiguousarray(node_lines).view(np.uint32).reshape(-1, 4)
        first = np.ascontiguousarray(tree_first_line, dtype=np.uint64).reshape(-1)
        self._check(self._L.ddt_group_load_model_sparse(self._h, C.byref(params), nl.ctypes.data, nl.shape[0], first.ctypes.data))
        self.params = params
        return self

    def load_model_multiclass(self, params: Params, wlines: np.ndarray, flines: np.ndarray, num_classes: int, interleaved: bool = True):
        w = np.ascontiguousarray(wlines).view(np.uint32).reshape(-1)
        f = np.ascontiguousarray(flines).view(np.uint16).reshape(-1)
        self._check(self._L.ddt_group_load_model_multiclass(self._h, C.byref(params), w.ctypes.data, w.size // 4, f.ctypes.data, f.size // 8,
                                                             num_classes, 1 if interleaved else 0))
        self.params, self.num_classes = params, num_classes
        return self

    def load_model_replicated(self, params: Params, wlines: np.ndarray, flines: np.ndarray):
        """Every device holds the whole ensemble (the reference's tuple-partitioned mode): use with score_rows()."""
        w = np.ascontiguousarray(wlines).view(np.uint32).reshape(-1)
        f = np.ascontiguousarray(flines).view(np.uint16).reshape(-1)
        self._check(self._L.ddt_group_load_model_replicated(self._h, C.byref(params), w.ctypes.data, w.size // 4, f.ctypes.data, f.size // 8))
        self.params = params
        return self

    def score_rows(self, tuple_lines: np.ndarray) -> np.ndarray:
        """Device d scores its share of the rows through its own feeder; no collective."""
        t = np.ascontiguousarray(tuple_lines).view(np.uint32).reshape(-1, tuple_words(self.params.num_features))
        out = np.empty(t.shape[0], np.float32)
        self._check(self._L.ddt_group_score_rows(self._h, t.ctypes.data, t.shape[0], out.ctypes.data))
        return out

    def score(self, tuple_lines: np.ndarray, combine: int = COMBINE_ALLREDUCE) -> np.ndarray:
        t = np.ascontiguousarray(tuple_lines).view(np.uint32).reshape(-1, tuple_words(self.params.num_features))
        out = np.empty(t.shape[0], np.float32)
        self._check(self._L.ddt_group_score(self._h, t.ctypes.data, t.shape[0], out.ctypes.data, combine))
        return out

    def classify(self, tuple_lines: np.ndarray, combine: int = COMBINE_ALLREDUCE, want_scores: bool = True):
        """labels [n] int32 and (optionally) the combined per-class sums [num_classes][n]."""
        t = np.ascontiguousarray(tuple_lines).view(np.uint32).reshape(-1, tuple_words(self.params.num_features))
        labels = np.empty(t.shape[0], np.int32)
        cs = np.empty((self.num_classes, t.shape[0]), np.float32) if want_scores else None
        self._check(self._L.ddt_group_classify(self._h, t.ctypes.data, t.shape[0], labels.ctypes.data, cs.ctypes.data if want_scores else None, combine))
        return labels, cs
