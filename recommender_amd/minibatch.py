"""Minibatch operators on factor tables: what a training step over batches needs next to the rating-by-rating kernels.

    embedding           rows of a table by id, scaled                     (beside the implicit term's gather, z = sum y[j] / sqrt N)
    embedding_grad      its gradient, by sorted tokens
    softmax_loss        softmax cross entropy against the whole catalogue (beside ExplicitMF.top_n: the same scores, which
    softmax_loss_grads  ... and its gradients                              are never stored here either)
    grad_norm           global norm of a set of gradients
    clip_grads          ... and their clipping by it

The reference has no counterpart: it updates rating by rating.  All arguments are torch ROCm tensors on one device, float32 or
bfloat16; ids and targets are int32, and a negative one is padding.  Every call runs on the current stream of that device
without waiting for it, allocates through torch only, and can be captured into a graph.  Results are the same bits on every
call.  There is no autograd: a gradient is its own call."""
from array import array

import torch

from . import _abi

_DTYPES = {torch.float32: 0, torch.bfloat16: 1}       # MFSGD_F32, MFSGD_BF16


def _rows(t, name):
    """(tensor, row stride) of a two-dimensional tensor whose rows are contiguous; others are copied."""
    if not isinstance(t, torch.Tensor) or t.dim() != 2:
        raise ValueError(f"{name} must be a two-dimensional tensor")
    if t.dtype not in _DTYPES:
        raise TypeError(f"{name} must be float32 or bfloat16, not {t.dtype}")
    n, d = t.shape
    if d < 1:
        raise ValueError(f"{name} has rows of no elements")
    if (d > 1 and t.stride(1) != 1) or (n > 1 and t.stride(0) < d):
        t = t.contiguous()
    return t, (t.stride(0) if n > 1 else d)


def _ids(t, name):
    if not isinstance(t, torch.Tensor) or t.dtype != torch.int32:
        raise TypeError(f"{name} must be an int32 tensor")
    return t.contiguous()


def _vector(t, n, name):
    if t is None:
        return None
    if not isinstance(t, torch.Tensor) or t.dtype != torch.float32 or t.shape != (n,):
        raise ValueError(f"{name} must be a float32 tensor of {n} elements")
    return t.contiguous()


class _On:
    """Makes the tensors' device current for a call and holds its stream; all tensors must be on that one device."""

    def __init__(self, *tensors):
        _abi.require_gpu()
        self.device = tensors[0].device
        index = tensors[0].get_device()
        for t in tensors:
            if t is not None and (t.get_device() != index or index < 0):
                raise ValueError("all tensors must be on one ROCm device")
        self.guard = None

    def __enter__(self):
        index = self.device.index
        if index != torch.cuda.current_device():
            self.guard = torch.cuda.device(self.device)
            self.guard.__enter__()
        self.stream = torch._C._cuda_getCurrentRawStream(index)
        return self

    def __exit__(self, *exc):
        if self.guard is not None:
            self.guard.__exit__(*exc)

    def workspace(self, nbytes):
        if nbytes < 0:
            raise ValueError("the batch or the table is too large")
        return torch.empty(nbytes, dtype=torch.uint8, device=self.device)


def _span(t):
    """Addresses a tensor reaches, or None if it holds nothing."""
    if t.numel() == 0:
        return None
    last = sum((n - 1) * s for n, s in zip(t.shape, t.stride()))
    return t.data_ptr(), t.data_ptr() + (last + 1) * t.element_size()


def _overlap(a, b):
    x, y = _span(a), _span(b)
    return x is not None and y is not None and x[0] < y[1] and y[0] < x[1]


def _share(a, b):
    """Whether two tensors have elements in common.  Columns of one wider table have not, though their spans overlap; other
    tensors with overlapping spans are taken to."""
    if not _overlap(a, b):
        return False
    wide = a.stride(0)
    if a.dtype != b.dtype or b.stride(0) != wide or any(t.dim() == 2 and t.shape[1] > 1 and t.stride(1) != 1 for t in (a, b)):
        return True
    apart, rest = divmod(b.data_ptr() - a.data_ptr(), a.element_size())
    widths = [t.shape[1] if t.dim() == 2 else 1 for t in (a, b)]
    apart %= max(wide, 1)                               # b's columns begin here in a's rows, and a's next row behind them
    return bool(rest) or apart < widths[0] or apart + widths[1] > wide


def embedding(table, ids, scale=1.0):
    """scale * table[ids]: [*ids.shape, d] of the table's type.  A negative id gives a zero row, an id behind the table a row
    that is not a number."""
    table, stride = _rows(table, "table")
    ids = _ids(ids, "ids")
    n_rows, d = table.shape
    with _On(table, ids) as on:
        out = torch.empty((*ids.shape, d), dtype=table.dtype, device=table.device)
        _abi.check(_abi.lib().mfsgd_hip_embedding(table.data_ptr(), stride, n_rows, d, ids.data_ptr(), ids.numel(), scale,
                                                  _DTYPES[table.dtype], out.data_ptr(), on.stream))
    return out


def embedding_grad(grad, ids, n_rows, scale=1.0, out=None, accumulate=False):
    """Gradient of `embedding` for its table: [n_rows, d], row v = scale * the sum of grad's rows whose id is v (in fp32; up to
    16 of them in the order of ids, more in stretches that the whole batch's ids decide), zero where no id is v.  `grad` is
    [*ids.shape, d].  With `out` the result is written there; with `accumulate` it is added to `out` (one gradient of a table
    used twice; or, with scale = -learning rate, the update of the table itself), whose other rows stay untouched."""
    if not isinstance(grad, torch.Tensor) or grad.dim() < 1:
        raise ValueError("grad must be a tensor")
    ids = _ids(ids, "ids")
    if tuple(grad.shape[:-1]) != tuple(ids.shape):
        raise ValueError("grad must be [*ids.shape, d]")
    n, d, n_rows = ids.numel(), grad.shape[-1], int(n_rows)
    if n_rows < 0:
        raise ValueError("n_rows must not be negative")
    grad, stride = _rows(grad if grad.dim() == 2 else grad.reshape(n, d), "grad")
    if out is None:
        if accumulate:
            raise ValueError("accumulate needs an out to add to")
    else:
        if not isinstance(out, torch.Tensor) or tuple(out.shape) != (n_rows, d) or out.dtype != grad.dtype:
            raise ValueError("out must be [n_rows, d] of grad's type")
        if (d > 1 and out.stride(1) != 1) or (n_rows > 1 and out.stride(0) < d):
            raise ValueError("out's rows must be contiguous and must not overlap")
        if _overlap(out, grad) or _overlap(out, ids):
            raise ValueError("out must not overlap grad or ids")
    with _On(grad, ids, out) as on:
        if out is None:
            out = torch.empty((n_rows, d), dtype=grad.dtype, device=grad.device)
        ws = on.workspace(_abi.lib().mfsgd_embedding_grad_workspace(n, n_rows, d))
        _abi.check(_abi.lib().mfsgd_hip_embedding_grad(
            grad.data_ptr(), stride, ids.data_ptr(), n, n_rows, d, scale, _DTYPES[grad.dtype], 1 if accumulate else 0,
            out.data_ptr(), out.stride(0) if n_rows > 1 else d, ws.data_ptr(), ws.numel(), on.stream))
    return out


def _loss_args(x, table, targets, bias, scale):
    x, xs = _rows(x, "x")
    table, ts = _rows(table, "table")
    targets = _ids(targets, "targets")
    n, d = x.shape
    if table.shape[1] != d or table.dtype != x.dtype:
        raise ValueError("x and table must have rows of one length and type")
    if d > 256:
        raise ValueError("softmax_loss: rows of at most 256 elements")
    if table.shape[0] < 1:
        raise ValueError("softmax_loss: the table has no items")
    if tuple(targets.shape) != (n,):
        raise ValueError("targets must have an element for every row of x")
    if not 1e-20 <= scale <= 1e20:
        raise ValueError("scale must be from 1e-20 to 1e20")
    return x, xs, table, ts, targets, _vector(bias, table.shape[0], "bias")


def _aligned(table, stride):
    """MFSGD_TABLE_ALIGNED where it holds: the workspace then leaves out what only other tables need."""
    return 2 if table.data_ptr() % 16 == 0 and stride % 8 == 0 and stride < 1 << 20 else 0


def softmax_loss(x, table, targets, bias=None, scale=1.0):
    """Cross entropy of the softmax over all items: (loss [n], lse [n]) in float32, with the logits
    z = scale * x @ table.T + bias, lse = logsumexp(z), loss = lse - z[targets].  Rows of at most 256 elements.  A padding row
    (target < 0) has loss and lse 0 and its x is not looked at; a target behind the table gives a loss that is not a number.  A
    bias of -inf takes an item out of the catalogue, whatever its row holds; as a target it gives the loss +inf (and no
    gradient).  float32's lowest value does the same for an item whose row is finite; bias / scale has to stay in float32
    otherwise.  A logit that is +inf or not a number makes its row's loss and lse not a number, the target's logit as any other;
    so may any logit of an infinite float32 element.  scale is from 1e-20 to 1e20; elements of x and table are of at most 1e20."""
    x, xs, table, ts, targets, bias = _loss_args(x, table, targets, bias, scale)
    n, d = x.shape
    with _On(x, table, targets, bias) as on:
        both = torch.empty((2, n), dtype=torch.float32, device=x.device)
        ws = on.workspace(_abi.lib().mfsgd_softmax_loss_workspace(n, table.shape[0], d, _DTYPES[x.dtype], _aligned(table, ts)))
        _abi.check(_abi.lib().mfsgd_hip_softmax_loss(
            x.data_ptr(), xs, table.data_ptr(), ts, targets.data_ptr(), None if bias is None else bias.data_ptr(), n,
            table.shape[0], d, scale, _DTYPES[x.dtype], both.data_ptr(), both.data_ptr() + 4 * n, ws.data_ptr(), ws.numel(),
            on.stream))
    loss, lse = both.unbind()
    return loss, lse


def softmax_loss_grads(x, table, targets, bias=None, scale=1.0, weights=1.0):
    """(loss, lse, dx, dtable, dbias): `softmax_loss` and the gradients of sum(weights * loss).  `weights` is a number or a
    float32 tensor with an element for every row (1 / n: the mean over n rows).  dx and dtable have the type of x, summed in
    fp32 (of bfloat16 rows the probabilities, times a row's weight for dtable, are rounded to bfloat16 before they are multiplied;
    not the target's share); dbias is float32, None without a bias."""
    x, xs, table, ts, targets, bias = _loss_args(x, table, targets, bias, scale)
    n, d = x.shape
    n_items = table.shape[0]
    each = _vector(weights, n, "weights") if isinstance(weights, torch.Tensor) else None
    with _On(x, table, targets, bias, each) as on:
        both = torch.empty((2, n), dtype=torch.float32, device=x.device)
        dx = torch.empty((n, d), dtype=x.dtype, device=x.device)
        dtable = torch.empty((n_items, d), dtype=x.dtype, device=x.device)
        dbias = None if bias is None else torch.empty(n_items, dtype=torch.float32, device=x.device)
        ws = on.workspace(_abi.lib().mfsgd_softmax_loss_workspace(n, n_items, d, _DTYPES[x.dtype], 1 + _aligned(table, ts)))
        _abi.check(_abi.lib().mfsgd_hip_softmax_loss_grads(
            x.data_ptr(), xs, table.data_ptr(), ts, targets.data_ptr(), None if bias is None else bias.data_ptr(),
            None if each is None else each.data_ptr(), 1.0 if each is not None else float(weights), n, n_items, d, scale,
            _DTYPES[x.dtype], both.data_ptr(), both.data_ptr() + 4 * n, dx.data_ptr(), dtable.data_ptr(),
            None if dbias is None else dbias.data_ptr(), ws.data_ptr(), ws.numel(), on.stream))
    loss, lse = both.unbind()
    return loss, lse, dx, dtable, dbias


def _dense(t):
    """Every element of the storage stretch exactly once, in any order of dimensions."""
    if t.is_contiguous():
        return True
    at = 1
    for s, n in sorted((s, n) for n, s in zip(t.shape, t.stride()) if n != 1):
        if s != at:
            return False
        at *= n
    return True


class _Set:
    """A set of tensors and the host arrays of their addresses, sizes and types (which live as long as it does)."""

    def __init__(self, tensors, name):
        self.tensors = [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)
        if not self.tensors:
            raise ValueError(f"{name} is empty")
        try:
            self.dtypes = array("i", [_DTYPES[t.dtype] for t in self.tensors])
        except (KeyError, AttributeError):
            raise TypeError(f"{name} must be float32 or bfloat16 tensors") from None
        self.sizes = array("q", [t.numel() for t in self.tensors])
        self.odd = [i for i, t in enumerate(self.tensors) if not t.is_contiguous()]
        for i in self.odd:
            if self.sizes[i] and not _dense(self.tensors[i]):
                raise ValueError(f"{name} must be dense tensors (no gaps, no element twice)")
        self.addresses = array("Q", [t.data_ptr() for t in self.tensors])
        self.n = len(self.tensors)

    def args(self):
        return self.sizes.buffer_info()[0], self.dtypes.buffer_info()[0], self.n


def grad_norm(tensors):
    """sqrt of the sum of all squares of all tensors (float32 and bfloat16 in any mix), as a float32 tensor of no dimensions."""
    grads = _Set(tensors, "tensors")
    with _On(*grads.tensors) as on:
        norm = torch.empty((), dtype=torch.float32, device=on.device)
        sizes, dtypes, n = grads.args()
        ws = on.workspace(_abi.lib().mfsgd_grad_norm_workspace(sizes, n))
        _abi.check(_abi.lib().mfsgd_hip_grad_norm(grads.addresses.buffer_info()[0], sizes, dtypes, n, norm.data_ptr(), ws.data_ptr(),
                                                  ws.numel(), on.stream))
    return norm


def clip_grads(tensors, max_norm, out=None):
    """Scales all tensors by min(1, max_norm / norm), norm being their global norm, in place or into `out` (tensors of the same
    sizes and types, in the same order of elements).  Returns the norm before clipping, without waiting for it."""
    grads = _Set(tensors, "tensors")
    if not max_norm > 0:
        raise ValueError("max_norm must be positive")
    to = grads
    if out is not None:
        to = _Set(out, "out")
        if to.dtypes != grads.dtypes or to.sizes != grads.sizes or any(
                to.tensors[i].shape != grads.tensors[i].shape or to.tensors[i].stride() != grads.tensors[i].stride()
                for i in grads.odd + to.odd):
            raise ValueError("out must have a tensor like each of tensors")
    with _On(*grads.tensors, *(to.tensors if to is not grads else ())) as on:
        norm = torch.empty((), dtype=torch.float32, device=on.device)
        sizes, dtypes, n = grads.args()
        ws = on.workspace(_abi.lib().mfsgd_grad_norm_workspace(sizes, n))
        _abi.check(_abi.lib().mfsgd_hip_clip_grads(grads.addresses.buffer_info()[0], to.addresses.buffer_info()[0], sizes, dtypes, n,
                                                   max_norm, norm.data_ptr(), ws.data_ptr(), ws.numel(), on.stream))
    return norm


def check_step(users, items, user_vecs, item_vecs, b_i):
    """What ExplicitMF.ranking_step takes, checked before anything runs: a step is done whole or not at all."""
    for t, name in ((users, "users"), (items, "items")):
        if not isinstance(t, torch.Tensor) or t.dtype != torch.int32:
            raise TypeError(f"ranking_step: {name} must be an int32 ROCm tensor")
        if t.dim() != 1 or t.shape != users.shape:
            raise ValueError("ranking_step: users and items must have one dimension and the same length")
    for t, name in ((user_vecs, "user_vecs"), (item_vecs, "item_vecs")):
        if not isinstance(t, torch.Tensor) or t.dtype not in _DTYPES:
            raise TypeError(f"ranking_step: {name} must be a float32 or bfloat16 ROCm tensor, which is updated in place")
    if user_vecs.dim() != 2 or item_vecs.dim() != 2 or user_vecs.shape[1] != item_vecs.shape[1] or user_vecs.dtype != item_vecs.dtype:
        raise ValueError("ranking_step: user_vecs and item_vecs must have rows of one length and type")
    if b_i is not None:
        if not isinstance(b_i, torch.Tensor) or b_i.dtype != torch.float32:
            raise TypeError("ranking_step: b_i must be a float32 ROCm tensor, which is updated in place")
        if b_i.shape != item_vecs.shape[:1]:
            raise ValueError("ranking_step: b_i must have an element for every item")
    tables = [t for t in (user_vecs, item_vecs, b_i) if t is not None]
    if not all(_once(t) for t in tables):
        raise ValueError("ranking_step: a table that is updated in place must not hold an element twice")
    if any(_share(a, b) and not (a is item_vecs and same_table(user_vecs, item_vecs)) for i, a in enumerate(tables) for b in tables[:i]):
        raise ValueError("ranking_step: user_vecs, item_vecs and b_i must not share memory, unless user_vecs is item_vecs")


def _once(t):
    """Whether every element has a place of its own: each dimension steps over all that the ones with smaller steps reach."""
    reach = 0
    for s, n in sorted((s, n) for s, n in zip(t.stride(), t.shape) if n > 1):
        if s <= reach:
            return False
        reach += s * (n - 1)
    return True


def same_table(a, b):
    return a.data_ptr() == b.data_ptr() and a.shape == b.shape and a.stride() == b.stride()
