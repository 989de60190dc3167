"""Layers beside the encodings and MLPs of nets.py: a row lookup with scaling (``Embedding``), a root-mean-square norm with the
residual's addition (``RMSNorm``) and a gated feed-forward block (``GatedMLP``), on the kernels of libnerf_hip.so
(nerf_embedding_*, nerf_rmsnorm_*, nerf_gated_mlp_*).  The reference has none of them; its per-image codes ``latent_emb[n]``
(nets.py:132) are the lookup's unscaled case.

Each is a function on tensors (``embedding``, ``rms_norm``, ``gated_mlp``) and a module that owns one ``params`` tensor, as the
modules of nets.py do.  Element types: float32, float16, bfloat16.  Sums are held in float32 and rounded once, results are the
same bits every time, gradients included.  Calls go to the device of their tensors and that device's current stream; workspaces
come from torch's allocator on every call, so calls may overlap, and be captured into graphs, freely.

Derivatives are those of torch.autograd's backward pass, once.  Forward-mode tangents, torch.func's transforms and make_fx are refused;
torch.jit.trace records the calls, torch.compile breaks its graph at them.

Capturing a backward pass: as with every torch autograd graph, no eager graph of the same leaves may be alive then (its
gradient accumulation belongs to the stream it ran on); ``torch.autograd.grad`` inside the capture avoids accumulation altogether.
"""
import math

import torch
import torch.nn as nn
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from ._lib import check, lib

DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
PRECISIONS = {'float32': torch.float32, 'float16': torch.float16, 'bfloat16': torch.bfloat16}
ACTIVATIONS = {'silu': 0, 'gelu': 1, 'relu': 2}


_current_device, _current_stream = torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream
_transforms, _tracing = torch._C._functorch.peek_interpreter_stack, torch._C._get_tracing_state
_modes, _mode_of = torch._C._len_torch_dispatch_stack, torch._C._get_dispatch_mode
_early_modes, _early_mode_of = torch._ops._len_torch_dispatch_stack_pre_dispatch, torch._ops._get_dispatch_mode_pre_dispatch
_PROXY = torch._C._TorchDispatchModeKey.PROXY


def _launch(device, fn, what, *args):
    """fn(*args, stream): on the tensors' device, made current for the launch, and that device's current stream."""
    # make_fx on real tensors, also above autograd: it would record the allocation and not the launch
    if _modes() and _mode_of(_PROXY) is not None or _early_modes() and _early_mode_of(_PROXY) is not None:
        raise RuntimeError('%s: a graph of torch operations cannot hold this kernel (torch.fx.experimental.proxy_tensor.make_fx)' % what)
    if device == _current_device():
        rc = fn(*args, _current_stream(device))
    else:
        with torch.cuda.device(device):
            rc = fn(*args, _current_stream(device))
    if rc:
        check(rc, what)


def _dtype(t, what):
    d = DTYPES.get(t.dtype)
    if d is None:
        raise TypeError('%s must be float32, float16 or bfloat16 (got %s)' % (what, t.dtype))
    return d


def _device(what, first, second, third=None):
    """Index of the GPU that all of them are on."""
    device = first.get_device()
    if device < 0 or second.get_device() != device or (third is not None and third.get_device() != device):
        for t in (first, second, third):
            if t is not None and not t.is_cuda:
                raise RuntimeError('nerf_amd kernels need tensors on the GPU (got %s); there is no CPU path' % t.device)
        raise ValueError('%s: tensors on different devices (%s)' % (what, ', '.join(str(t.device) for t in (first, second, third) if t is not None)))
    return device


def _rows16(t):
    """Contiguous and 16-byte aligned (a copy where it is not: a view may start anywhere)."""
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _workspace(nbytes, what, like):
    """A workspace on `like`'s device; None where none is needed."""
    if nbytes <= 0:
        if nbytes < 0:
            raise ValueError('%s: sizes out of range' % what)
        return None
    return like.new_empty(nbytes, dtype=torch.uint8)


def _at(t):
    return None if t is None else t.data_ptr()


def _recorded(a, b, c=None):
    """Whether a call goes through its autograd function: where a gradient will be asked for, and inside forward-mode differentiation
    (whose tangents travel beside tensors that need no gradient), torch.func's transforms and torch.jit.trace.  The kernels write
    through raw pointers, which none of those sees.  The function refuses the first two by name, as it has no `jvp` and no
    `setup_context`; a traced program records it as a call, with its checks of arguments."""
    return (torch.is_grad_enabled() and (a.requires_grad or b.requires_grad or (c is not None and c.requires_grad))
            or forward_ad._current_level >= 0 or _transforms() is not None or _tracing() is not None)


def _first_order(fn):
    """Backward passes are kernels, not differentiable again: `once_differentiable`, which says so where a graph of the backward pass
    is being made, and which the ordinary backward pass need not go through (it takes 5 us of a small layer's 50)."""
    marked = once_differentiable(fn)

    def backward(ctx, *grads):
        return marked(ctx, *grads) if torch.is_grad_enabled() else fn(ctx, *grads)
    return staticmethod(backward)


# ---- row lookup -----------------------------------------------------------------------------------------------------------

def embedding(index, table, scale=1.0):
    """scale * table[index]: index int64 [...], table [n_entries, dim] -> [..., dim] of the table's type.

    An index outside [0, n_entries) gives a row of zeros and no gradient (nets.py:132 raises there; a kernel cannot).  The
    table's gradient is dense; the rows of an entry are added in an order that `index` fixes."""
    call = _EmbeddingFn.apply if _recorded(table, index) else _embedding_fwd
    return call(table, index, float(scale))


def _embedding_fwd(table, index, scale):
    if index.dtype != torch.int64:
        raise TypeError('index must be int64 (got %s)' % index.dtype)
    if table.dim() != 2 or table.shape[1] < 1:
        raise ValueError('table must be [n_entries, dim] (got %s)' % (tuple(table.shape),))
    _dtype(table, 'table')
    device = _device('embedding', index, table)
    table, index = table.contiguous(), index.contiguous()
    entries, dim = table.shape
    out = table.new_empty(index.shape + (dim,))
    _launch(device, lib().nerf_embedding_fwd, 'nerf_embedding_fwd', table.data_ptr(), DTYPES[table.dtype], entries, dim,
            index.data_ptr(), index.numel(), scale, out.data_ptr())
    return out


class _EmbeddingFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, index, scale):
        ctx.save_for_backward(index)
        ctx.shape, ctx.scale = table.shape, scale
        return _embedding_fwd(table, index, scale)

    @_first_order
    def backward(ctx, dout):
        (index,) = ctx.saved_tensors
        entries, dim = ctx.shape
        index, d = index.contiguous(), dout.contiguous()
        code, rows = DTYPES[d.dtype], index.numel()
        dtable = d.new_empty((entries, dim))
        n = lib().nerf_embedding_bwd_workspace_bytes(code, entries, dim, rows)
        ws = _workspace(n, 'nerf_embedding_bwd', d)
        _launch(d.get_device(), lib().nerf_embedding_bwd, 'nerf_embedding_bwd', index.data_ptr(), d.data_ptr(), code, rows, entries, dim,
                ctx.scale, dtable.data_ptr(), _at(ws), n)
        return dtable, None, None


class Embedding(nn.Module):
    """`n_entries` rows of `n_output_dims`, looked up by index (one flat concept of nets.py: a ``params`` table)."""

    def __init__(self, n_entries, n_output_dims, scale=1.0, precision='float32', device='cuda', seed=None):
        super().__init__()
        if precision not in PRECISIONS:
            raise ValueError('precision must be float32, float16 or bfloat16')
        self.n_output_dims, self.scale = n_output_dims, float(scale)
        g = None if seed is None else torch.Generator(device='cpu').manual_seed(seed)
        init = (torch.rand(n_entries, n_output_dims, generator=g) * 2 - 1) * 1e-4     # as the hash table starts
        self.params = nn.Parameter(init.to(device=device, dtype=PRECISIONS[precision]))

    def forward(self, index):
        return embedding(index, self.params, self.scale)


# ---- norm -----------------------------------------------------------------------------------------------------------------

def rms_norm(x, weight, residual=None, eps=1e-6):
    """x / sqrt(mean(x^2) + eps) * weight over the last axis.  With `residual` (x's shape and type): (the norm of s, s) with
    s = x + residual rounded to x's type.  weight [dim]: x's type or float32."""
    call = _NormFn.apply if _recorded(x, weight, residual) else _norm_fwd
    return call(x, weight, residual, float(eps))


def _norm_fwd(x, weight, residual, eps):
    code = _dtype(x, 'x')
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError('x must have a last axis of at least one column (got %s)' % (tuple(x.shape),))
    if weight.dim() != 1 or weight.shape[0] != x.shape[-1]:
        raise ValueError('weight must be [%d] (got %s)' % (x.shape[-1], tuple(weight.shape)))
    if weight.dtype != x.dtype and weight.dtype != torch.float32:
        raise TypeError('weight must be %s or float32 (got %s)' % (x.dtype, weight.dtype))
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype):
        raise ValueError('residual must be of x\'s shape and type (got %s %s beside %s %s)'
                         % (tuple(residual.shape), residual.dtype, tuple(x.shape), x.dtype))
    if not eps >= 0:
        raise ValueError('eps must not be negative')
    device = _device('rms_norm', x, weight, residual)
    x, w = x.contiguous(), weight.contiguous()
    dim = x.shape[-1]
    y = torch.empty_like(x)
    res = total = None
    if residual is not None:
        res, total = residual.contiguous(), torch.empty_like(x)
    _launch(device, lib().nerf_rmsnorm_fwd, 'nerf_rmsnorm_fwd', x.data_ptr(), _at(res), w.data_ptr(), code, DTYPES[w.dtype],
            x.numel() // dim, dim, eps, _at(total), y.data_ptr())
    return y if total is None else (y, total)


class _NormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, residual, eps):
        out = _norm_fwd(x, weight, residual, eps)
        ctx.save_for_backward(x if residual is None else out[1], weight)
        ctx.eps = eps
        ctx.set_materialize_grads(False)
        return out

    @_first_order
    def backward(ctx, dy, dsum=None):
        total, weight = ctx.saved_tensors
        need_x, need_w, need_r = ctx.needs_input_grad[:3]
        if dy is None:      # only the sum was used
            return dsum if need_x else None, torch.zeros_like(weight) if need_w else None, dsum if need_r else None, None
        s, w, d = total.contiguous(), weight.contiguous(), dy.contiguous()
        dim = s.shape[-1]
        rows = s.numel() // dim
        ds = None if dsum is None else dsum.contiguous()
        dx = torch.empty_like(s) if need_x or need_r else None
        dw = torch.empty_like(w) if need_w else None
        n = lib().nerf_rmsnorm_bwd_workspace_bytes(rows, dim)
        ws = _workspace(n, 'nerf_rmsnorm_bwd', s)
        _launch(s.get_device(), lib().nerf_rmsnorm_bwd, 'nerf_rmsnorm_bwd', s.data_ptr(), w.data_ptr(), d.data_ptr(), _at(ds), DTYPES[s.dtype],
                DTYPES[w.dtype], rows, dim, ctx.eps, _at(dx), _at(dw), _at(ws), n)
        return dx if need_x else None, dw, dx if need_r else None, None


class RMSNorm(nn.Module):
    def __init__(self, n_dims, eps=1e-6, device='cuda'):
        super().__init__()
        self.eps = float(eps)
        self.params = nn.Parameter(torch.ones(n_dims, device=device))

    def forward(self, x, residual=None):
        return rms_norm(x, self.params, residual, self.eps)


# ---- gated block ----------------------------------------------------------------------------------------------------------

def gated_mlp(x, params, n_neurons, n_output_dims, activation='silu'):
    """(act(x Wg^T) * (x Wu^T)) Wd^T over the last axis of x.

    params: the flat weights Wg [n_neurons, n_in], Wu [n_neurons, n_in], Wd [n_output_dims, n_neurons], row-major, one after another
    (FullyFusedMLP's layout), of x's type -- or float32 beside a 16-bit x: they are rounded on every call then, and their
    gradient is float32.  activation: silu, gelu (erf form) or relu.  The hidden values are held in x's type (float16: they
    overflow above 65504)."""
    call = _GatedFn.apply if _recorded(x, params) else _gated_fwd
    return call(x, params, n_neurons, n_output_dims, activation)


def _gated_shape(x, params, n_neurons, n_output_dims, activation):
    """Checks the arguments; (element type, n_in, n_neurons, n_out, activation) as the library takes them, and the device."""
    code = _dtype(x, 'x')
    if activation not in ACTIVATIONS:
        raise ValueError('activation must be one of %s (got %r)' % (', '.join(ACTIVATIONS), activation))
    if x.dim() < 1 or x.shape[-1] < 1 or n_neurons < 1 or n_output_dims < 1:
        raise ValueError('x must have a last axis, and it, n_neurons and n_output_dims at least one column')
    if params.dim() != 1 or params.numel() != (2 * x.shape[-1] + n_output_dims) * n_neurons:
        raise ValueError('params must be [%d] for widths %d -> %d -> %d (got %s)' % (
            (2 * x.shape[-1] + n_output_dims) * n_neurons, x.shape[-1], n_neurons, n_output_dims, tuple(params.shape)))
    if params.dtype != x.dtype and params.dtype != torch.float32:
        raise TypeError('params must be %s or float32 (got %s)' % (x.dtype, params.dtype))
    device = _device('gated_mlp', x, params)
    return code, x.shape[-1], int(n_neurons), int(n_output_dims), ACTIVATIONS[activation], device


def _gated_fwd(x, params, n_neurons, n_output_dims, activation):
    return _gated_run(x, params, _gated_shape(x, params, n_neurons, n_output_dims, activation), False)[0]


def _gated_run(x, params, shape, keep):
    code, n_in, neurons, n_out, act, device = shape
    x, w = _rows16(x), _rows16(params.to(x.dtype))
    rows = x.numel() // n_in
    y = x.new_empty(x.shape[:-1] + (n_out,))
    saved = None
    n = (lib().nerf_gated_mlp_fwd_workspace_bytes if keep else lib().nerf_gated_mlp_alone_workspace_bytes)(code, rows, n_in, neurons, n_out)
    ws = _workspace(n, 'nerf_gated_mlp_fwd', x)
    if keep:
        kept = lib().nerf_gated_mlp_saved_floats(code, rows, n_in, neurons, n_out)
        saved = x.new_empty(kept, dtype=torch.float32) if kept else None
    _launch(device, lib().nerf_gated_mlp_fwd, 'nerf_gated_mlp_fwd', w.data_ptr(), x.data_ptr(), code, rows, n_in, neurons, n_out, act,
            y.data_ptr(), _at(saved), _at(ws), n)
    return y, saved


class _GatedFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, params, n_neurons, n_output_dims, activation):
        ctx.shape = _gated_shape(x, params, n_neurons, n_output_dims, activation)
        y, saved = _gated_run(x, params, ctx.shape, any(ctx.needs_input_grad))
        ctx.save_for_backward(x, params, saved)
        return y

    @_first_order
    def backward(ctx, dy):
        x, params, saved = ctx.saved_tensors
        code, n_in, neurons, n_out, act, device = ctx.shape
        need_x, need_p = ctx.needs_input_grad[:2]
        x, w, d = _rows16(x), _rows16(params.to(x.dtype)), _rows16(dy)
        rows = x.numel() // n_in
        dx = torch.empty_like(x) if need_x else None
        dparams = params.new_empty(params.shape) if need_p else None
        n = lib().nerf_gated_mlp_bwd_workspace_bytes(code, rows, n_in, neurons, n_out)
        ws = _workspace(n, 'nerf_gated_mlp_bwd', x)
        _launch(device, lib().nerf_gated_mlp_bwd, 'nerf_gated_mlp_bwd', w.data_ptr(), x.data_ptr(), d.data_ptr(), _at(saved), code, rows,
                n_in, neurons, n_out, act, _at(dx), _at(dparams), DTYPES[params.dtype], _at(ws), n)
        return dx, dparams, None, None, None


class GatedMLP(nn.Module):
    """Gated counterpart of nets.FullyFusedMLP: one flat ``params`` tensor, Xavier-uniform.

    precision: the type the block computes in.  ``params`` is a float32 master copy; ``module.to(torch.bfloat16)`` (or
    float16, matching `precision`) keeps the weights themselves in it, which is what a serving program wants -- otherwise every call
    rounds them."""

    def __init__(self, n_input_dims, n_output_dims, n_neurons, activation='silu', precision='float32', device='cuda', seed=None):
        super().__init__()
        if precision not in PRECISIONS:
            raise ValueError('precision must be float32, float16 or bfloat16')
        if activation not in ACTIVATIONS:
            raise ValueError('activation must be one of %s (got %r)' % (', '.join(ACTIVATIONS), activation))
        self.n_input_dims, self.n_output_dims, self.n_neurons = n_input_dims, n_output_dims, n_neurons
        self.activation, self.dtype = activation, PRECISIONS[precision]
        g = None if seed is None else torch.Generator(device='cpu').manual_seed(seed)
        chunks = []
        for o, n in ((n_neurons, n_input_dims), (n_neurons, n_input_dims), (n_output_dims, n_neurons)):
            chunks.append((torch.rand(o * n, generator=g) * 2 - 1) * math.sqrt(6.0 / (o + n)))
        self.params = nn.Parameter(torch.cat(chunks).to(device))

    def forward(self, x):
        return gated_mlp(x.to(self.dtype), self.params, self.n_neurons, self.n_output_dims, self.activation)
