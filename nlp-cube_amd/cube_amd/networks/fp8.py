"""nn.Linear in 8-bit floating point (`cube_linear_fp8`): weights quantised once, rows on the way.  For the Linear layers of a
transformer that runs beside the parser (the LM encoder of cube/networks/lm.py:121-211 is one); inference only."""
import torch

from cube_amd import hip


class Fp8Weight(torch.Tensor):
    """What an Fp8Linear answers with for `weight`: shape, type and device as of a Linear's weight; whatever computes with it gets the
    values that the 8-bit rows stand for.  Read only.  (torch's encoder layers look at the weights of their Linear layers, and call the
    layers only where one of them is of a class of its own, as this is.)"""

    @staticmethod
    def __new__(cls, rows, dtype):
        return torch.Tensor._make_wrapper_subclass(cls, (rows.rows, rows.columns), dtype=dtype, device=rows.q.device)

    def __init__(self, rows, dtype):
        self._rows = rows

    def __repr__(self):
        return "Fp8Weight(%d, %d, dtype=%s, device=%s)" % (*self.shape, self.dtype, self.device)

    @classmethod
    def __torch_function__(cls, func, types, args=(), kwargs=None):   # its being here is what the layers look for
        with torch._C.DisableTorchFunctionSubclass():
            return func(*args, **(kwargs or {}))

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        if func._schema.is_mutable:
            raise ValueError("an Fp8Linear's weight cannot be written: %s" % func)
        args, kwargs = torch.utils._pytree.tree_map(lambda t: t._rows.float().to(t.dtype) if isinstance(t, cls) else t, (args, kwargs or {}))
        return func(*args, **kwargs)


class Fp8Linear(torch.nn.Module):
    """Stands for `linear` (same call, same shapes, the input's type out): e4m3 weights with one power-of-two scale per row and 128
    columns, activations quantised the same way per call, fp32 sums.  Made on the device of `linear`'s weight, an MI355X."""

    def __init__(self, linear):
        super().__init__()
        self.in_features, self.out_features = linear.in_features, linear.out_features
        rows = hip.quant_fp8(linear.weight.detach())
        self.register_buffer("q", rows.q)
        self.register_buffer("scale", rows.scale)
        self.register_buffer("bias", None if linear.bias is None else linear.bias.detach().float())
        self.register_buffer("kind", torch.empty(0, dtype=linear.weight.dtype, device=rows.q.device), persistent=False)   # the type that .half() and the like change

    @property
    def rows(self):
        """The weight as the kernels take it, from the buffers as they are now."""
        return hip.Fp8Rows(self.q, self.scale, self.in_features)

    def _apply(self, fn, *args, **kwargs):
        bias = self.bias
        super()._apply(fn, *args, **kwargs)
        if bias is not None:
            self.bias = bias.to(self.q.device)   # .half() and the like round it: what is added to the sums stays fp32
        return self

    @property
    def weight(self):
        return Fp8Weight(self.rows, self.kind.dtype)

    def forward(self, x):
        rows = x.reshape(-1, self.in_features)
        if rows.stride(1) != 1 or rows.stride(0) < self.in_features:   # transposed or broadcast rows
            rows = rows.contiguous()
        y = hip.linear_fp8(rows, self.rows, self.bias)
        return y.reshape(x.shape[:-1] + (self.out_features,))

    def extra_repr(self):
        return "in_features=%d, out_features=%d, bias=%s" % (self.in_features, self.out_features, self.bias is not None)


def quantise_linears(module):
    """Every nn.Linear below `module` (itself excepted) -> Fp8Linear, in place; one that stands in several places is one layer in all of
    them afterwards too.  -> how many layers."""
    made = {}
    for parent in list(module.modules()):
        for name, child in list(parent._modules.items()):   # (named_children leaves out a second name of the same child)
            if type(child) is torch.nn.Linear:
                if child not in made:
                    made[child] = Fp8Linear(child).train(child.training)
                setattr(parent, name, made[child])
    return len(made)
