"""What the 8-bit linear layers share as modules."""
from torch import nn


class KeepsBias(nn.Module):
    """Layers whose bias goes with their weights: into their state and out of it, and to other devices.  Its type stays what it is when the
    model is converted, as the scales' does: it is rounded once, to the output's."""

    _version = 2  # states of version 1 have no bias: a layer that loads one keeps its own

    def _keep_bias(self, bias, copy):
        """A copy, so that a state that is loaded does not reach the caller's tensor; of a parameter only where `copy` is wanted."""
        if isinstance(bias, nn.Parameter):
            self.bias = nn.Parameter(bias.detach().clone(), bias.requires_grad) if copy else bias
        else:
            self.register_buffer("bias", None if bias is None else bias.detach().clone().requires_grad_(bias.requires_grad))

    def __setstate__(self, state):
        super().__setstate__(state)
        if "bias" in self.__dict__:  # of a layer that was pickled when its bias was a plain attribute
            self._keep_bias(self.__dict__.pop("bias"), copy=False)

    def _apply(self, fn, recurse=True):
        held = self._buffers.get("bias")
        super()._apply(fn, recurse)
        if held is not None and self.bias.dtype != held.dtype:
            self.bias = held.to(self.bias.device)
        return self

    def _load_from_state_dict(self, state_dict, prefix, local_metadata, *args, **kwargs):
        version = local_metadata.get("version")
        if (version is None or version < 2) and self.bias is not None:
            state_dict.setdefault(prefix + "bias", self.bias)
        return super()._load_from_state_dict(state_dict, prefix, local_metadata, *args, **kwargs)


class SettlesAnew(nn.Module):
    """Layers that fetch their weights early only from the second call on (``_settled``), counted from when the weights were last written."""

    _settled = False

    def _apply(self, fn, recurse=True):
        super()._apply(fn, recurse)
        self._settled = False
        return self

    def __setstate__(self, state):
        super().__setstate__(state)
        self._settled = False  # a copy's buffers are written on some stream too

    def _load_from_state_dict(self, *args, **kwargs):
        self._settled = False  # the buffers are about to be overwritten by a copy on some stream
        return super()._load_from_state_dict(*args, **kwargs)
