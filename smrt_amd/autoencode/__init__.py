"""Auto-encoders on the MI355X HIP backend (reference package: smrt/autoencode)."""
from .topography import *      # noqa: F401,F403
from .vae import *             # noqa: F401,F403
from .data_parallel import *   # noqa: F401,F403
from .ae import *              # noqa: F401,F403

# The layers work on torch tensors and need torch to be imported, which takes longer than all the rest of the package (1.0 s without it, 3.0 s
# with it): it waits until one of their names is asked for.
_LAYERS = {"dense": "layers", "dense_backward": "layers", "dense_grouped": "layers", "dense_grouped_backward": "layers", "layer_norm": "layers",
           "layer_norm_backward": "layers", "pack_rows": "layers", "unpack_rows": "layers", "PackedRows": "layers", "ClassDecoders": "class_decoders",
           "layers": None, "class_decoders": None}

__all__ = [s for s in dir() if not s.startswith("_")] + list(_LAYERS)


def __getattr__(name):
    if name not in _LAYERS:
        raise AttributeError("module %r has no attribute %r" % (__name__, name))
    from importlib import import_module
    module = import_module("." + (_LAYERS[name] or name), __name__)
    value = globals()[name] = getattr(module, name) if _LAYERS[name] else module
    return value


def __dir__():
    return sorted(set(globals()) | set(_LAYERS))
