"""MI355X-native Prioritized DCI k-nearest-neighbour search.

Drop-in for the Python API of niopeng/dciknn_cuda (`DCI`, `MDCI`), backed by
hand-written gfx950 HIP kernels behind a C-ABI shared library, and the operators that
training or serving a model on its rows and neighbours takes (see `tokens.py`).
"""
__version__ = "0.1.0"

_TOKENS = ["embed", "embed_grad", "token_logprobs", "distill_loss", "distill_step", "gated_scan", "grad_norm", "clip_grads", "verify_drafts"]
__all__ = ["DCI", "MDCI"] + _TOKENS


def __getattr__(name):
    # DCI, MDCI and the operators on tokens need the compiled libraries (there is no fallback: without them this
    # raises ImportError); the build script and the workload generators of this package
    # must be importable before anything is compiled, hence the late import.
    if name in _TOKENS:
        from . import tokens
        globals().update({n: getattr(tokens, n) for n in _TOKENS})
        return globals()[name]
    if name in __all__:
        from . import core
        globals().update(DCI=core.DCI, MDCI=core.MDCI)
        return globals()[name]
    raise AttributeError("module %r has no attribute %r" % (__name__, name))
