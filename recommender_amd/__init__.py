"""recommender_amd - MI355X-native blocked-SGD matrix factorization behind the Python surface of
dtrager02/Recommender (ExplicitMF, BlockScheduler, SubSample, sgd / sgd2 / mse2).

Only the hot path lives here: csrc/ (hand-written HIP kernels + the C-ABI of include/mfsgd.h) and the
host-side mirror of the reference's interface.  There is no CPU fallback."""
from .SubSample import SubSample  # noqa: F401
from .RayBlockScheduler import BlockScheduler, consumer  # noqa: F401
from .SGDRecommender import ExplicitMF  # noqa: F401
from .Recommender import Recommender  # noqa: F401
from .numba_methods import sgd, sgd2, block_sgd, mse, mse2, rmse_exact  # noqa: F401

_MINIBATCH = ("embedding", "embedding_grad", "softmax_loss", "softmax_loss_grads", "grad_norm", "clip_grads")

__all__ = ["ExplicitMF", "Recommender", "BlockScheduler", "SubSample", "consumer",
           "sgd", "sgd2", "block_sgd", "mse", "mse2", "rmse_exact", *_MINIBATCH]


def __getattr__(name):
    """The minibatch operators come with torch, which the rest of the package imports only where it is used."""
    if name in _MINIBATCH or name == "minibatch":
        from importlib import import_module
        module = import_module(".minibatch", __name__)
        globals().update({n: getattr(module, n) for n in _MINIBATCH})
        return globals()[name] if name in _MINIBATCH else module
    raise AttributeError(f"module {__name__!r} has no attribute {name!r}")
