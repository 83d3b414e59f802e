"""weightbridge_b200: trainer -> rollout weight transfer for B200 (sm_100a).

Public API (the names of the reference package ``wbridge``, ``wbridge/__init__.py:3-17``):
``WeightSender``, ``WeightReceiver``, ``WeightReceiverController``, ``WeightData``,
``dtype_str_to_torch``, ``dtype_to_str``; plus ``TransferConfig`` and the layout adapters
``MegatronLayout`` / ``FSDPLayout`` (trainers) and ``SGLangLayout`` (rollout), and the operators
of an RL step beside the sync: ``token_logprobs`` (and ``policy_gap``, which checks a sync by them),
``AdamW`` and ``grad_norm``.
"""
from .core.shard import (WeightData, check_shard_compatibility, original_total_numel,
                         shards_iterator)
from .utils.config import TransferConfig
from .utils.dtypes import dtype_str_to_torch, dtype_to_str


def __getattr__(name):
    # the control plane pulls in zmq/fastapi; import it on first use
    if name in ("WeightSender", "WeightReceiver", "WeightReceiverController", "SyncStats"):
        from . import control
        return getattr(control, name)
    if name == "MegatronLayout":
        from .parallel.megatron import MegatronLayout
        return MegatronLayout
    if name in ("FSDPLayout", "HFLayout"):
        from .parallel import fsdp
        return getattr(fsdp, name)
    if name in ("SGLangLayout", "VLLMLayout"):
        from .parallel import sglang
        return getattr(sglang, name)
    if name in ("token_logprobs", "TokenLogprobs"):
        from .ops import logprobs
        return getattr(logprobs, name)
    if name in ("policy_gap", "PolicyGap"):
        from .control import policy
        return getattr(policy, name)
    if name in ("AdamW", "grad_norm"):
        from .ops import optim
        return getattr(optim, name)
    raise AttributeError(name)


__all__ = [
    "WeightData", "WeightSender", "WeightReceiver", "WeightReceiverController", "TransferConfig",
    "check_shard_compatibility", "shards_iterator", "original_total_numel", "dtype_str_to_torch",
    "dtype_to_str", "MegatronLayout", "FSDPLayout", "HFLayout", "SGLangLayout", "VLLMLayout",
    "token_logprobs", "TokenLogprobs", "policy_gap", "PolicyGap", "AdamW", "grad_norm",
]
__version__ = "0.1.0"
