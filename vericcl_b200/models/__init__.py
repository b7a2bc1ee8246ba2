"""Collective front ends (the "model families" of a collective library).

* :class:`CollectiveEngine` — AllReduce / AllGather / ReduceScatter on torch
  tensors with synthesized, verified schedules.
* :class:`GradBucketAllReduce` — data-parallel gradient buckets with a fused
  scale, one schedule replayed for every bucket.
* :class:`ExpertExchange` — tokens to the experts of every rank and back around
  an AllToAll, with gradients.
"""
from .collectives import CollectiveEngine
from .experts import ExpertExchange
from .grad_bucket import GradBucketAllReduce, DEFAULT_BUCKET_BYTES

__all__ = ["CollectiveEngine", "ExpertExchange", "GradBucketAllReduce", "DEFAULT_BUCKET_BYTES"]
