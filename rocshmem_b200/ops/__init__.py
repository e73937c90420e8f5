"""Operations on symmetric tensors: collectives, MoE dispatch/combine, GEMMs and fused paths; attention operators."""
from . import collectives  # noqa: F401
