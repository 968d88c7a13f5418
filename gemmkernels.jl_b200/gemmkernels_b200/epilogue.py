"""Epilogue vocabulary (src/epilogue.jl)."""
from __future__ import annotations


class Default:                    # src/epilogue.jl:14-34
    def __repr__(self):
        return "Epilogue.Default()"


class Bias:
    """Epilogue.Bias(pointer(bias)) (src/epilogue.jl:40-73): Float32 bias added after the
    regs_to_shared_d transform and before shared_to_global_d.  The reference indexes it by column
    (length N); `axis="row"` selects one value per row (length M) instead."""

    def __init__(self, bias, axis: str = "col"):
        if axis not in ("col", "row"):
            raise ValueError("axis must be 'col' or 'row'")
        self.bias = bias
        self.axis = axis

    def __repr__(self):
        return f"Epilogue.Bias(<{self.axis}>)"


class Fused:
    """The layer-level epilogues: one launch of gk_gemm_fused.  No counterpart in the reference.  The activation
    is None (none), Transform.ReLU(), GELU() or SiLU(); C, D and the pre-activation have one element type."""


class BiasActivationResidual(Fused):
    """D = act(alpha*A*B + bias) + beta*C.

    `bias` is Float32, one value per row of D (`axis="row"`, length M; per group in `matmul_grouped`: (M, groups))
    or per column (`axis="col"`, length N), or None.  C is the residual, added after the activation.
    `preactivation`, a column-major array like D, receives alpha*A*B + bias for the backward pass."""

    def __init__(self, bias=None, axis: str = "row", activation=None, preactivation=None):
        if axis not in ("col", "row"):
            raise ValueError("axis must be 'col' or 'row'")
        self.bias, self.axis, self.activation, self.preactivation = bias, axis, activation, preactivation

    def __repr__(self):
        return f"Epilogue.BiasActivationResidual(<{self.axis}>, {self.activation!r})"


class ActivationGradient(Fused):
    """D = (alpha*A*B + beta*C) * act'(Z): the gradient that a layer hands down, taken through the activation
    behind which Z was kept (`preactivation`, column-major like D; may be D itself)."""

    def __init__(self, preactivation, activation=None):
        self.preactivation, self.activation = preactivation, activation

    def __repr__(self):
        return f"Epilogue.ActivationGradient({self.activation!r})"
