"""reels_amd: MI355X (gfx950) HIP implementation of Reels.jl's int8 frozen-weight LoRA linear.

The compute lives in libreels_hip.so (C ABI: include/reels_hip.h); this package is the host-side
mirror of the reference layer API (src/layers/quantization.jl, lora.jl, linear.jl, attention.jl).
"""
from ._lib import ReelsHIPError, ReelsHIPUnavailable, library_path  # noqa: F401
from .activations import (  # noqa: F401
    CompressedActivations,
    GeluTanhCompressedFunction,
    compress_activations,
    gelu_tanh_compressed,
)
from .attention import (  # noqa: F401
    TiledAttentionCache,
    memory_efficient_attention,
    memory_efficient_attention_backward,
)
from .gradients import clip_gradients, gradient_norm  # noqa: F401
from .layers import (  # noqa: F401
    DenseLayer,
    FrozenWeightTransfer,
    I8LoRALinearFunction,
    LoRALinear,
    QuantizedMatrix,
    _weight_mul,
    _weight_transpose_mul,
    frozen_weight_transfer,
    gelu_tanh,
    gelu_tanh_backward,
    i8lora_backward,
    i8lora_backward_gelu,
    i8lora_forward,
    i8lora_forward_gelu,
    linear,
    lora_backward,
    lora_forward,
    lora_parameters,
    merged_weight,
    move_weight,
    quantize_frozen_matrix,
    set_adapter_enabled,
    workspace_bytes,
)
from .microscaled import MicroscaledMatrix, microscaled_linear, quantize_microscaled  # noqa: F401
from .modulation import (  # noqa: F401
    KeptRows,
    ModulatedNormFunction,
    ModulatedNormGradients,
    ModulatedNormQuantized,
    ModulatedNormResult,
    modulated_norm,
    modulated_norm_backward,
    modulated_norm_quantized,
)
from .normalization import (  # noqa: F401
    RMSNormFunction,
    RMSNormGradients,
    RMSNormQuantized,
    RMSNormResult,
    rms_norm,
    rms_norm_backward,
    rms_norm_quantized,
)
from .quantized import quantize_rows, quantized_linear  # noqa: F401
from .rotary import (  # noqa: F401
    RotaryFunction,
    grid_positions,
    rotary,
    rotary_axes,
    rotary_backward,
    rotary_qk,
    rotary_qk_backward,
)
