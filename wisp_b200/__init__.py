"""wisp_b200: B200-native (sm_100a) paged fused-MoE layer.

The drop-in surface is ``wisp_b200.integrations.vllm`` (``install_wisp_moe``,
``is_installed``, ``WispMoEState``); the native library is
``wisp_b200/lib/libwisp_b200.so`` with the C ABI in ``include/wisp_b200.h``.
``wisp_b200.mx4`` has the MXFP4 operators (quantisation, grouped products, a
whole MoE layer for a few tokens) that ``WispMoEStateMX4`` pages experts for,
``wisp_b200.norm`` the norms around a block.
"""
__version__ = "0.1.0"
