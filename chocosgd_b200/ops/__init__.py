"""Hand-written sm_100a kernels (``csrc/``) and their Python bindings.

``_lib``      loader of the in-tree shared library (ctypes) and of the autograd nodes on top of it
``sgd``       fused multi-segment Nesterov / momentum / weight-decay update
``compress``  stand-alone sign pack/unpack, top-k, random-k, QSGD kernels
``gossip``    fused CHOCO step kernels with in-kernel NVLink push (the product path)
``gemm``      tcgen05 / TMEM GEMM
``norm``      layer normalisation, forward and backward
``dropout``   dropout from a counter-based generator, optionally with the residual sum; no stored mask
``ffn``       gated feed-forward block, forward and backward, and its form for few tokens
``nn``        layer classes used by the model zoo (conv / batch-norm / linear / LSTM / layer norm /
              dropout / gated feed-forward)
"""
