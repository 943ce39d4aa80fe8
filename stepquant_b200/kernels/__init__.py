"""Device operators of the packed-state decode path (libstepquant_b200).

``pool``       PackedStatePool and the page layout; launches the fused step
               (synchronous pools) or readout + background writeback.
``writeback``  deferred / chunked background writeback under CUDA-graph capture.
``resources``  SM-bounded writeback streams (green contexts).
``profiles``   per-batch writeback budgets.

The operators around the recurrent state of a layer:

``norm``       residual root-mean-square norm, e4m3 activations with block scales.
``matmul``     product of e4m3 matrices with block scales.
``conv``       short causal convolution, for prompts and single tokens.
``scan``       selective state space scan, its single-token form and state pool.
"""
