"""go-tensor's B200 backend, Python side.

* ``gotensor.backend.CudaBackend`` — the CUDA device behind go-tensor's
  ``backend.Backend`` interface (the primitive path);
* ``gotensor.model.Model`` — the native fused training step of a Sequential
  model (the fused path), with data parallelism over NCCL.

* ``gotensor.loss.linear_cross_entropy`` — a classifier head's loss and gradients
  over a large vocabulary without keeping the logits;
* ``gotensor.optim.AdamW`` — one AdamW step over many tensors, states in the
  dtype or in 8 bits.

All call the C interfaces in ``include/`` through ctypes; nothing here runs
on the CPU in their place.
"""
from ._lib import ACT_NONE, ACT_RELU, ACT_SIGMOID, ACT_TANH, FLOAT32, FLOAT64, GTError  # noqa: F401
