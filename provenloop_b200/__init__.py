"""provenloop_b200 -- B200-native (sm_100a) CKKS engine for TenSafe's
encrypted LoRA-delta hot path.

* ``provenloop_b200.tensafe_he``: drop-in for the PyO3 module ``tensafe_he``.
* ``provenloop_b200.backend``: engine adapter, ZeRo-MOAI deltas, DP noise.
* ``provenloop_b200.adapters``: plaintext LoRA adapters of many requests beside
  a shared projection, their gradients, and the clipping of these.
* ``provenloop_b200.logits``: penalties, biases and grammar masks on next-token
  logits, with the greedy pick.
* ``provenloop_b200.losses``: token log-probabilities, policy and preference
  losses, with their gradients for the logits.
* ``include/tsgpu.h`` / ``libtsgpu.so``: the C ABI underneath.
"""
__version__ = "0.1.0"
