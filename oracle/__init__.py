"""CPU oracle of the two hot paths - TEST INFRASTRUCTURE, not product code.

Only tests/, __graft_entry__.smoke() and bench.py's CPU baseline (`cpu_baseline`, `--impl
reference`) may import this package, and only as the checker or the timed CPU restatement of the
reference; the product path (talm_b200) never imports it and fails loudly without its CUDA
library.

  oracle.nf4   numpy restatement of the NF4 dequantisation (solution/nf4_dequant.py:38-80,
               solution/qgroup.py:72-91, solution/test_fuzz.py:860-869)
  oracle.head  torch CPU restatement of the fused head (solution/test_kernels.py:70-83,
               solution/test_fuzz.py:145-185, solution/fused_head.py:126-182)

Pinning: both are checked against golden vectors that tests/golden/make_golden.py generated by
importing the reference's own Python functions (`_nf4_manual`, `reference_head`,
`_head_reference`, `labelled_first`, `LayerGroup` packing) on CPU.
"""

import multiprocessing
import multiprocessing.util
import time

if multiprocessing.parent_process() is not None:
    # A rank of a CPU test puts its tensors on a queue and exits, but the parent fetches them by file
    # descriptor from the sender: a rank that has already gone leaves it without. The sender stays
    # for a moment after its queue has been told to finish (10) and before the socket that the parent
    # connects to is unlinked (0; finalizers of a lower priority run later).
    multiprocessing.util.Finalize(None, time.sleep, args=(5,), exitpriority=5)
