"""CPU oracle of the two hot paths - TEST INFRASTRUCTURE, not product code.

Only tests/, __graft_entry__.smoke() and bench.py's CPU baseline (`cpu_baseline`, `--impl
reference`) may import this package, and only as the checker or the timed CPU restatement of the
reference; the product path (talm_b200) never imports it and fails loudly without its CUDA
library.

  oracle.nf4   numpy restatement of the NF4 dequantisation (solution/nf4_dequant.py:38-80,
               solution/qgroup.py:72-91, solution/test_fuzz.py:860-869)
  oracle.head  torch CPU restatement of the fused head (solution/test_kernels.py:70-83,
               solution/test_fuzz.py:145-185, solution/fused_head.py:126-182)

  oracle.adapter  float64 restatement of the adapted 4-bit projection
  oracle.ranks  how the ranks of a CPU test hand their results over

Pinning: the first two are checked against golden vectors that tests/golden/make_golden.py generated by
importing the reference's own Python functions (`_nf4_manual`, `reference_head`,
`_head_reference`, `labelled_first`, `LayerGroup` packing) on CPU.
"""

import multiprocessing

if multiprocessing.parent_process() is not None:  # a rank of a CPU test
    from . import ranks

    ranks.send_by_value()
