"""MI355X (gfx950) implementation of the GLIF_3 V1 cell hot path of
JavierGalvan9/V1_GLIF_model: the event-driven synaptic-current operator with its
custom gradient, and the fused GLIF_3 step with BPTT, as HIP kernels behind the
C ABI in include/glif.h.

Python mirror of the reference interface:
  ops.make_pre_ind_table, ops.calculate_synaptic_currents   (models.py:103-373)
  models.V1Column                                          (models.py:450-1135)
Sequence operators and the readout that is trained with the column and runs beside it:
  sequence.layer_norm, dropout, linear, short_conv, state_space_scan; readout.SequenceReadout
Synthetic networks of the benchmark configurations: synthetic.make_network.
"""
__version__ = "0.1.0"
