"""The argument structures of include/cula_kda.h for the operators of a state space block, for tests that call the C entries themselves."""
import ctypes

from cula_b200 import _native

P, I, L, F = ctypes.c_void_p, ctypes.c_int, ctypes.c_longlong, ctypes.c_float
GARBAGE = 0x13                                                       # an address that is no one's, and not aligned


def _structure(name, *members):
    return type(name, (ctypes.Structure,), {"_fields_": [(m, t) for t, names in members for m in names.split()]})


ScanArgs = _structure("ScanArgs", (P, "x dt z Bm Cm"), (L, "x_row dt_row z_row b_row c_row x_seq dt_seq z_seq b_seq c_seq"),
                      (P, "A skip dt_bias h0 y hT states y_pre dy dhT dx ddt dz dBm dCm dA dskip dbias dh0 part_bc part_A part_skip part_bias "
                          "seg_state seg_dt cu_seqlens chunk_indices chunk_offsets seq_order"), (L, "rows"),
                      (I, "T D S G n_seqs num_chunks total_tokens seg_chunks cta_rows softplus fp32 vec_bc"))
StepArgs = _structure("StepArgs", (P, "x dt z Bm Cm A skip dt_bias state indices y"), (L, "x_row dt_row z_row b_row c_row"),
                      (I, "rows D S G pool softplus fp32 vec"), (P, "status"))
ConvStepArgs = _structure("ConvStepArgs", (P, "x w bias cache indices y"), (L, "x_row"), (I, "rows D W pool silu"), (P, "status"))
NormArgs = _structure("NormArgs", (P, "x r w y r_out rstd scale v dy dr_out dx dr part_w dw"), (L, "R x_row r_row"), (I, "D group fp32 res fp8"), (F, "eps"))


def call(entry, args, stream=None):
    return getattr(_native.lib(), "cula_kda_" + entry)(ctypes.byref(args), stream)
