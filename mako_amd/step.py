"""ctypes binding of include/mako_step.h: the operators around the sampler in a speculative decode step.

The operators are the HIP library's; this module only moves pointers.  It raises if libmako_sampler.so is missing -- there
is no CPU fallback.
"""
import ctypes as C

import numpy as np

from . import api

LOGITS_F32, LOGITS_BF16, LOGITS_F16 = 0, 1, 2
LOGITS_TYPES = {"float32": LOGITS_F32, "bfloat16": LOGITS_BF16, "float16": LOGITS_F16}
BLOCKS_OK, BLOCKS_SHORT, BLOCKS_WIDE, BLOCKS_TOKENS = 0, 1, 2, 3
MAX_ROWS, MAX_VOCAB, MAX_DRAFTS = 65535, 1048576, 64

# mako_row_cut
CUT_DTYPE = np.dtype(
    [
        ("total", "<f8"),
        ("max_logit", "<f4"),
        ("temperature", "<f4"),
        ("cut_logit", "<f4"),
        ("cut_token", "<i4"),
        ("n_kept", "<u4"),
        ("top_token", "<i4"),
    ]
)


class CutDesc(C.Structure):
    _fields_ = [
        ("logits", C.c_void_p),
        ("logits_type", C.c_uint32),
        ("n_rows", C.c_uint32),
        ("logits_stride", C.c_int64),
        ("n_vocab", C.c_uint32),
        ("rows_per_params", C.c_uint32),
        ("params", C.c_void_p),
        ("mask", C.c_void_p),
        ("mask_stride", C.c_int64),
        ("out_cuts", C.c_void_p),
        ("out_probs", C.c_void_p),
        ("probs_stride", C.c_int64),
    ]


class VerifyDesc(C.Structure):
    _fields_ = [
        ("n_requests", C.c_uint32),
        ("max_drafts", C.c_uint32),
        ("n_vocab", C.c_uint32),
        ("target_type", C.c_uint32),
        ("target", C.c_void_p),
        ("target_stride", C.c_int64),
        ("target_cuts", C.c_void_p),
        ("target_mask", C.c_void_p),
        ("target_mask_stride", C.c_int64),
        ("draft", C.c_void_p),
        ("draft_type", C.c_uint32),
        ("reserved", C.c_uint32),
        ("draft_stride", C.c_int64),
        ("draft_cuts", C.c_void_p),
        ("draft_mask", C.c_void_p),
        ("draft_mask_stride", C.c_int64),
        ("draft_tokens", C.c_void_p),
        ("n_drafts", C.c_void_p),
        ("u", C.c_void_p),
        ("seq_len", C.c_void_p),
        ("out_tokens", C.c_void_p),
        ("out_accepted", C.c_void_p),
        ("out_seq_len", C.c_void_p),
    ]


class BlocksDesc(C.Structure):
    _fields_ = [
        ("n_requests", C.c_uint32),
        ("block_size", C.c_uint32),
        ("seq_len", C.c_void_p),
        ("new_len", C.c_void_p),
        ("block_table", C.c_void_p),
        ("table_stride", C.c_int64),
        ("max_blocks", C.c_uint32),
        ("free_capacity", C.c_uint32),
        ("n_blocks", C.c_void_p),
        ("out_n_blocks", C.c_void_p),
        ("free_blocks", C.c_void_p),
        ("n_free", C.c_void_p),
        ("out_n_free", C.c_void_p),
        ("max_tokens", C.c_uint32),
        ("reserved", C.c_uint32),
        ("out_start", C.c_void_p),
        ("out_status", C.c_void_p),
        ("out_slots", C.c_void_p),
        ("out_positions", C.c_void_p),
        ("out_request", C.c_void_p),
    ]


EXPORTS = [
    "mako_step_create",
    "mako_step_destroy",
    "mako_step_last_error",
    "mako_step_cut_rows",
    "mako_step_verify_drafts",
    "mako_step_assign_blocks",
]

_ready = set()


def load(path=None):
    """The C-ABI library (api.load()) with this header's functions declared."""
    lib = api.load(path)
    if id(lib) not in _ready:
        lib.mako_step_create.argtypes = [C.POINTER(C.c_void_p), C.c_int, C.c_uint32, C.c_uint32]
        lib.mako_step_destroy.argtypes = [C.c_void_p]
        lib.mako_step_destroy.restype = None
        lib.mako_step_last_error.restype = C.c_char_p
        lib.mako_step_last_error.argtypes = [C.c_void_p]
        lib.mako_step_cut_rows.argtypes = [C.c_void_p, C.POINTER(CutDesc), C.c_void_p]
        lib.mako_step_verify_drafts.argtypes = [C.c_void_p, C.POINTER(VerifyDesc), C.c_void_p]
        lib.mako_step_assign_blocks.argtypes = [C.c_void_p, C.POINTER(BlocksDesc), C.c_void_p]
        _ready.add(id(lib))
    return lib


class StepContext:
    """Owner of a mako_step_ctx: rows (requests) of up to max_rows, vocabularies of up to max_vocab."""

    def __init__(self, max_rows, max_vocab, device=0, lib_path=None):
        self.ptr = None
        self.lib = load(lib_path)
        p = C.c_void_p()
        rc = self.lib.mako_step_create(C.byref(p), device, max_rows, max_vocab)
        if rc != api.MAKO_OK:
            raise api.MakoError("mako_step_create: %d" % rc)
        self.ptr = p.value
        self.max_rows, self.max_vocab = max_rows, max_vocab

    def close(self):
        if getattr(self, "ptr", None):
            self.lib.mako_step_destroy(self.ptr)
            self.ptr = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def last_error(self):
        return self.lib.mako_step_last_error(self.ptr).decode()

    def _call(self, name, desc, stream):
        rc = getattr(self.lib, name)(self.ptr, C.byref(desc), stream.ptr if stream else None)
        if rc != api.MAKO_OK:
            raise api.MakoError("%s: %d %s" % (name, rc, self.last_error()))

    def cut_rows(self, desc, stream=None):
        """Enqueues mako_step_cut_rows of a CutDesc."""
        self._call("mako_step_cut_rows", desc, stream)

    def verify_drafts(self, desc, stream=None):
        """Enqueues mako_step_verify_drafts of a VerifyDesc."""
        self._call("mako_step_verify_drafts", desc, stream)

    def assign_blocks(self, desc, stream=None):
        """Enqueues mako_step_assign_blocks of a BlocksDesc."""
        self._call("mako_step_assign_blocks", desc, stream)
