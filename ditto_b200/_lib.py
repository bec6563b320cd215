"""ctypes binding of libditto_b200.so (the C ABI declared in include/ditto_b200.h).

There is no CPU fallback: if the shared library is missing this module raises,
and every operator built on it fails with it.
"""
import ctypes
import os

_HERE = os.path.dirname(os.path.abspath(__file__))

OK = 0
ERR_INVALID_ARG = -1
ERR_UNSUPPORTED = -2
ERR_CUDA = -3
ERR_TIMEOUT = -4
ERR_WORKSPACE = -5
ERR_DRIVER = -6

DTYPE_FP16 = 0
DTYPE_BF16 = 1
OP_BMM_SOFTMAX_BMM = 0
OP_GEMM_RELU_GEMM = 1
OP_LESS_SCRATCH = 0x2000
FLAG_P_VIA_SMEM = 1
FLAG_ONE_TILE = 2
FLAG_TWO_TILES = 4
FLAG_NARROW = 8
FLAG_FEW = 16             # two threads a row, a CTA per tile or as many as the split says
FLAG_SPLIT_UNIT = 256     # 1, 2, 3, 4 of these: 1, 2, 4, 8 CTAs share a tile's keys
EPILOGUE_PAIR_MMA = 0x200
EPILOGUE_QUAD_MMA = 0x400
EPILOGUE_WIDE_MMA = 0x800
EPILOGUE_FLOW_MMA = 0x1000

STATUS_BAD_PAGE = 0x10001    # values of the status word beside those of expired waits
STATUS_NO_PAGES = 0x10002

Strides2, Strides3 = ctypes.c_longlong * 2, ctypes.c_longlong * 3


def _block(name, text):
    """A C struct of the header: "type: names" lines."""
    types = {"ptr": ctypes.c_void_p, "int": ctypes.c_int, "float": ctypes.c_float, "ll": ctypes.c_longlong, "s2": Strides2, "s3": Strides3}
    fields = [(f, types[kind]) for line in text.strip().splitlines() for kind, names in [line.split(":")] for f in names.split()]
    return type(name, (ctypes.Structure,), {"_fields_": fields})


MaskedArgs = _block("MaskedArgs", """
ptr: q k v out lse
s3: q_strides k_strides v_strides out_strides
int: batch M L heads kv_heads head_dim dtype causal
float: scale cap
ptr: slopes prefix documents""")
PagedArgs = _block("PagedArgs", """
ptr: q key_pages value_pages out
s2: q_strides out_strides
s3: key_strides value_strides
ptr: table lengths starts
ll: table_stride
int: tokens batch pages page table_cols heads kv_heads head_dim dtype
float: scale cap
ptr: slopes prefix""")
AppendArgs = _block("AppendArgs", """
ptr: keys values key_pages value_pages
s2: k_strides v_strides
s3: key_strides value_strides
ptr: table lengths starts
ll: table_stride
int: tokens batch pages page table_cols kv_heads head_dim""")
PoolsArgs = _block("PoolsArgs", """
ptr: base
int: count pages
ll: page_bytes stride_bytes""")
TablesArgs = _block("TablesArgs", """
ptr: table lengths references
ll: stride
int: sequences cols page pages""")

EXPORTS = (
    "ditto_b200_bmm_softmax_bmm",
    "ditto_b200_gemm_relu_gemm",
    "ditto_b200_gemm_relu_gemm_static_scratch",
    "ditto_b200_multi_head_attention",
    "ditto_b200_ffn",
    "ditto_b200_ffn_ws",
    "ditto_b200_workspace_bytes",
    "ditto_b200_mlp_cluster_slots",
    "ditto_b200_mlp_tiles_cut",
    "ditto_b200_masked_workspace_bytes",
    "ditto_b200_masked_attention",
    "ditto_b200_masked_attention_backward",
    "ditto_b200_paged_workspace_bytes",
    "ditto_b200_paged_attention",
    "ditto_b200_cache_append",
    "ditto_b200_cache_workspace_bytes",
    "ditto_b200_cache_copy",
    "ditto_b200_cache_reserve",
    "ditto_b200_cache_fork",
    "ditto_b200_cache_free",
    "ditto_b200_cache_compact",
    "ditto_b200_selftest_umma",
    "ditto_b200_selftest_umma_pair",
    "ditto_b200_selftest_ex2",
    "ditto_b200_selftest_wait_limit",
    "ditto_b200_check_status",
    "ditto_b200_strerror",
    "ditto_b200_last_cuda_error",
    "ditto_b200_kernel_launches",
    "ditto_b200_version",
)

# masked attention, the paged cache and its pages
MASKED_EXPORTS = tuple(name for name in EXPORTS if "masked" in name or "paged" in name or "_cache_" in name)


class DittoError(RuntimeError):
    """A non-zero status from the C ABI."""

    def __init__(self, code, where):
        self.code = code
        lib = load()
        msg = lib.ditto_b200_strerror(code).decode()
        detail = lib.ditto_b200_last_cuda_error().decode() if code in (ERR_CUDA, ERR_DRIVER) else ""
        super().__init__(f"{where}: {msg} (code {code}){' -- ' + detail if detail else ''}")


def library_path():
    return os.environ.get("DITTO_B200_LIB", os.path.join(_HERE, "lib", "libditto_b200.so"))


_lib = None


def load():
    """Load the shared library once and attach argument types."""
    global _lib
    if _lib is not None:
        return _lib
    path = library_path()
    if not os.path.exists(path):
        raise ImportError(
            f"{path} not found: build it with `python -m ditto_b200.build_lib` (needs nvcc); "
            "ditto_b200 has no CPU fallback")
    lib = ctypes.CDLL(path)
    vp, i, f, sz = ctypes.c_void_p, ctypes.c_int, ctypes.c_float, ctypes.c_size_t
    lib.ditto_b200_bmm_softmax_bmm.argtypes = [vp, vp, vp, vp, i, i, i, i, i, i, i, f, i, vp, sz, vp, vp]
    lib.ditto_b200_bmm_softmax_bmm.restype = i
    lib.ditto_b200_gemm_relu_gemm.argtypes = [vp, vp, vp, vp, i, i, i, i, i, i, i, i, vp, sz, vp, vp]
    lib.ditto_b200_gemm_relu_gemm.restype = i
    lib.ditto_b200_gemm_relu_gemm_static_scratch.argtypes = [vp, vp, vp, vp, i, i, i, i, i, i, i, i, vp, vp]
    lib.ditto_b200_gemm_relu_gemm_static_scratch.restype = i
    lib.ditto_b200_multi_head_attention.argtypes = [vp, vp, i, i, i, i, i, f, i, vp, vp]
    lib.ditto_b200_multi_head_attention.restype = i
    lib.ditto_b200_ffn.argtypes = [vp, vp, vp, vp, vp, vp, i, i, i, i, i, i, i, i, i, vp, vp]
    lib.ditto_b200_ffn.restype = i
    lib.ditto_b200_ffn_ws.argtypes = [vp, vp, vp, vp, vp, vp, i, i, i, i, i, i, i, i, i, vp, sz, vp, vp]
    lib.ditto_b200_ffn_ws.restype = i
    lib.ditto_b200_workspace_bytes.argtypes = [i, i, i, i, i, i, i]
    lib.ditto_b200_workspace_bytes.restype = sz
    lib.ditto_b200_mlp_cluster_slots.argtypes = [i, i]
    lib.ditto_b200_mlp_cluster_slots.restype = i
    lib.ditto_b200_mlp_tiles_cut.argtypes = [i, i, i, i, i, i, ctypes.POINTER(i)]
    lib.ditto_b200_mlp_tiles_cut.restype = i
    lib.ditto_b200_masked_workspace_bytes.argtypes = [vp, i]
    lib.ditto_b200_masked_workspace_bytes.restype = sz
    lib.ditto_b200_masked_attention.argtypes = [vp, vp, sz, vp, vp]
    lib.ditto_b200_masked_attention.restype = i
    lib.ditto_b200_masked_attention_backward.argtypes = [vp, vp, ctypes.POINTER(ctypes.c_longlong), vp, vp, vp, vp, sz, vp, vp]
    lib.ditto_b200_masked_attention_backward.restype = i
    lib.ditto_b200_paged_workspace_bytes.argtypes = [vp]
    lib.ditto_b200_paged_workspace_bytes.restype = sz
    lib.ditto_b200_paged_attention.argtypes = [vp, vp, sz, vp, vp]
    lib.ditto_b200_paged_attention.restype = i
    lib.ditto_b200_cache_append.argtypes = [vp, vp, vp]
    lib.ditto_b200_cache_append.restype = i
    lib.ditto_b200_cache_workspace_bytes.argtypes = [vp, i]
    lib.ditto_b200_cache_workspace_bytes.restype = sz
    lib.ditto_b200_cache_copy.argtypes = [vp, vp, vp, i, vp, vp]
    lib.ditto_b200_cache_copy.restype = i
    lib.ditto_b200_cache_reserve.argtypes = [vp, vp, vp, sz, vp, vp]
    lib.ditto_b200_cache_reserve.restype = i
    lib.ditto_b200_cache_fork.argtypes = [vp, vp, vp, vp, i, vp, sz, vp, vp]
    lib.ditto_b200_cache_fork.restype = i
    lib.ditto_b200_cache_free.argtypes = [vp, vp, i, vp, vp]
    lib.ditto_b200_cache_free.restype = i
    lib.ditto_b200_cache_compact.argtypes = [vp, vp, vp, ctypes.c_longlong, vp, vp, sz, vp, vp]
    lib.ditto_b200_cache_compact.restype = i
    lib.ditto_b200_selftest_umma.argtypes = [vp, vp, vp, i, i, i, i, i, vp, vp]
    lib.ditto_b200_selftest_umma.restype = i
    lib.ditto_b200_selftest_umma_pair.argtypes = [vp, vp, vp, i, i, i, i, vp, vp]
    lib.ditto_b200_selftest_umma_pair.restype = i
    lib.ditto_b200_selftest_ex2.argtypes = [vp, vp, i, i, vp]
    lib.ditto_b200_selftest_ex2.restype = i
    lib.ditto_b200_selftest_wait_limit.argtypes = [i, vp, vp]
    lib.ditto_b200_selftest_wait_limit.restype = i
    lib.ditto_b200_check_status.argtypes = [vp, vp, ctypes.POINTER(ctypes.c_int)]
    lib.ditto_b200_check_status.restype = i
    lib.ditto_b200_strerror.argtypes = [i]
    lib.ditto_b200_strerror.restype = ctypes.c_char_p
    lib.ditto_b200_last_cuda_error.argtypes = []
    lib.ditto_b200_last_cuda_error.restype = ctypes.c_char_p
    lib.ditto_b200_kernel_launches.argtypes = []
    lib.ditto_b200_kernel_launches.restype = ctypes.c_ulonglong
    lib.ditto_b200_version.argtypes = []
    lib.ditto_b200_version.restype = i
    _lib = lib
    return lib


def check(code, where):
    if code != OK:
        raise DittoError(code, where)
