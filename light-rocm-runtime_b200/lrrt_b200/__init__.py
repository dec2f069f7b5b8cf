"""Python mirror of the lrrt interfaces on B200 (ctypes over the C ABIs).

``runtime`` wraps the lr_* calls (light-rocm-runtime include/lrrt/lrrt.h);
``qwen`` wraps the Qwen2 FP32 resident decode driver (include/lrrt_qwen.h);
``ops`` wraps the paged-cache operators (include/lrrt_ops.h) for torch tensors
and is imported on its own.
The compute path is the sm_100a cubins loaded through lr_module_load_hsaco; this
package only moves arguments across the C ABI.
"""
from .native import LrrtError, check, driver, runtime  # noqa: F401
