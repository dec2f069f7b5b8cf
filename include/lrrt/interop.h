/*
 * Queues over CUDA streams that another part of the program owns (no
 * counterpart in light-rocm-runtime, whose queues are always its own): work
 * given to such a queue runs on that stream, in order with everything else
 * the program puts there.
 */
#ifndef LRRT_INTEROP_H_
#define LRRT_INTEROP_H_

#include "lrrt/lrrt.h"

#ifdef __cplusplus
extern "C" {
#endif

/*
 * `stream` is a CUstream or cudaStream_t of the device's primary context
 * (NULL: that context's legacy default stream). lr_queue_destroy waits for the
 * stream and releases the queue, not the stream, which has to outlive it.
 */
LRRT_API lr_status_t lr_queue_wrap_stream(lr_device_t device, void *stream, lr_queue_t **queue);

/*
 * Whether work given to the queue (NULL: the device's default queue) is being
 * captured in a CUDA graph: nothing may be allocated or freed for it then. 1
 * too where the queue is the legacy default stream and another is captured.
 */
LRRT_API lr_status_t lr_queue_is_capturing(lr_device_t device, lr_queue_t *queue,
                                           uint32_t *capturing);

#ifdef __cplusplus
}
#endif

#endif /* LRRT_INTEROP_H_ */
