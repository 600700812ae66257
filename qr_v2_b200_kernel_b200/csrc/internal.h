// What the library's translation units share. Hidden: none of it is part of the C ABI.
#pragma once

#define QRB200_HIDDEN __attribute__((visibility("hidden")))

// qrb200.cu
QRB200_HIDDEN int qrb200_internal_check_device();         // the current device is an sm_100 GPU, its failure word registered
QRB200_HIDDEN int* qrb200_internal_status_word(int dev);  // device address of dev's mapped failure word, or null
QRB200_HIDDEN void qrb200_internal_count_launch();
// quant.cu: reads and clears its own device failure word; a site, 0, or -1 for a CUDA error
QRB200_HIDDEN int qrb200_internal_quant_site();
