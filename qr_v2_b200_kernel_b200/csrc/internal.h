// What the library's translation units share. Hidden: none of it is part of the C ABI.
#pragma once

#define QRB200_HIDDEN __attribute__((visibility("hidden")))

// qrb200.cu
QRB200_HIDDEN int qrb200_internal_check_device();  // the current device is an sm_100 GPU, its failure word registered with all of these
QRB200_HIDDEN void qrb200_internal_count_launch();
// quant.cu, fp8.cu, kv8.cu: each has a device failure word of its own, which the first reads and clears (a site, 0, or -1 for a
// CUDA error), and a pointer to the device's mapped one, which the second sets on the current device.
QRB200_HIDDEN int qrb200_internal_quant_site();
QRB200_HIDDEN int qrb200_internal_fp8_site();
QRB200_HIDDEN int qrb200_internal_kv8_site();
QRB200_HIDDEN bool qrb200_internal_quant_register(int* word);
QRB200_HIDDEN bool qrb200_internal_fp8_register(int* word);
QRB200_HIDDEN bool qrb200_internal_kv8_register(int* word);
