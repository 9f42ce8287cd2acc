// C++ host-mirror check (include/vectoraccelerate.hpp): runs each class on inputs read from a
// directory and writes the outputs there as raw little-endian arrays; tests/test_gpu_cpp.py
// compares them with the CPU oracle.  Usage: va_example DIR Q N D C k nprobe
#include <cstdio>
#include <cstdlib>
#include <fstream>
#include <string>
#include <vector>

#include "vectoraccelerate.hpp"

namespace va = vectoraccelerate;

template <class T>
static std::vector<T> load(const std::string& path, size_t n) {
    std::vector<T> v(n);
    std::ifstream f(path, std::ios::binary);
    if (!f.read(reinterpret_cast<char*>(v.data()), std::streamsize(n * sizeof(T)))) {
        std::fprintf(stderr, "cannot read %s\n", path.c_str());
        std::exit(2);
    }
    return v;
}

template <class T>
static void save(const std::string& path, const std::vector<T>& v) {
    std::ofstream f(path, std::ios::binary);
    f.write(reinterpret_cast<const char*>(v.data()), std::streamsize(v.size() * sizeof(T)));
}

int main(int argc, char** argv) {
    if (argc != 8) {
        std::fprintf(stderr, "usage: %s DIR Q N D C k nprobe\n", argv[0]);
        return 2;
    }
    const std::string dir = argv[1];
    const uint32_t Q = std::atoi(argv[2]), N = std::atoi(argv[3]), D = std::atoi(argv[4]), C = std::atoi(argv[5]),
                   k = std::atoi(argv[6]), nprobe = std::atoi(argv[7]);
    try {
        va::Context ctx(0);
        va::Matrix q{load<float>(dir + "/q.bin", size_t(Q) * D), Q, D};
        va::Matrix x{load<float>(dir + "/x.bin", size_t(N) * D), N, D};
        std::vector<float> cen = load<float>(dir + "/c.bin", size_t(C) * D);

        va::FusedL2TopKKernel topk(ctx);
        va::SearchResult l2 = topk.findNearestNeighbors(q, x, k, VA_METRIC_L2SQ);
        save(dir + "/l2_idx.bin", l2.indices);
        save(dir + "/l2_dist.bin", l2.distances);
        va::SearchResult cs = topk.findNearestNeighbors(q, x, k, VA_METRIC_COSINE);
        save(dir + "/cos_idx.bin", cs.indices);

        va::DeviceBuffer<float> xd(ctx, x.data), qd(ctx, q.data), cd(ctx, cen);
        const uint32_t half = N / 2;
        std::vector<float> first(x.data.begin(), x.data.begin() + size_t(half) * D);
        std::vector<float> rest(x.data.begin() + size_t(half) * D, x.data.end());
        va::DeviceBuffer<float> x0(ctx, first), x1(ctx, rest);
        va::IVFIndex ivf(ctx, cd, C, x0, half, D, nprobe);
        ivf.add(x1, N - half);
        va::SearchResult iv = ivf.search(qd, Q, k);
        save(dir + "/ivf_idx.bin", iv.indices);

        va::KMeansPipeline km(ctx, C, 5, 0.0f);
        va::KMeansPipeline::Result kr = km.fit(xd, N, D, cen);
        save(dir + "/km_cen.bin", kr.centroids);
        save(dir + "/km_assign.bin", kr.assignments);

        va::ProductQuantizationKernel pq(ctx, {D, 4, 16, 5, 0.0f});
        va::DeviceBuffer<float> cb = pq.train(xd, N, 11);
        va::DeviceBuffer<uint8_t> codes = pq.encode(xd, N, cb);
        va::SearchResult pr = pq.search(qd, Q, cb, codes, N, k);
        save(dir + "/pq_cb.bin", cb.download());
        save(dir + "/pq_codes.bin", codes.download());
        save(dir + "/pq_idx.bin", pr.indices);

        // MetalComputeProvider: distances of query 0 and the nearest candidates of every query
        va::MetalComputeProvider prov(ctx);
        std::vector<float> q0(q.data.begin(), q.data.begin() + D);
        save(dir + "/prov_l2.bin", prov.batchDistance(q0, x, va::MetalComputeProvider::Metric::euclidean));
        save(dir + "/prov_cos.bin", prov.batchDistance(q0, x, va::MetalComputeProvider::Metric::cosine));
        save(dir + "/prov_dot.bin", prov.batchDistance(q0, x, va::MetalComputeProvider::Metric::dotProduct));
        std::vector<uint32_t> nn;
        std::vector<float> nd;
        for (auto m : {va::MetalComputeProvider::Metric::euclidean, va::MetalComputeProvider::Metric::cosine,
                       va::MetalComputeProvider::Metric::dotProduct})
            for (auto& row : prov.findNearestBatch(q, x, k, m))
                for (auto& p : row) {
                    nn.push_back(p.first);
                    nd.push_back(p.second);
                }
        save(dir + "/prov_nn_idx.bin", nn);
        save(dir + "/prov_nn_dist.bin", nd);

        // AcceleratedVectorIndex: handles, removal of every 7th vector, search, filtered search
        va::AcceleratedVectorIndex index(ctx, D, 16);
        std::vector<uint32_t> hs = index.insert(x);
        std::vector<uint32_t> gone;
        for (uint32_t i = 0; i < N; i += 7) gone.push_back(hs[i]);
        const uint32_t removed = index.remove(gone);
        va::SearchResult ir = index.search(q, k);
        save(dir + "/index_idx.bin", ir.indices);
        auto odd = [](uint32_t h) { return (h & 1u) == 1u; };
        std::vector<uint32_t> fi;
        for (auto& p : index.search(q0, k, odd)) fi.push_back(p.first);
        save(dir + "/index_filtered_idx.bin", fi);
        index.compact();
        std::ofstream(dir + "/index_counts.txt") << removed << " " << index.count() << " " << index.contains(hs[0])
                                                 << " " << index.contains(hs[1]);

        // AcceleratedVectorIndex (IVF): half the vectors, train with the given centroids, the other
        // half joins the lists, every 5th vector removed, then batch search through the lists
        va::AcceleratedVectorIndex ivx(ctx, D, va::IVFConfiguration{C, nprobe, 0}, 64);
        va::Matrix xa{first, half, D}, xb{rest, N - half, D};
        ivx.insert(xa);
        ivx.train(cen);
        ivx.insert(xb);
        std::vector<uint32_t> gone5;
        for (uint32_t i = 0; i < N; i += 5) gone5.push_back(i);
        ivx.remove(gone5);
        va::SearchResult vr = ivx.search(q, k);
        save(dir + "/ivx_idx.bin", vr.indices);
        save(dir + "/ivx_dist.bin", vr.distances);
        auto lists = ivx.lists();
        save(dir + "/ivx_off.bin", lists.first);
        save(dir + "/ivx_ids.bin", lists.second);
        std::ofstream(dir + "/ivx_state.txt") << ivx.isTrained() << " " << ivx.info().ivf_routed << " " << ivx.count();

        // the loss of the queries over the collection (target of query i: row i), its gradients clipped
        // together, the norm of the queries in fp32 and in 8 bits
        {
            std::vector<int64_t> targets(Q);
            for (uint32_t i = 0; i < Q; ++i) targets[i] = i;
            va::DeviceBuffer<float> dq(ctx, load<float>(dir + "/q.bin", size_t(Q) * D)), dx(ctx, load<float>(dir + "/x.bin", size_t(N) * D));
            va::DeviceBuffer<int64_t> dt(ctx, targets);
            const va_xent_desc d{dq.data(), dx.data(), dt.data(), nullptr, D, D, -100, Q, N, D, VA_DTYPE_F32, 0.25f};
            va::SoftmaxCrossEntropyKernel entropy(ctx);
            auto r = entropy.forward(d);
            va::DeviceBuffer<float> gq(ctx, size_t(Q) * D), gx(ctx, size_t(N) * D), norm(ctx, 1);
            entropy.backward(d, r.logSumExp, gq.data(), gx.data());
            save(dir + "/xent_loss.bin", r.loss.download());
            save(dir + "/xent_mean.bin", r.reduced.download());
            void* const tensors[2] = {gq.data(), gx.data()};
            const uint64_t sizes[2] = {gq.size(), gx.size()};
            const int32_t types[2] = {VA_DTYPE_F32, VA_DTYPE_F32};
            va::GradientClipKernel(ctx).encode(va_tensor_list{tensors, nullptr, sizes, types, 2}, 0.01f, norm.data());
            save(dir + "/clip_norm.bin", norm.download());
            save(dir + "/clip_gq.bin", gq.download());
            save(dir + "/clip_gx.bin", gx.download());
            va::RMSNormKernel rms(ctx);
            va::DeviceBuffer<float> weight(ctx, std::vector<float>(D, 0.5f)), inverse(ctx, Q), y(ctx, size_t(Q) * D), back(ctx, size_t(Q) * D),
                scales(ctx, Q), gr(ctx, size_t(Q) * D);
            va::DeviceBuffer<int8_t> codes(ctx, size_t(Q) * D);
            va_rms_desc n{dq.data(), nullptr, weight.data(), nullptr, inverse.data(), D, D, D, Q, D, VA_DTYPE_F32, 1e-6f};
            rms.encode(n, y.data());
            rms.quantize(n, VA_CODE_INT8, codes.data(), scales.data());
            rms.dequantize(codes.data(), VA_CODE_INT8, scales.data(), Q, D, VA_DTYPE_F32, back.data());
            n.out_inverse_rms = nullptr;
            rms.backward(n, y.data(), inverse.data(), gr.data(), nullptr);
            save(dir + "/rms_y.bin", y.download());
            save(dir + "/rms_back.bin", back.download());
            save(dir + "/rms_gr.bin", gr.download());

            // a step of the queries and the collection along those gradients, moments in 8 bits; the collection in 4 bits and its
            // scores; an item of each query's ten likeliest
            std::vector<va_adamw_tensor> list(2);
            std::vector<va::DeviceBuffer<uint8_t>> moments;
            std::vector<va::DeviceBuffer<float>> scale;
            float* const params[2] = {dq.data(), dx.data()};
            for (int i = 0; i < 2; ++i) {
                const size_t groups = (sizes[i] + 255) / 256;
                for (int m = 0; m < 2; ++m) {
                    moments.emplace_back(ctx, std::vector<uint8_t>(sizes[i], 0));
                    scale.emplace_back(ctx, std::vector<float>(groups, 0.0f));
                }
                va_adamw_tensor& t = list[i];
                t = va_adamw_tensor{};
                t.param = t.out_param = params[i];
                t.grad = tensors[i];
                t.first = t.out_first = moments[2 * i].data(), t.second = t.out_second = moments[2 * i + 1].data();
                t.first_scales = t.out_first_scales = scale[2 * i].data(), t.second_scales = t.out_second_scales = scale[2 * i + 1].data();
                t.size = sizes[i], t.param_dtype = t.grad_dtype = VA_DTYPE_F32;
                t.rate_factor = t.decay_factor = 1.0f;
            }
            va::AdamWTensors listed(ctx, list, 8);
            va::AdamWKernel(ctx).encode(listed, va::AdamWKernel::parameters(1, 0.01));
            save(dir + "/adamw_q.bin", dq.download());
            save(dir + "/adamw_x.bin", dx.download());
            va::MicroscaledQuantizationKernel micro(ctx);
            va::MicroscaledRows items(ctx, N, D), queries(ctx, Q, D);
            va::DeviceBuffer<float> values(ctx, size_t(N) * D), scores(ctx, size_t(Q) * N), coded(ctx, size_t(Q) * N), u(ctx, std::vector<float>(Q, 0.375f));
            micro.quantize(dx.data(), VA_DTYPE_F32, items);
            micro.quantize(dq.data(), VA_DTYPE_F32, queries);
            micro.dequantize(items, VA_DTYPE_F32, values.data());
            micro.product(dq.data(), VA_DTYPE_F32, Q, items, VA_DTYPE_F32, scores.data(), 0.25f);
            micro.product(queries, items, VA_DTYPE_F32, coded.data(), 0.25f);
            save(dir + "/mx_values.bin", values.download());
            save(dir + "/mx_scores.bin", scores.download());
            save(dir + "/mx_coded.bin", coded.download());
            va::SoftmaxSamplingKernel sampling(ctx);
            va_sample_desc sd = va::SoftmaxSamplingKernel::describe(scores.data(), VA_DTYPE_F32, u.data(), Q, N);
            sd.top_k = 10;
            auto drawn = sampling.sample(sd);
            save(dir + "/sample_items.bin", drawn.items.download());
            save(dir + "/sample_log.bin", drawn.logProbability.download());
            auto falling = sampling.sample(sd, VA_SAMPLE_BY_LOGIT);
            save(dir + "/falling_items.bin", falling.items.download());
            save(dir + "/falling_log.bin", falling.logProbability.download());
        }

        std::string kind = "none";
        try {
            topk.findNearestNeighbors(q, x, 0);
        } catch (const va::VectorError& e) {
            kind = e.kind();
        }
        std::ofstream(dir + "/error_kind.txt") << kind;
    } catch (const va::VectorError& e) {
        std::fprintf(stderr, "VectorError(%s): %s\n", e.kind(), e.what());
        return 1;
    }
    std::printf("va_example: ok\n");
    return 0;
}
